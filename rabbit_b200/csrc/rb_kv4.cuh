// rb_kv4.cuh -- the paged 4-bit key / value cache: its layout in HBM, shared
// by the kernels that write it (rb_kv4.cu) and the attention that reads it
// (rb_kv4_attn.cu).
//
// The unit is a granule: 16 consecutive tokens of one KV head, 576 bytes for
// each of its NG = ceil(head_dim / 32) channel groups, contiguous:
//   K codes  [16 tokens][4 t][NG groups] 32-bit words
//   K scales [16 tokens][NG] bf16
//   V codes  [16 tokens][8 g'][NG] 16-bit words
//   V scales [16 tokens][NG] bf16
// A page of one layer is [n_kv_heads][page_size / 16] granules, a layer
// [n_pages] pages. Codes are stored plus 8 (4 bits, 1..15).
//
// The words are in the order in which the attention's matrix instructions
// take them, so a code goes from its word to a register of an operand with at
// most a shift and a mask:
//  * K word t of a group holds channels 8 t .. 8 t + 7 in its nibbles; lane
//    (g, t) of a warp multiplies the channels of words t of token g, for all
//    groups, and reads them as one piece of 4 NG bytes.
//  * V word g of a group holds channels 4 g .. 4 g + 3; lane (g, t) takes the
//    words g of four tokens, for all groups one piece of 2 NG bytes. In shared
//    memory the lanes' pieces of one load are 8 pieces (g) of each of 4 tokens
//    (t): piece g of token j lies at place g' = g ^ (4 * bit 1 of j), which
//    puts the four tokens of a load (kv4_token) into different banks.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/rabbit_cuda.h"
#include "rb_runtime.h"

namespace rb {

constexpr int kKv4Group = 32;      // channels that share a scale
constexpr int kKv4Granule = 16;    // tokens of a granule
constexpr int kKv4MaxGroups = 8;   // head_dim <= 256

// Offsets in a granule of NG groups.
__host__ __device__ constexpr int kv4_row(int ng) { return 16 * ng; }  // code bytes of a token
__host__ __device__ constexpr int kv4_ks(int ng) { return 256 * ng; }
__host__ __device__ constexpr int kv4_v(int ng) { return 288 * ng; }
__host__ __device__ constexpr int kv4_vs(int ng) { return 544 * ng; }
__host__ __device__ constexpr int kv4_bytes(int ng) { return 576 * ng; }

// Place of V piece g of token j.
__host__ __device__ constexpr int kv4_vplace(int j, int g) { return g ^ ((j & 2) << 1); }

// Error bits of a cache's error word; set by atomicOr, so none hides another.
#define RB_KV4_ERR_SLOT 16
#define RB_KV4_ERR_PAGE 32
#define RB_KV4_ERR_LEN 64
#define RB_KV4_ERR_ROWS 128
#define RB_KV4_ERR_WAIT 256  // a bounded wait ran out

// One layer of a cache as the kernels see it.
struct Kv4View {
    uint8_t *base;
    int nkv, hd, ng, page, n_pages;
    int shift;  // page = 2^shift, or -1
    int *err;
    size_t head_nbytes, page_nbytes;  // of a page: one KV head's part, all of it
    int64_t n_slots;
    __host__ __device__ size_t head_bytes() const { return head_nbytes; }
    __host__ __device__ size_t page_bytes() const { return page_nbytes; }
    __host__ __device__ int64_t slots() const { return n_slots; }
    __device__ __forceinline__ uint8_t *granule(int64_t slot, int head) const {
        return row(slot) + (size_t)head * head_bytes();
    }
    // The slot's granule of KV head 0.
    __device__ __forceinline__ uint8_t *row(int64_t slot) const {
        // (a division in 64 bits takes five times the instructions of one in 32)
        const int64_t p = shift >= 0 ? slot >> shift : slot >> 31 ? slot / page : (int)slot / page;
        const int r = (int)(slot - p * page);
        return base + (size_t)p * page_bytes() + (size_t)(r / kKv4Granule) * kv4_bytes(ng);
    }
};

}  // namespace rb

struct rabbit_cuda_kv4 {
    int device = -1;
    rb::DevCtx *ctx = nullptr;
    int n_layers = 0;
    rb::Kv4View view = {};      // of layer 0
    size_t layer_bytes = 0;
    int *d_err = nullptr;       // the error word, and what a check took of it
    std::mutex taking;          // one check at a time
    bool withhold = false;      // test hook for the next attention
    rb::Kv4View layer(int l) const {
        rb::Kv4View v = view;
        v.base += (size_t)l * layer_bytes;
        return v;
    }
};
