// rb_kv4_attn.cu -- attention over the paged 4-bit key / value cache.
#include <math.h>

#include <atomic>
#include <new>

#include "rb_kv4_chunk.cuh"
#include "rb_kv4_decode.cuh"
#include "rb_launch.h"

struct rabbit_cuda_kv4_scratch {
    int device = -1, ng = 0;
    float *part = nullptr;
    unsigned *count = nullptr;
};

namespace rb {

static_assert(kMaxDevices <= 32, "a bit for each device");

template <int NG, int RB, bool SPLIT>
static cudaError_t launch_decode(const Kv4AttnArgs &a, const rabbit_cuda_kv4 *kv, cudaStream_t s) {
    using C = DecodeCfg<NG, RB, SPLIT>;
    static_assert(C::kSmem + 5120 <= kMaxDynSmem, "shared memory of a CTA, the static part with it");
    auto kern = k_kv4_decode<NG, RB, SPLIT>;
    static std::atomic<uint32_t> ready{0};  // devices whose limit is raised
    if (!(ready.load() >> kv->device & 1u)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        ready.fetch_or(1u << kv->device);
    }
    const int grid = kv->ctx->sm_count;
    return launch_pdl(kern, dim3(grid < kDecodeMaxGrid ? grid : kDecodeMaxGrid), dim3(C::kThreads), C::kSmem, s, a);
}

// CTAs of the chunk kernel from which it is taken. Its time goes by the positions of one
// CTA and the CTAs an SM takes in turn; the other's, which spreads a KV head's positions
// over the SMs, by the whole batch's granules times ceil(rows / 16). us, chunk / decode kernel,
// bf16, 8 KV heads, for equal numbers of query rows a KV head and sequence:
//   sequences x rows      1000 positions   4096        16384
//   4 x 64 (32 CTAs)      29 / 31          91 / 51     343 / 136
//   4 x 128 (64)          29 / 46          92 / 83     343 / 250
//   10 x 20 (80)          29 / 34          92 / 59     351 / 163
//   10 x 64 (80)          29 / 50          93 / 96     353 / 307
//   16 x 20 (128)         29 / 44          93 / 81     345 / 249
//   16 x 64 (128)         30 / 70          93 / 140    345 / 479
//   64 x 20 (512)         73 / 124         331 / 241   -
//   64 x 48 (512)         76 / 188         332 / 355   -
// The rule goes by the CTAs alone, since the host does not know the lengths. It gives away
// 1.1 to 2.1 times for 17 to 32 rows over more than 2000 positions (decoding with drafts),
// and up to 1.6 times elsewhere.
constexpr int kChunkMinCtas = 72;

template <int NG>
static cudaError_t launch_chunk(const Kv4AttnArgs &a, int tiles, const rabbit_cuda_kv4 *kv, cudaStream_t s) {
    using C = ChunkCfg<NG>;
    static_assert(C::kSmem + 4096 <= kMaxDynSmem, "shared memory of a CTA, the static part with it");
    auto kern = k_kv4_chunk<NG>;
    static std::atomic<uint32_t> ready{0};  // devices whose limit is raised
    if (!(ready.load() >> kv->device & 1u)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        ready.fetch_or(1u << kv->device);
    }
    return launch_pdl(kern, dim3(tiles, a.c.nkv, a.n_seqs), dim3(C::kThreads), C::kSmem, s, a);
}

// Rows of a tile: as many as a KV head has query rows of a sequence, up to what
// the output leaves of the registers; a granule's codes are made once for all.
template <int NG, bool SPLIT>
static cudaError_t launch_rows(const Kv4AttnArgs &a, const rabbit_cuda_kv4 *kv, cudaStream_t s) {
    if constexpr (NG <= 4) {
        const int64_t rows = (int64_t)a.max_q * (a.nh / a.c.nkv);
        if constexpr (!SPLIT) {
            // Where only few sequences of a batch have many rows, the others would each take a
            // chunk of 64 for their own one: so half a chunk a sequence on average. 64 sequences
            // of 1024 positions, 4 heads a KV head, 1 / 4 / 16 of them with 256 rows and the rest
            // with one (20 / 68 / 268 rows on average): 150 / 211 / 460 us here, 121 / 267 / 726
            // us in the decode kernel; one of them with 64 rows (8): 106 and 74 us.
            const int64_t tiles = (rows + ChunkCfg<NG>::kRows - 1) / ChunkCfg<NG>::kRows;
            const int64_t most = rows < ChunkCfg<NG>::kRows / 2 ? rows : ChunkCfg<NG>::kRows / 2;
            if (rows > 16 && tiles * a.c.nkv * a.n_seqs >= kChunkMinCtas &&
                (int64_t)a.T * (a.nh / a.c.nkv) >= most * a.n_seqs)
                return launch_chunk<NG>(a, (int)tiles, kv, s);
        }
        if (rows > 8) return launch_decode<NG, 2, SPLIT>(a, kv, s);
    }
    return launch_decode<NG, 1, SPLIT>(a, kv, s);
}

template <bool SPLIT>
static cudaError_t launch_attention(const Kv4AttnArgs &a, const rabbit_cuda_kv4 *kv, cudaStream_t s) {
    switch (a.c.ng) {
        case 1: return launch_rows<1, SPLIT>(a, kv, s);
        case 2: return launch_rows<2, SPLIT>(a, kv, s);
        case 3: return launch_rows<3, SPLIT>(a, kv, s);
        case 4: return launch_rows<4, SPLIT>(a, kv, s);
        case 5: return launch_rows<5, SPLIT>(a, kv, s);
        case 6: return launch_rows<6, SPLIT>(a, kv, s);
        case 7: return launch_rows<7, SPLIT>(a, kv, s);
        default: return launch_rows<8, SPLIT>(a, kv, s);
    }
}

}  // namespace rb

using namespace rb;

extern "C" {

int rabbit_cuda_kv4_scratch_create(const rabbit_cuda_kv4 *kv, rabbit_cuda_kv4_scratch **out) {
    if (!kv || !out) return fail(RABBIT_CUDA_ERR_ARGS, "kv4_scratch_create: NULL argument");
    *out = nullptr;
    auto *ws = new (std::nothrow) rabbit_cuda_kv4_scratch();
    if (!ws) return fail(RABBIT_CUDA_ERR_MEM, "kv4_scratch_create: out of host memory");
    ws->device = kv->device;
    ws->ng = kv->view.ng;
    // two partial results a CTA (the item its run continues, the one it leaves
    // unfinished) of the largest tile: outputs, then (reference, sum) pairs
    const size_t ctas = kDecodeMaxGrid;
    const size_t rows = ws->ng <= 4 ? 16 : 8;
    const size_t bytes = sizeof(float) * 2 * ctas * rows * (32 * ws->ng + 2);
    DeviceScope scope(kv->device);
    if (scope.status != RABBIT_CUDA_OK) {
        delete ws;
        return scope.status;
    }
    cudaError_t e;
    if ((e = cudaMalloc(&ws->part, bytes)) != cudaSuccess ||
        (e = cudaMalloc(&ws->count, sizeof(unsigned) * ctas)) != cudaSuccess ||
        (e = cudaMemset(ws->count, 0, sizeof(unsigned) * ctas)) != cudaSuccess ||
        (e = cudaStreamSynchronize(nullptr)) != cudaSuccess) {
        rabbit_cuda_kv4_scratch_free(ws);
        cudaGetLastError();
        return e == cudaErrorMemoryAllocation
                   ? fail(RABBIT_CUDA_ERR_MEM, "kv4_scratch_create: %zu bytes of device memory", bytes)
                   : cuda_fail(e, "kv4_scratch_create: device memory");
    }
    *out = ws;
    return ok();
}

int rabbit_cuda_kv4_scratch_free(rabbit_cuda_kv4_scratch *ws) {
    if (!ws) return ok();
    {
        DeviceScope scope(ws->device);
        if (ws->part) cudaFree(ws->part);
        if (ws->count) cudaFree(ws->count);
    }
    delete ws;
    return ok();
}

int rabbit_cuda_kv4_attention_dev(rabbit_cuda_kv4 *kv, int layer, rabbit_cuda_kv4_scratch *ws,
                                  int dtype, const void *d_q, int64_t q_stride, void *d_out,
                                  int64_t out_stride, int n_tokens, int n_heads,
                                  const rabbit_cuda_kv4_batch *b, float scale, int window,
                                  void *stream) {
    if (!kv || !ws || !b || layer < 0 || layer >= kv->n_layers || !dtype_size(dtype) ||
        n_tokens < 0 || n_heads < 1 || n_heads > 65535 || n_heads % kv->view.nkv ||
        (int64_t)n_tokens * n_heads > 0x7fffffff || window < 0 || !isfinite(scale))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "kv4_attention: NULL cache, scratch or batch, a bad layer, dtype, count, scale or "
                    "window, or n_heads not a multiple of n_kv_heads");
    if (b->n_seqs < 0 || b->n_seqs > 65535 || b->max_pages < 0 || b->max_q_len < 0)
        return fail(RABBIT_CUDA_ERR_ARGS, "kv4_attention: a bad count in the batch");
    if (ws->device != kv->device || ws->ng != kv->view.ng)
        return fail(RABBIT_CUDA_ERR_ARGS, "kv4_attention: the scratch is of another cache");
    if (n_tokens == 0 || b->n_seqs == 0) return ok();
    if (!b->d_q_start && b->n_seqs > n_tokens)
        return fail(RABBIT_CUDA_ERR_ARGS, "kv4_attention: %d sequences of one row, %d rows", b->n_seqs,
                    n_tokens);
    const int size = dtype_size(dtype);
    Kv4AttnArgs a;
    a.c = kv->layer(layer);
    const int64_t row = (int64_t)n_heads * a.c.hd;
    a.qs = q_stride ? q_stride : row;
    a.os = out_stride ? out_stride : row;
    if (!d_q || !d_out || !b->d_kv_len || (!b->d_page_table && b->max_pages) || a.qs < row ||
        a.os < row || (reinterpret_cast<uintptr_t>(d_q) & (size - 1)) ||
        (reinterpret_cast<uintptr_t>(d_out) & (size - 1)) ||
        ((reinterpret_cast<uintptr_t>(b->d_q_start) | reinterpret_cast<uintptr_t>(b->d_kv_len) |
          reinterpret_cast<uintptr_t>(b->d_page_table)) & 3) || (d_q == d_out && a.qs != a.os))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "kv4_attention: NULL pointer, a stride below n_heads * head_dim (or different in "
                    "place), or a pointer not aligned to its element");
    a.q = d_q;
    a.out = d_out;
    a.q_start = b->d_q_start;
    a.kv_len = b->d_kv_len;
    a.table = b->d_page_table;
    a.n_seqs = b->n_seqs;
    a.max_pages = b->max_pages;
    a.max_q = b->max_q_len ? b->max_q_len : 1;
    if (a.max_q > n_tokens) a.max_q = n_tokens;
    a.T = n_tokens;
    a.nh = n_heads;
    a.window = window;
    a.dtype = dtype;
    a.scale = (scale != 0.f ? scale : 1.0f / sqrtf((float)a.c.hd)) * 1.44269504088896340736f;
    a.vec = ((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_out)) & 15) == 0 &&
            a.qs * size % 16 == 0 && a.os * size % 16 == 0;
    a.part = ws->part;
    a.count = ws->count;
    a.wait_ns = wait_limit_ns();
    a.withhold = kv->withhold;
    kv->withhold = false;
    DeviceScope scope(kv->device);
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    scope.launch(dtype == RABBIT_CUDA_F32 ? launch_attention<true>(a, kv, s) : launch_attention<false>(a, kv, s),
                 "kv4_attention");
    return scope.done();
}

int rabbit_cuda_kv4_debug_withhold(rabbit_cuda_kv4 *kv) {
    if (!kv) return fail(RABBIT_CUDA_ERR_ARGS, "kv4_debug_withhold: NULL cache");
    kv->withhold = true;
    return ok();
}

}  // extern "C"
