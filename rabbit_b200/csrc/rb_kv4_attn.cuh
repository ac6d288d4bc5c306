// rb_kv4_attn.cuh -- what the attention kernels over the 4-bit cache share:
// their arguments, how a batch is cut into equal parts, and the pieces of the
// arithmetic on matrix instructions.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "rb_device.cuh"
#include "rb_kv4.cuh"

namespace rb {

struct Kv4AttnArgs {
    Kv4View c;
    const void *q;
    void *out;
    int64_t qs, os;  // elements between rows
    const int *q_start, *kv_len, *table;
    int n_seqs, max_pages, max_q, T, nh, window, dtype;
    bool vec;        // rows of q and out are 16-byte aligned
    float scale;     // times log2 e: scores are powers of two
    float *part;     // scratch: partial outputs [2 grid][rows][channels], then [2 grid][rows] pairs
    unsigned *count; // scratch: arrivals per CTA that begins a shared item, zero between calls
    uint64_t wait_ns;
    bool withhold;   // test hook: one arrival is left out
};

// A CTA whose wait ran out leaves its work where it is: it makes no further arrival
// (what waits for one runs out as well) and starts no further copy, and lets its copies
// in flight, which write its shared memory, end before it does. They take
// microseconds; this bounds that wait whatever the caller's limit is.
constexpr uint64_t kKv4DrainNs = 2000000000ull;

#ifdef __CUDACC__
// Wait for a phase of a CTA's barrier; false, and reported, after the call's limit.
__device__ __forceinline__ bool kv4_wait(uint64_t *bar, uint32_t parity, const Kv4AttnArgs &a, uint32_t max_sleep_ns = 256) {
    if (mbar_wait(bar, parity, a.wait_ns, nullptr, max_sleep_ns)) return true;
    atomicOr(a.c.err, RB_KV4_ERR_WAIT);
    return false;
}
#endif

constexpr int kKv4MaxLen = 1 << 30;  // positions of a sequence: sums of two stay within an int

// One sequence of a batch. Every entry is checked here before it is used.
struct Kv4Seq {
    int row0, nq;  // query rows; nq 0: none, or a bad range
    int len;       // cached positions
    int g0, n;     // granules that some row sees: [g0, g0 + n)
};

// What is wrong with a sequence's arrays is returned as error bits.
__host__ __device__ inline int kv4_seq(int s0, int s1, int len, int T, int max_q, int64_t room,
                                       int window, Kv4Seq &s) {
    int bad = 0;
    s.row0 = s0;
    s.nq = s1 - s0;
    if (s0 < 0 || s1 < s0 || s1 > T || s1 - s0 > max_q) {
        bad |= RB_KV4_ERR_ROWS;
        s.nq = 0;
    }
    if (len < 0 || len > room || len >= kKv4MaxLen) {
        bad |= RB_KV4_ERR_LEN;
        len = 0;
    }
    s.len = len;
    // the first row, at len - nq, sees furthest back
    const int first = len - s.nq;
    const int lo = window > 0 && first >= window ? first - window + 1 : 0;
    s.g0 = lo / kKv4Granule;
    s.n = len > lo ? (len + kKv4Granule - 1) / kKv4Granule - s.g0 : 0;
    return bad;
}

// Work is counted in units: an item (sequence, row tile, KV head) that sees some
// granule has kKv4Fixed units for what it costs whatever its length (its query
// operands, its merge) and one for each granule. The units of all items in
// order are cut into `parts` runs of equal length, run b of [u(b), u(b + 1)), u(b)
// = floor(b total / parts). A run works on the granules whose units are in it; one
// that ends within an item's fixed units leaves the whole item to the next. Runs
// are at least kKv4MinRun long, more than an item's fixed units, so each has some
// granule's unit.
constexpr int kKv4Fixed = 24, kKv4MinRun = 28;
__host__ __device__ inline int kv4_items(const Kv4Seq &s, int group, int rows, int nkv) {
    return s.nq && s.n > 0 ? nkv * ((s.nq * group + rows - 1) / rows) : 0;
}
__host__ __device__ inline int64_t kv4_cost(const Kv4Seq &s, int group, int rows, int nkv) {
    return (int64_t)kv4_items(s, group, rows, nkv) * (s.n + kKv4Fixed);
}
__host__ __device__ inline int64_t kv4_parts(int64_t total, int grid) {
    const int64_t most = total / kKv4MinRun;
    return most < 1 ? 1 : most < grid ? most : grid;
}
__host__ __device__ inline int64_t kv4_cut(int64_t b, int64_t total, int64_t parts) {
    return b * total / parts;
}
// The run that unit x falls into.
__host__ __device__ inline int kv4_run_of(int64_t x, int64_t total, int64_t parts) {
    return (int)(((x + 1) * parts - 1) / total);
}

// A run's share of one item.
struct Kv4Share {
    int from, take;   // granules [from, from + take) of the item's
    bool begins, ends;
    int64_t start;    // the unit of the item's first granule
};
// A walk over a run's items: `off` units of an item of sequence `s` lie before
// unit `u`. The share of the item in [u, u1), or take 0 where it has none.
__host__ __device__ inline Kv4Share kv4_share(const Kv4Seq &s, int off, int64_t u, int64_t u1) {
    Kv4Share r;
    r.start = u - off + kKv4Fixed;
    const int64_t to = u1 < r.start + s.n ? u1 : r.start + s.n;
    r.from = off > kKv4Fixed ? off - kKv4Fixed : 0;
    r.take = to > r.start + r.from ? (int)(to - r.start) - r.from : 0;
    r.begins = r.from == 0;
    r.ends = r.from + r.take == s.n;
    return r;
}

#ifdef __CUDACC__
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t a0, const uint32_t a1,
                                        const uint32_t a2, const uint32_t a3, const uint32_t b0,
                                        const uint32_t b1, const float c0, const float c1,
                                        const float c2, const float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

__device__ __forceinline__ float exp2_fast(float x) {  // 0 at -inf; within 2^-22
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// (a & m) | o
template <uint32_t M, uint32_t O>
__device__ __forceinline__ uint32_t and_or(uint32_t a) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "n"(M), "n"(O));
    return d;
}

// N bytes (a multiple of 2) at p, aligned to the largest power of two that
// divides N (16 at most), as 32-bit words; an odd last half word's upper half
// is zero.
template <int N>
__device__ __forceinline__ void load_piece(uint32_t (&w)[(N + 3) / 4], const void *p) {
    if constexpr (N % 16 == 0) {
#pragma unroll
        for (int i = 0; i < N / 16; ++i) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = v.x;
            w[4 * i + 1] = v.y;
            w[4 * i + 2] = v.z;
            w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            const uint2 v = reinterpret_cast<const uint2 *>(p)[i];
            w[2 * i] = v.x;
            w[2 * i + 1] = v.y;
        }
    } else if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
    } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
        w[N / 4] = h[N / 2 - 1];
    }
}
// bf16 number `i` of a piece, as fp32.
template <int NW>
__device__ __forceinline__ float piece_bf16(const uint32_t (&w)[NW], int i) {
    return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
}

// Token of a granule's first half that row j of a score tile stands for; the
// same in the second half, 8 later. The order keeps the lanes' loads of K (rows
// 2 i and 2 i + 1) and of V (rows 2 t, then 2 t + 1, of the four t) in different
// banks.
__device__ __forceinline__ int kv4_token(int j) { return j & 1 ? 4 + ((j >> 1) ^ 1) : j >> 1; }

// Signed codes of the lowest nibble of each half word, and of the next one, as
// fp16 pairs: a nibble under the exponent of 1024 is 1024 + u, of the next
// nibble 1024 + 16 u; one addition or multiply-add, exact, leaves u - 8.
__device__ __forceinline__ void signed_codes(uint32_t &e0, uint32_t &e1, uint32_t x) {
    const __half2 bias = __half2half2(__ushort_as_half(0xE408)),   // -1032
        sixteenth = __half2half2(__ushort_as_half(0x2C00)),        // 1 / 16
        bias16 = __half2half2(__ushort_as_half(0xD480));           // -72
    auto half2_of = [](uint32_t v) { return *reinterpret_cast<__half2 *>(&v); };
    auto bits = [](__half2 v) { return *reinterpret_cast<uint32_t *>(&v); };
    e0 = bits(__hadd2(half2_of(and_or<0x000f000fu, 0x64006400u>(x)), bias));
    e1 = bits(__hfma2(half2_of(and_or<0x00f000f0u, 0x64006400u>(x)), sixteenth, bias16));
}

// The value pieces of two tokens (a: even column, b: odd) as fp16 pairs of
// signed codes, channel 4 g + i of group `grp` in e[i]. Signed, where the K side
// may take its bias off by the accumulator's start: sums of values over a long
// context cancel, and with the bias in them would keep 2^-24 of 8 sum w
// instead of 2^-24 of themselves.
template <int NW>
__device__ __forceinline__ void value_codes(uint32_t (&e)[4], const uint32_t (&a)[NW],
                                            const uint32_t (&b)[NW], int grp) {
    const uint32_t x = __byte_perm(a[grp >> 1], b[grp >> 1], grp & 1 ? 0x7632 : 0x5410);
    signed_codes(e[0], e[1], x);
    signed_codes(e[2], e[3], x >> 8);
}

// The transpose of an 8 x 8 matrix of fp16 whose row g, columns 2 t and 2 t + 1
// are lane (g, t)'s pair.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// A key word as fp16 pairs, nibbles (0, 4), (2, 6), (1, 5), (3, 7) of it.
// SIGNED: the codes; else u 2^-24 for the first two and 16 u 2^-24 for the
// others, as they lie.
template <bool SIGNED>
__device__ __forceinline__ void key_codes(uint32_t (&e)[4], uint32_t x) {
    const uint32_t y = x >> 8;
    if constexpr (SIGNED) {
        signed_codes(e[0], e[2], x);
        signed_codes(e[1], e[3], y);
    } else {
        e[0] = x & 0x000f000fu;
        e[1] = y & 0x000f000fu;
        e[2] = x & 0x00f000f0u;
        e[3] = y & 0x00f000f0u;
    }
}
#endif

}  // namespace rb
