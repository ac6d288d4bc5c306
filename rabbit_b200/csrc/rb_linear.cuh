// rb_linear.cuh -- products y = x W^T with e4m3 or 16-bit operands on the
// sm_100a tensor cores: the kernel behind rabbit_cuda_linear_dev and
// rabbit_cuda_linear_grouped_dev.
//
// The weights are the MMA's A operand, the tokens its B operand: a tile takes as many
// tokens as its expert has for it, so ragged groups and single tokens do not pay
// for 128 rows, and a CTA's 128 weight rows are in one row of 128 x 128 scale
// blocks. Gated, the 128 rows are 64 of the gate and the same 64 of the up matrix.
//
// Roles of a CTA's 16 warps, over the same sequence of tiles and of steps of 128 bytes of K:
//   warp 0       TMA: the step's weight rows and, without a list, token rows into a ring of
//                stages (128-byte rows, 128-byte swizzle);
//   warp 1       tensor memory; one thread issues the step's MMAs and commits;
//   warps 2, 3   (e4m3) the step's scales, sw * sx for each token, into shared memory; (16-bit)
//                one thread's fence between the proxies for gathered rows;
//   warps 4..11  readout: warp w reads lanes 32 (w % 4) .. + 31 (weight rows), and the
//                even or odd blocks of 16 tokens; outputs go through shared memory, so that
//                they leave in rows of 16 bytes a thread;
//   warps 12..15 with a list and tiles of more than 32 tokens: the token rows by cp.async, 16
//                bytes a thread. (A gather by TMA takes 80 cycles for four rows of 128 bytes: too
//                long for many; of few rows it spares the MMAs' thread the fence between the
//                proxies, some 0.3 us a step.)
// Accumulation (MODE):
//   kLinWhole  16-bit: in tensor memory over all of K, read once;
//   kLinParts  16-bit, for fp32 outputs or a long K: the tensor cores' sum is cut off,
//              not rounded, at each MMA, an error that grows with their number (K 2048 and 14336:
//              2.3e-6 and 1.8e-5 of random terms' sum, 1.2e-5 and 9.3e-5 of terms' of one sign); so each 256
//              channels are read out and added in 32-bit registers (4e-7, 1.2e-6);
//   kLinF8     e4m3: each step is a scale block, read out and added to 32-bit registers as
//              acc += (sw sx) * product, while the MMAs of the next steps fill other buffers
//              of tensor memory (512 columns / the tile's, at least two).
// PAIR: two CTAs share a tile of 256 weight rows: each has its rows of A and half the
// tokens' rows of B, and CTA 0 issues one MMA of M = 256 for both (cta_group::2), so a step
// brings 32 KB instead of 48 KB to each SM for the same work.
// Otherwise, short products (few tiles) are split over K by a cluster of `split` CTAs: each
// leaves its part in its own shared memory and sums a share of the outputs over the cluster in
// the order of the ranks, so there is no workspace and the same bits come each time.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "rb_device.cuh"
#include "rb_runtime.h"
#include "rb_tcgen05.cuh"
#include "rb_types.cuh"

namespace rb {

enum { kLinWhole, kLinParts, kLinF8 };

constexpr int kLinThreads = 512;
constexpr int kLinReaders = 256;          // threads of the readout warps
constexpr int kLinMaxExperts = 1024;
constexpr int kLinBufs = 8;               // buffers of tensor memory, at most
constexpr int kLinStages = 12;            // stages of the ring, at most
constexpr int kLinPart = 4;               // steps of a part (kLinParts)
constexpr uint32_t kLinTile = 128 * 128;  // bytes of a step's 128 weight rows
constexpr uint32_t kLinOut = 32 * 128 * 4;  // outputs on their way: 32 tokens

// Error bits of an object's error word.
#define RB_LIN_ERR_OFFSETS 16
#define RB_LIN_ERR_ROWS 32
#define RB_LIN_ERR_WAIT 256
#define RB_LIN_ERR_OPEN 512  // after it, what was under way did not end either

struct LinArgs {
    const int *offsets;   // [E + 1], or NULL: one expert with all rows
    const int *rows;      // [R] rows of x, or NULL
    bool gather;          // by warps 12..15; with a list and without: by TMA
    const uint8_t *x;     // to gather: x, its row in bytes, and the bytes of n_in
    uint32_t x_bytes;
    int k_bytes;
    const float *xs, *ws; // e4m3: scales
    uint32_t xs_stride;
    void *y;
    int64_t y_stride;
    bool vec, pairs;      // y's rows take pieces of 16 bytes, of two elements
    int gated;
    int N, E, R, x_rows;
    int steps;            // of 128 bytes, over K
    int mt;               // tiles of outputs
    int bn;               // tokens of a tile, at most: 16 or a multiple of 32
    int unit;             // tokens of a tile come in multiples of it
    int box;              // token rows of a box
    int stages;
    int bufs, buf_shift;  // buffers: 2^buf_shift
    int split;            // CTAs of a cluster that splits K
    int band;             // token tiles that go together, for the L2
    uint32_t format;      // operand format of the instruction descriptor
    int *err;
    uint64_t wait_ns;
    int withhold;         // test hook: the copies end before a tile's last step; a bit for each CTA of a pair
};

// Shared memory: the ring (aligned to 1024), the outputs on their way, then LinShared,
// the scales [bufs][1 or 2][bn, at least 32], off [E + 1] and pre [E + 1].
struct LinShared {
    uint64_t full[kLinStages], empty[kLinStages];
    uint64_t rows[kLinStages];  // to gather: this CTA's token rows have arrived
    uint64_t told[kLinStages];  // and the MMAs may read them (and the other CTA's), in the leader
    uint64_t dfull[kLinBufs], dempty[kLinBufs], mfree[kLinBufs];
    uint64_t mdone;
    uint32_t tmem;
    int abort;
    // for lin_settle: steps copied, the bytes of each stage's last by this CTA; steps and buffers
    // committed, whether on mdone, too
    int issued, stepped, filled, ended;
    uint32_t bytes[kLinStages];
    int4 src[8];  // a list's rows of x, gathered by TMA
    uint32_t written[2][8];  // of the tile, and of the one before: a bit for each token to write
};
static_assert(sizeof(LinShared) % 16 == 0, "the scales behind it are read 16 bytes at a time");
__host__ __device__ constexpr int lin_sc(int bn) { return bn < 32 ? 32 : bn; }
__host__ __device__ constexpr uint32_t lin_stage_bytes(bool pair, int bn) {
    return kLinTile + (uint32_t)bn * (pair ? 64 : 128);
}
// All but the ring.
__host__ __device__ constexpr size_t lin_fixed(bool f8, int gated, int bn, int bufs, int E) {
    return 1024 + kLinOut + sizeof(LinShared) +
           (f8 ? (size_t)bufs * (1 + gated) * lin_sc(bn) * 4 : 0) + 8 * (size_t)(E + 1);
}

struct LinTile {
    int e, mt, row0, n, cols;  // expert, tile of outputs, first row of y, tokens, in units
};

// Tile `i` of the launch; false past the last.
__device__ __forceinline__ bool lin_tile(const LinArgs &a, const int *off, const int *pre, int i,
                                         LinTile &t) {
    if (i >= pre[a.E] * a.mt) return false;
    int lo = 0, hi = a.E;  // the expert: pre[lo] * mt <= i < pre[lo + 1] * mt
    while (hi - lo > 1) {
        const int m = (lo + hi) / 2;
        if (pre[m] * a.mt <= i) lo = m;
        else hi = m;
    }
    const int l = i - pre[lo] * a.mt, nt = pre[lo + 1] - pre[lo];
    const int rows = off[lo + 1] - off[lo];
    // bands of token tiles; in a band the outputs' tiles one after the other
    const int b = l / (a.band * a.mt), r = l - b * a.band * a.mt;
    const int w = min(a.band, nt - b * a.band);
    const int mt = r / w, ti = b * a.band + (r - mt * w);
    // equal tiles: at most bn, none empty
    const int per = ((rows + nt - 1) / nt + a.unit - 1) / a.unit * a.unit;
    t.e = lo;
    t.mt = mt;
    t.row0 = off[lo] + ti * per;
    t.n = min(per, rows - ti * per);
    t.cols = (t.n + a.unit - 1) / a.unit * a.unit;
    return true;
}

template <int N>
struct LinInt {
    static constexpr int value = N;
};

// A place in a ring and the parity of its use.
struct LinRing {
    int at = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int n) {
        if (++at == n) {
            at = 0;
            phase ^= 1;
        }
    }
};

// An arrival in either CTA of a pair, and mbar_try_wait for such, of the cluster's scope. What changes hands is
// tensor memory, which the tcgen05 fences on both sides order, or rows in shared memory, for which the two fences
// below are: before the arrival and behind the wait. So both are relaxed. (With a release and an acquire of all memory
// a step of 0.44 us took 0.8 and 8192 tokens of 8 f16 experts 5.8 ms instead of 3.4: they wait for the
// thread's accesses under way.)
__device__ __forceinline__ void cluster_bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Fences of the cluster's scope for shared memory alone: this CTA's before an arrival, either's behind a wait.
__device__ __forceinline__ void cluster_release_shared() {
    asm volatile("fence.release.sync_restrict::shared::cta.cluster;" ::: "memory");
}
__device__ __forceinline__ void cluster_acquire_shared() {
    asm volatile("fence.acquire.sync_restrict::shared::cluster.cluster;" ::: "memory");
}
__device__ __forceinline__ bool cluster_try_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
        : "memory");
    return ok != 0;
}

// Bounded wait of one thread. OTHER: on a barrier at which the pair's other CTA arrives (cluster_bar_arrive).
template <bool OTHER = false>
__device__ __forceinline__ bool lin_wait1(uint64_t *bar, uint32_t parity, const LinArgs &a,
                                          volatile int *abort) {
    auto passed = [&] { return OTHER ? cluster_try_wait(bar, parity) : mbar_try_wait(bar, parity); };
    if (passed()) return true;
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t it = 1;; ++it) {
        if (passed()) return true;
        if ((it & 15u) == 0) {
            if (*abort) return false;
            if (globaltimer_ns() - t0 > a.wait_ns) {
                atomicOr(a.err, RB_LIN_ERR_WAIT);
                *abort = 1;
                return false;
            }
        }
    }
}
// Of a warp: it goes one way.
__device__ __forceinline__ bool lin_wait(uint64_t *bar, uint32_t parity, const LinArgs &a,
                                         volatile int *abort) {
    return __all_sync(0xffffffffu, lin_wait1(bar, parity, a, abort));
}

__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}
// Address in the cluster's window of `p` (this CTA's shared memory) in CTA `rank`.
__device__ __forceinline__ uint32_t cluster_addr(const void *p, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Two fp32 numbers in a register pair; acc += v * f and acc += v on both.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void unpack2(uint64_t p, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ void fma2(uint64_t &acc, uint64_t v, uint64_t f) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(v), "l"(f));
}
__device__ __forceinline__ void add2(uint64_t &acc, uint64_t v) {
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc) : "l"(v));
}
__device__ __forceinline__ int cluster_ld1(uint32_t at) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
// Counts `bytes` of a barrier's phase as arrived.
__device__ __forceinline__ void mbar_complete_tx(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ float4 cluster_ld4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(at)
                 : "memory");
    return v;
}
// Writes of the generic proxy (cp.async) that this thread waited for are seen by the
// asynchronous one (the MMAs issued after).
__device__ __forceinline__ void fence_async() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// 16 bytes (n of them read, the rest zero) into shared memory.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// 16 consecutive columns of this thread's lane, and the wait before their first use.
__device__ __forceinline__ void lin_ld16(uint32_t taddr, float (&v)[16]) {
    tmem_ld16(taddr, reinterpret_cast<int(&)[16]>(v), 0);
}
__device__ __forceinline__ void lin_ld_done(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]),
                   "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]),
                   "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}

// g / (1 + exp(-g)) with h = exp(-|g| / 2): g / (1 + h h) above zero and g h h / (1 + h h) below, where
// exp(-g) would leave fp32 from -88.7 on, and its quotient before that, while g exp(g) is a normal number down to
// -91.8. The divisor lies in 1 .. 2, where the fast division is off by two steps of 2^-23 at most.
// OUT of 32 bits: h to one step, 2^-20 in all. (With the exact division on top, 4099 tokens of 64 e4m3 experts
// took 465 us.) OUT of 16 bits: h = 2^(|g| c), c = -1 / (2 ln 2), by the instruction for powers of two (2^-22)
// of a product that is off by 3/4 |g| 2^-24: (10 + |g|) 2^-23 in all, 2^-16 at -92 where half a step of the
// output is 2^-12 or more.
template <typename OUT>
__device__ __forceinline__ float lin_silu(float g) {
    float h;
    if constexpr (sizeof(OUT) == 4) h = expf(-0.5f * fabsf(g));
    else asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(fabsf(g) * -0.72134752f));
    return __fdividef(g < 0.f ? g * h * h : g, fmaf(h, h, 1.f));
}

// Two outputs of a row from column c on.
template <typename T>
__device__ __forceinline__ void lin_put2(const LinArgs &a, int64_t row, int c, float v0, float v1) {
    T *y = static_cast<T *>(a.y) + row * a.y_stride + c;
    if (a.pairs && c + 2 <= a.N) {
        struct alignas(2 * sizeof(T)) Two {
            T a, b;
        };
        *reinterpret_cast<Two *>(y) = Two{from_f32<T>(v0), from_f32<T>(v1)};
    } else {
        if (c < a.N) y[0] = from_f32<T>(v0);
        if (c + 1 < a.N) y[1] = from_f32<T>(v1);
    }
}
// Piece `seg` of 8 of a token's row of 128 sums, which `get(i)` reads four at a time, to
// row `row` of y, whose columns from `n0` on they are. FAR: reads that take long.
template <bool GATED, bool FAR, typename T, typename F>
__device__ __forceinline__ void lin_put(const LinArgs &a, int64_t row, int n0, int seg, F &&get) {
#pragma unroll
    for (int p = 0; p < (GATED ? 1 : 2); ++p) {
        if (!a.vec) break;
        const int c = (p * 8 + seg) * 8;
        const float4 l = get(c), h = get(c + 4);
        float v[8] = {l.x, l.y, l.z, l.w, h.x, h.y, h.z, h.w};
        if constexpr (GATED) {
            const float4 ul = get(64 + c), uh = get(64 + c + 4);
            const float u[8] = {ul.x, ul.y, ul.z, ul.w, uh.x, uh.y, uh.z, uh.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = lin_silu<T>(v[i]) * u[i];
        }
        T *y = static_cast<T *>(a.y) + row * a.y_stride + n0 + c;
        if (n0 + c + 8 <= a.N) {
            store8<true>(y, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (n0 + c + i < a.N) y[i] = from_f32<T>(v[i]);
        }
    }
    if (a.vec) return;
    // rows that do not lie on 16 bytes: four columns at a time, the eight threads' side by side
#pragma unroll FAR ? 4 : 1
    for (int c = 4 * seg; c < (GATED ? 64 : 128); c += 32) {
        float4 f = get(c);
        if constexpr (GATED) {
            const float4 u = get(64 + c);
            f = make_float4(lin_silu<T>(f.x) * u.x, lin_silu<T>(f.y) * u.y, lin_silu<T>(f.z) * u.z,
                            lin_silu<T>(f.w) * u.w);
        }
        lin_put2<T>(a, row, n0 + c, f.x, f.y);
        lin_put2<T>(a, row, n0 + c + 2, f.z, f.w);
    }
}
// Whether token c of a tile is written.
__device__ __forceinline__ bool lin_written(const LinArgs &a, const LinTile &t, int c) {
    if (c >= t.n) return false;
    if (!a.rows) return true;
    const int r = __ldg(a.rows + t.row0 + c);
    return r >= 0 && r < a.x_rows;
}

// off and pre from the offsets, by the whole block (a barrier has to follow). With offsets out
// of order or range the call has no tile at all: tiles of ranges that overlap could be more than
// the launch was made for.
__device__ __forceinline__ void lin_experts(const LinArgs &a, int *off, int *pre, int per) {
    bool bad = false;
    for (int e = threadIdx.x; e <= a.E; e += kLinThreads) {
        const int o = a.offsets ? a.offsets[e] : e ? a.R : 0;
        off[e] = o;
        bad |= o < 0 || o > a.R || (a.offsets && e && a.offsets[e - 1] > o);
    }
    bad = __syncthreads_or(bad);
    if (bad && threadIdx.x == 0) atomicOr(a.err, RB_LIN_ERR_OFFSETS);
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    int before = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
        const int e = e0 + lane;
        int n = e < a.E && !bad ? (off[e + 1] - off[e] + per - 1) / per : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int m = __shfl_up_sync(0xffffffffu, n, d);
            if (lane >= d) n += m;
        }
        if (e < a.E) pre[e + 1] = before + n;
        before += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) pre[0] = 0;
}

// The ring's last `issued` uses have been given back. The commits that do it arrive in both CTAs
// of a pair, whenever the products are through; until each has arrived neither CTA may end,
// or the arrival would go to the shared memory of another block. (The products' own commits have
// all been waited for by the readout.)
__device__ __forceinline__ bool lin_emptied(const LinArgs &a, LinShared &s, int issued, volatile int *abort) {
    for (int j = max(0, issued - a.stages); j < issued; ++j)
        if (!lin_wait1(&s.empty[j % a.stages], (j / a.stages) & 1, a, abort)) return false;
    return true;
}

// At the end of a block in which a wait ran out, after the (pair's) last barrier but one: what is
// under way ends before the tensor memory is given back and the block ends. Thread 0: the products (mdone),
// what they were committed to in this CTA (`bufs` buffers, where nobody else arrives on those
// barriers: there mdone is all), and the copies of both CTAs, which complete on the leader's barriers. A pair's CTAs
// may have got to different steps, at most the ring's stages apart; a barrier's count is made up by
// what the one behind did not copy, or did not expect. In a CTA without a wait that ran out all of
// this has been waited for; then nothing of the other's arrives there, either.
template <bool PAIR>
__device__ __forceinline__ void lin_settle(const LinArgs &a, LinShared &s, int bufs) {
    if (threadIdx.x == 0) {
        const bool leader = !PAIR || cluster_rank() == 0;
        auto of = [&](const int *p, uint32_t r) {  // a number of CTA r
            return PAIR ? cluster_ld1(cluster_addr(p, r)) : *p;
        };
        bool closed = true;
        auto wait = [&](uint64_t *bar, int n, int size) {  // for the last uses of a ring of n so far
            for (int j = max(0, n - size); j < n; ++j)
                closed &= mbar_wait(&bar[j % size], (j / size) & 1, a.wait_ns, nullptr, 0);
        };
        if (of(&s.ended, 0)) wait(&s.mdone, 1, 1);
        wait(s.empty, of(&s.stepped, 0), a.stages);
        if (bufs) wait(s.dfull, of(&s.filled, 0), bufs);
        if (leader) {
            const int n0 = s.issued, n1 = of(&s.issued, 1);
            for (int j = n0; j < n1; ++j)  // only the other CTA's
                mbar_arrive_expect_tx(&s.full[j % a.stages], of(reinterpret_cast<const int *>(&s.bytes[j % a.stages]), 1));
            for (int j = n1; j < n0; ++j)  // expected, and not copied
                mbar_complete_tx(&s.full[j % a.stages], s.bytes[j % a.stages]);
            wait(s.full, max(n0, n1), a.stages);
        }
        if (!closed) atomicOr(a.err, RB_LIN_ERR_OPEN);
    }
    __syncthreads();
}

// The gathering warps' part of a tile: tokens c0 .. c0 + here - 1 of it into rows 0.. of the
// token rows `at` bytes into each stage, ROWS of them a thread (part, part + 16, ..).
template <int ROWS>
__device__ __forceinline__ bool lin_gather(const LinArgs &a, LinShared &s, uint32_t at, uint32_t stage_bytes,
                                           const LinTile &t, int c0, int here, int k0, int k1,
                                           LinRing &st, volatile int *abort) {
    const int tid = threadIdx.x - 384, piece = tid & 7, part = tid >> 3;
    const uint32_t to = at + part * 128 + ((piece ^ (part & 7)) << 4);
    int r[ROWS];  // of x; -1: none, zeros
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int c = c0 + part + 16 * j;
        r[j] = -1;
        if (part + 16 * j < here && c < t.n) {
            r[j] = __ldg(a.rows + t.row0 + c);
            if (r[j] < 0 || r[j] >= a.x_rows) {
                atomicOr(a.err, RB_LIN_ERR_ROWS);
                r[j] = -1;
            }
        }
    }
    for (int k = k0; k < k1; ++k) {
        if (!lin_wait(&s.empty[st.at], st.phase ^ 1, a, abort)) return false;
        const uint32_t dst = to + st.at * stage_bytes;
        const int b = k * 128 + piece * 16, n = min(max(a.k_bytes - b, 0), 16);
        const uint8_t *x = a.x + (n > 0 ? b : 0);
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (16 * j < here)
                cp_async16(dst + j * 2048, x + (int64_t)max(r[j], 0) * a.x_bytes, r[j] >= 0 ? n : 0);
        // (the fence that lets the tensor cores see them is the waiting thread's: here it
        // would wait for every copy under way)
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&s.rows[st.at])) : "memory");
        st.next(a.stages);
    }
    return true;
}

// One thread, of each CTA of a pair: once this CTA's rows of a step are there, the fence
// between the proxies, and word to the thread that issues the MMAs (of CTA 0). In that thread
// itself the fence held up the MMAs: 8192 tokens of 8 f16 experts took 0.3 ms more.
template <bool PAIR>
__device__ __forceinline__ void lin_tell(const LinArgs &a, LinShared &s, const int *off, const int *pre,
                                         int first, int stride, int k0, int k1, volatile int *abort) {
    LinTile t;
    LinRing st;
    for (int i = first; lin_tile(a, off, pre, i, t); i += stride)
        for (int k = k0; k < k1; ++k) {
            if (!lin_wait1(&s.rows[st.at], st.phase, a, abort)) return;
            fence_async();
            if (PAIR) {
                cluster_release_shared();
                cluster_bar_arrive(cluster_addr(&s.told[st.at], 0));
            } else {
                mbar_arrive(&s.told[st.at]);
            }
            st.next(a.stages);
        }
}

template <int MODE, bool PAIR, bool GATED, typename OUT>
__global__ void __launch_bounds__(kLinThreads, 1)
    k_linear(const __grid_constant__ LinArgs a, const __grid_constant__ CUtensorMap mw,
             const __grid_constant__ CUtensorMap mx) {
    extern __shared__ uint8_t lin_raw[];
    constexpr bool F8 = MODE == kLinF8;
    static_assert(!F8 || !PAIR, "k_linear_rows has these");
    constexpr int PART = MODE == kLinF8 ? 1 : MODE == kLinParts ? kLinPart : 1 << 30;
    uint8_t *ring = lin_raw + ((1024u - (smem_u32(lin_raw) & 1023u)) & 1023u);
    const uint32_t stage_bytes = lin_stage_bytes(PAIR, a.bn);
    float *outs = reinterpret_cast<float *>(ring + (size_t)a.stages * stage_bytes);
    LinShared &s = *reinterpret_cast<LinShared *>(reinterpret_cast<uint8_t *>(outs) + kLinOut);
    float *scales = reinterpret_cast<float *>(&s + 1);
    const int sc_row = lin_sc(a.bn), sc_buf = (1 + GATED) * sc_row;
    int *off = reinterpret_cast<int *>(scales + (F8 ? a.bufs * sc_buf : 0)), *pre = off + a.E + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort = &s.abort;
    const uint32_t rank = PAIR || a.split > 1 ? cluster_rank() : 0;
    const bool leader = !PAIR || rank == 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
            mbar_init(&s.rows[i], 128);
            mbar_init(&s.told[i], PAIR ? 2 : 1);
        }
        for (int i = 0; i < a.bufs; ++i) {
            mbar_init(&s.dfull[i], F8 ? 3 : 1);  // the MMAs, and the scales' two warps
            mbar_init(&s.dempty[i], 8);          // this CTA's readout
            mbar_init(&s.mfree[i], 16);          // the pair's
        }
        mbar_init(&s.mdone, 1);
        s.abort = 0;
        s.issued = s.stepped = s.filled = s.ended = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        if (PAIR) tmem_alloc_pair(&s.tmem, 512);
        else tmem_alloc(&s.tmem, 512);
    }
    launch_dependents();
    wait_prerequisite();
    lin_experts(a, off, pre, a.bn);
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();  // both CTAs' barriers are ready
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    // a pair has every (CTAs / 2)-th tile, a CTA by itself each gridDim.x-th, a cluster that
    // splits K one
    const int team = PAIR ? 2 : a.split;
    const int first = blockIdx.x / team, stride = !PAIR && a.split > 1 ? 1 << 30 : gridDim.x / team;
    const int k0 = PAIR ? 0 : (int)((int64_t)a.steps * rank / a.split);
    const int k1 = PAIR ? a.steps : (int)((int64_t)a.steps * (rank + 1) / a.split);
    const int outputs = GATED ? 64 : 128;  // of a CTA's tile
    LinTile t;

    // Registers: 512 x 128 at the launch (linear_create checks it); 128 x 72 + 128 x 56 +
    // 256 x 192 from here.
    if (warp < 4) {
        if constexpr (MODE != kLinWhole) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {  // ------------------------------------------------ TMA
        const uint64_t keep = policy_evict_last(), once = policy_evict_first();
        LinRing st;
        int issued = 0;
        bool ok = true;
        const bool chosen = elect_one();
        const int held = a.withhold >> (PAIR ? rank : 0) & 1;
        for (int i = first; ok && lin_tile(a, off, pre, i, t); i += a.withhold ? 1 << 30 : stride) {
            const int n0 = (PAIR ? 2 * t.mt + rank : t.mt) * outputs;
            const int here = PAIR ? t.cols / 2 : t.cols;  // token rows of this CTA
            const int boxes = a.rows ? 0 : (here + a.box - 1) / a.box;
            const int quads = !PAIR && a.rows && !a.gather ? t.cols / 4 : 0;
            const uint32_t bytes = (PAIR ? 2 : 1) * (kLinTile + boxes * a.box * 128) + quads * 512;
            if (lane < 4 * quads) {
                int r = lane < t.n ? __ldg(a.rows + t.row0 + lane) : 0;
                if (r < 0 || r >= a.x_rows) {
                    atomicOr(a.err, RB_LIN_ERR_ROWS);
                    r = 0;  // read for nothing: lin_written leaves the row out
                }
                reinterpret_cast<int *>(s.src)[lane] = r;
            }
            __syncwarp();
            // weights that no other tile of tokens reads leave the L2 first
            const uint64_t pol = pre[t.e + 1] - pre[t.e] > 1 ? keep : once;
            if (chosen) {
                for (int k = k0; k < k1 - held; ++k, ++issued) {
                    if (!(ok = lin_wait1(&s.empty[st.at], st.phase ^ 1, a, abort))) break;
                    uint8_t *base = ring + (size_t)st.at * stage_bytes, *xb = base + kLinTile;
                    const int c0 = k * (F8 ? 128 : 64);
                    s.bytes[st.at] = PAIR ? bytes / 2 : bytes;
                    if (leader) mbar_arrive_expect_tx(&s.full[st.at], bytes);
                    if constexpr (PAIR) {
                        const uint32_t bar = cluster_addr(&s.full[st.at], 0);
                        tma_load_4d_pair(base, &mw, c0, n0, 0, t.e, bar, pol);
                        if (GATED) tma_load_4d_pair(base + kLinTile / 2, &mw, c0, n0, 1, t.e, bar, pol);
                        for (int b = 0; b < boxes; ++b)
                            tma_load_2d_pair(xb + b * a.box * 128, &mx, c0, t.row0 + rank * here + b * a.box, bar);
                    } else {
                        tma_load_4d(base, &mw, c0, n0, 0, t.e, &s.full[st.at], pol);
                        if (GATED) tma_load_4d(base + kLinTile / 2, &mw, c0, n0, 1, t.e, &s.full[st.at], pol);
                        for (int b = 0; b < boxes; ++b)
                            tma_load_2d(xb + b * a.box * 128, &mx, c0, t.row0 + b * a.box, &s.full[st.at]);
                        for (int j = 0; j < quads; ++j) {
                            const int4 r = s.src[j];
                            tma_gather4(xb + j * 512, &mx, c0, r.x, r.y, r.z, r.w, &s.full[st.at]);
                        }
                    }
                    st.next(a.stages);
                }
            }
            ok = __all_sync(0xffffffffu, ok);
        }
        if (chosen) {
            if (ok) lin_emptied(a, s, issued, abort);
            s.issued = issued;
        }
        __syncwarp();
    } else if (warp == 1) {  // ------------------------------------------ MMA
        if (leader && elect_one()) {
            LinRing st, db;
            bool ok = true;
            int stepped = 0, filled = 0;
            const uint64_t wd0 = swizzled_desc(smem_u32(ring)), xd0 = swizzled_desc(smem_u32(ring + kLinTile));
            for (int i = first; ok && lin_tile(a, off, pre, i, t); i += stride) {
                const uint32_t idesc = float_idesc(a.format, PAIR ? 256 : 128, t.cols);
                int part = 0;
                for (int k = k0; k < k1; ++k) {
                    if (!(ok = lin_wait1<PAIR>(&s.full[st.at], st.phase, a, abort))) break;
                    if (a.gather) {
                        if (!(ok = lin_wait1<PAIR>(F8 ? &s.rows[st.at] : &s.told[st.at], st.phase, a, abort))) break;
                        if (F8) fence_async();  // (no warp is free to do it)
                    }
                    if (PAIR) cluster_acquire_shared();
                    const uint64_t step = (uint64_t)(st.at * stage_bytes) >> 4;
                    if (part == 0)
                        if (!(ok = lin_wait1<PAIR>(PAIR ? &s.mfree[db.at] : &s.dempty[db.at], db.phase ^ 1, a, abort))) break;
                    tc_fence_after();
                    const uint32_t d = tmem + db.at * a.bn;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_float_ss<F8, PAIR>(d, wd0 + step + 2 * j, xd0 + step + 2 * j, idesc, j > 0 || part > 0);
                    if (PAIR) mma_commit_pair(&s.empty[st.at]);
                    else mma_commit(&s.empty[st.at]);
                    ++stepped;
                    st.next(a.stages);
                    if (++part == PART || k == k1 - 1) {
                        if (PAIR) mma_commit_pair(&s.dfull[db.at]);
                        else mma_commit(&s.dfull[db.at]);
                        ++filled;
                        db.next(a.bufs);
                        part = 0;
                    }
                }
            }
            if (!ok) {  // lin_settle waits for it
                if (PAIR) mma_commit_pair(&s.mdone);
                else mma_commit(&s.mdone);
            }
            s.stepped = stepped;
            s.filled = filled;
            s.ended = !ok;
        }
    } else if (F8) {  // ---------------------------------------------- scales
        const int nb = (a.N + 127) / 128;  // rows of scale blocks of a matrix
        const int64_t up = (int64_t)nb * a.steps;
        bool ok = true;
        // Of a tile of more than 128 tokens, one warp has the first 128 and the other the rest of
        // each buffer; else each has every other one, whole.
        uint32_t count = 0;  // buffers before the tile
        // NT tokens a lane, the scales of the next AHEAD steps on their way (a step of a few
        // tokens takes 0.4 us, as long as half a read from HBM)
        auto tile = [&](auto nt, auto ahead) {
            constexpr int NT = decltype(nt)::value, AHEAD = decltype(ahead)::value;
            const bool both = t.cols > 128;
            const int mine = both ? 0 : (warp - 2) ^ (count & 1);  // the tile's first buffer that is
            const int c1 = lane + (both ? (warp - 2) * 128 : 0), by = both ? 1 : 2;
            int r[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int c = c1 + 32 * j;
                r[j] = t.row0 + c;
                if (c < t.n && a.rows) {
                    r[j] = __ldg(a.rows + r[j]);
                    if (r[j] >= a.x_rows) r[j] = -1;
                }
                if (c >= t.n) r[j] = -1;
            }
            const int n0 = t.mt * outputs;
            const float *ws = a.ws + ((int64_t)t.e * (1 + GATED) * nb + min(n0 / 128, nb - 1)) * a.steps;
            float v[AHEAD][NT], w[AHEAD][2];
            auto fetch = [&](int k, int h) {
                if (k >= k1) return;
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    v[h][j] = r[j] >= 0 ? __ldg(a.xs + (uint64_t)r[j] * a.xs_stride + k) : 0.f;
                w[h][0] = __ldg(ws + k);
                w[h][1] = GATED ? __ldg(ws + up + k) : 0.f;
            };
            const int ks = k0 + mine;
            uint32_t use = count + mine;  // of the buffers, in order
            count += k1 - k0;
#pragma unroll
            for (int h = 0; h < AHEAD; ++h) fetch(ks + h * by, h);
            int k = ks;
            while (ok && k < k1) {
#pragma unroll
                for (int h = 0; h < AHEAD; ++h) {
                    if (k >= k1) break;
                    const int at = use & (a.bufs - 1);
                    if (!(ok = lin_wait(&s.dempty[at], (use >> a.buf_shift & 1) ^ 1, a, abort))) break;
                    float *sc = scales + at * sc_buf;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        if (c1 + 32 * j < sc_row) {
                            sc[c1 + 32 * j] = v[h][j] * w[h][0];
                            if (GATED) sc[sc_row + c1 + 32 * j] = v[h][j] * w[h][1];
                        }
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cnt(&s.dfull[at], both ? 1 : 2);
                    use += by;
                    fetch(k + AHEAD * by, h);
                    k += by;
                }
            }
        };
        for (int i = first; ok && lin_tile(a, off, pre, i, t); i += stride) {
            if (t.cols <= 32) tile(LinInt<1>(), LinInt<GATED ? 5 : 8>());
            else tile(LinInt<4>(), LinInt<2>());
        }
    } else if (!F8 && warp == 2 && a.gather) {  // ------- word of gathered rows
        if (elect_one()) lin_tell<PAIR>(a, s, off, pre, first, stride, k0, k1, abort);
        __syncwarp();
    }
    } else if (warp >= 12) {  // ------------------------------------- gather
        if constexpr (MODE != kLinWhole) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (a.gather) {
            LinRing st;
            bool ok = true;
            for (int i = first; ok && lin_tile(a, off, pre, i, t); i += stride) {
                const int here = PAIR ? t.cols / 2 : t.cols;
                ok = lin_gather<PAIR ? 8 : 16>(a, s, smem_u32(ring) + kLinTile, stage_bytes, t,
                                               PAIR ? rank * here : 0, here, k0, k1, st, abort);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {  // ---------------------------------------------------- readout
        if constexpr (MODE != kLinWhole) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int q = warp & 3, h = (warp - 4) >> 2;
        const int nl = q * 32 + lane;  // weight row of the tile
        const int tid = threadIdx.x - 128, seg = tid & 7;
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        float *part = reinterpret_cast<float *>(ring);
        LinRing db;
        bool ok = true;
        uint32_t tile = 0;
        const uint32_t mfree = PAIR ? cluster_addr(&s.mfree[0], 0) : 0;
        auto release = [&]() {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) cluster_bar_arrive(mfree + db.at * 8);
                else mbar_arrive(&s.dempty[db.at]);
            }
            db.next(a.bufs);
        };
        // sums of this warp's 16 tokens of block pair b: to y, or to the cluster's sum
        auto put = [&](int b, const float (&v)[16]) {
            const int c = 32 * b + 16 * h;
            if (!PAIR && a.split > 1) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (c < t.cols) part[(c + j) * 128 + nl] = v[j];
                return;
            }
            named_sync(1, kLinReaders);  // the outputs before have left
#pragma unroll
            for (int j = 0; j < 16; ++j) outs[(16 * h + j) * 128 + nl] = v[j];
            named_sync(1, kLinReaders);
            const int token = tid >> 3;
            if (s.written[tile & 1][b] >> token & 1)
                lin_put<GATED, false, OUT>(a, t.row0 + 32 * b + token, (PAIR ? 2 * t.mt + (int)rank : t.mt) * outputs, seg,
                        [&](int i) { return *reinterpret_cast<const float4 *>(outs + token * 128 + i); });
        };
        // A tile's sums in registers, NC blocks of 16 tokens a warp (with those of 256 tokens in
        // the way, a step of 16 took 0.2 us more)
        auto sums = [&](auto blocks) {
            constexpr int NC = decltype(blocks)::value;
            uint64_t acc[NC][8];  // block pair, two tokens
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[c][j] = 0;
            const int n = t.cols - 16 * h;  // columns from this warp's first on
            for (int k = k0; k < k1; k += PART) {
                if (!(ok = lin_wait(&s.dfull[db.at], db.phase, a, abort))) break;
                tc_fence_after();
                const uint32_t d = tmem + lanes + db.at * a.bn + 16 * h;
                const float *sc = scales + db.at * sc_buf + (GATED && q >= 2 ? sc_row : 0) + 16 * h;
                auto add = [&](int c, const float(&v)[16]) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint64_t v0 = pack2(v[4 * j], v[4 * j + 1]), v1 = pack2(v[4 * j + 2], v[4 * j + 3]);
                        if (F8) {
                            const ulonglong2 f = reinterpret_cast<const ulonglong2 *>(sc + 32 * c)[j];
                            fma2(acc[c][2 * j], v0, f.x);
                            fma2(acc[c][2 * j + 1], v1, f.y);
                        } else {
                            add2(acc[c][2 * j], v0);
                            add2(acc[c][2 * j + 1], v1);
                        }
                    }
                };
                // 32 columns in flight at a time
#pragma unroll
                for (int c = 0; c < NC; c += 2) {
                    float v[2][16];
                    const bool one = 32 * c < n, two = c + 1 < NC && 32 * (c + 1) < n;
                    if (one) lin_ld16(d + 32 * c, v[0]);
                    if (two) lin_ld16(d + 32 * (c + 1), v[1]);
                    if (one) {
                        lin_ld_done(v[0]);
                        add(c, v[0]);
                    }
                    if (two) {
                        lin_ld_done(v[1]);
                        if (c + 1 < NC) add(c + 1, v[1]);
                    }
                }
                release();
            }
            // (a wait that ran out ends it for every warp of the block before a barrier
            // among them)
            ok = named_all(1, kLinReaders, ok);
            if (!ok) return;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if (32 * c >= t.cols) break;
                float v[16];
#pragma unroll
                for (int j = 0; j < 8; ++j) unpack2(acc[c][j], v[2 * j], v[2 * j + 1]);
                put(c, v);
            }
        };
        for (int i = first; ok && lin_tile(a, off, pre, i, t); i += stride) {
            ++tile;
            const uint32_t w = __ballot_sync(0xffffffffu, lin_written(a, t, tid));
            if (lane == 0) s.written[tile & 1][warp - 4] = w;
            if constexpr (MODE != kLinWhole) {
                if (t.cols <= 32) sums(LinInt<1>());
                else if (t.cols <= 64) sums(LinInt<2>());
                else sums(LinInt<8>());
            } else {
                ok = named_all(1, kLinReaders, lin_wait(&s.dfull[db.at], db.phase, a, abort));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + lanes + db.at * a.bn + 16 * h;
                for (int c = 0; 32 * c < t.cols; ++c) {
                    float v[16];
                    lin_ld16(d + 32 * c, v);
                    lin_ld_done(v);
                    put(c, v);
                    __syncwarp();
                }
                release();
            }
        }
    }
    __syncwarp();
    if (!PAIR && a.split > 1) {  // one tile a cluster: its parts summed in the order of the ranks
        cluster_sync_all();
        if (warp >= 4 && warp < 12 && !*abort && lin_tile(a, off, pre, first, t)) {
            const uint32_t part = smem_u32(ring);
            for (int j = threadIdx.x - 128;; j += kLinReaders) {
                const int item = j * a.split + rank, token = item >> 3;
                if (token >= t.n) break;
                if (!lin_written(a, t, token)) continue;
                lin_put<GATED, true, OUT>(a, t.row0 + token, t.mt * outputs, item & 7, [&](int i) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int r = 0; r < a.split; ++r) {
                        uint32_t at;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                                     : "=r"(at) : "r"(part + (uint32_t)(token * 128 + i) * 4), "r"(r));
                        const float4 u = cluster_ld4(at);
                        v.x += u.x;
                        v.y += u.y;
                        v.z += u.z;
                        v.w += u.w;
                    }
                    return v;
                });
            }
        }
        cluster_sync_all();  // nobody leaves while its part is read
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();  // both have read their products
    if (*abort) lin_settle<PAIR>(a, s, F8 ? 0 : a.bufs);
    tc_fence_after();
    if (warp == 1) {
        if (PAIR) tmem_dealloc_pair(tmem, 512);
        else tmem_dealloc(tmem, 512);
    }
    if (PAIR) cluster_sync_all();
}

}  // namespace rb
