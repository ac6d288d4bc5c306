// rb_linear.cuh -- products y = x W^T with e4m3 or 16-bit operands on the
// sm_100a tensor cores: the kernel behind rabbit_cuda_linear_dev and
// rabbit_cuda_linear_grouped_dev.
//
// The weights are the MMA's A operand (128 rows, so a tile of them is one row of
// 128 x 128 scale blocks), the tokens its B operand: a tile takes as many tokens as
// its expert has for it, in steps of 16, so ragged groups and single tokens do not pay for
// 128 rows. A tile of y is 128 outputs x up to `bn` tokens; gated, the
// gate's and the up matrix's 128 rows are two MMAs over the same tokens.
//
// Roles of a CTA's 12 warps, over the same sequence of tiles and of steps of 128 bytes of K:
//   warp 0      TMA: the step's weight rows (one box of each matrix) and token rows
//               (boxes, or gather4 through d_rows) into a ring of stages;
//   warp 1      tensor memory; one lane issues the step's MMAs and commits;
//   warp 2      (e4m3) the step's scales, sw * sx for each token, into shared memory;
//   warps 4..11 readout: warp w reads lanes 32 (w % 4) .. + 31 (outputs), and the even or odd
//               blocks of 16 tokens.
// 16-bit: the accumulator stays in tensor memory over all of K and is read once.
// e4m3: a step is one scale block. Its product is read out and added to 32-bit registers as
// acc += (sw sx) * product, while the MMAs of the next steps fill other buffers of tensor
// memory (512 columns / the tile's width, at least two).
//
// Short products (few tiles) are split over K by a cluster of `split` CTAs: each leaves its
// part in its own shared memory and sums a share of the tokens over the cluster in the order
// of the ranks, so there is no workspace and the same bits come each time.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "rb_device.cuh"
#include "rb_runtime.h"
#include "rb_tcgen05.cuh"
#include "rb_types.cuh"

namespace rb {

constexpr int kLinThreads = 384;
constexpr int kLinMaxExperts = 1024;
constexpr int kLinBufs = 8;      // buffers of tensor memory, at most
constexpr int kLinStages = 12;   // stages of the ring, at most
constexpr uint32_t kLinTile = 128 * 128;  // bytes of 128 weight rows of a step

// Error bits of an object's error word.
#define RB_LIN_ERR_OFFSETS 16
#define RB_LIN_ERR_ROWS 32
#define RB_LIN_ERR_WAIT 256

struct LinArgs {
    const int *offsets;   // [E + 1], or NULL: one expert with all rows
    const int *rows;      // [R] rows of x, or NULL
    const float *xs, *ws; // e4m3: scales
    int64_t xs_stride;
    void *y;
    int64_t y_stride;
    int out_dtype;
    int N, E, R, x_rows;
    int steps;            // of 128 bytes, over K
    int mt;               // tiles of 128 outputs
    int bn;               // tokens of a tile, at most; a multiple of 16
    int box;              // token rows of a box
    int stages;
    int split;            // CTAs of a cluster
    int band;             // token tiles that go together, for the L2
    uint32_t format;      // operand format of the instruction descriptor
    int *err;
    uint64_t wait_ns;
};

struct LinShared {
    uint64_t full[kLinStages], empty[kLinStages];
    uint64_t dfull[kLinBufs], sfull[kLinBufs], dempty[kLinBufs];
    uint64_t mdone;
    uint32_t tmem;
    int abort;
    alignas(16) float sc[kLinBufs][256];  // scales of a step: tokens (gated: gate's, then up's)
    int off[kLinMaxExperts], cnt[kLinMaxExperts];  // first row and rows of each expert
    int pre[kLinMaxExperts + 1];                   // token tiles of the experts before
};

// Bytes of shared memory: the ring (aligned to 1024), then LinShared.
__host__ __device__ constexpr uint32_t lin_stage_bytes(bool gated, int bn) {
    return (gated ? 2 : 1) * kLinTile + (uint32_t)bn * 128;
}
__host__ __device__ constexpr size_t lin_smem(bool gated, int bn, int stages) {
    return 1024 + (size_t)stages * lin_stage_bytes(gated, bn) + sizeof(LinShared);
}

struct LinTile {
    int e, mt, row0, n, n16;  // expert, tile of outputs, first row of y, tokens, in steps of 16
};

// Tile `i` of the launch; false past the last.
__device__ __forceinline__ bool lin_tile(const LinArgs &a, const LinShared &s, int i, LinTile &t) {
    if (i >= s.pre[a.E] * a.mt) return false;
    int lo = 0, hi = a.E;  // the expert: pre[lo] * mt <= i < pre[lo + 1] * mt
    while (hi - lo > 1) {
        const int m = (lo + hi) / 2;
        if (s.pre[m] * a.mt <= i) lo = m;
        else hi = m;
    }
    const int l = i - s.pre[lo] * a.mt, nt = s.pre[lo + 1] - s.pre[lo];
    const int rows = s.cnt[lo];
    // bands of token tiles; in a band the outputs' tiles one after the other
    const int b = l / (a.band * a.mt), r = l - b * a.band * a.mt;
    const int w = min(a.band, nt - b * a.band);
    const int mt = r / w, ti = b * a.band + (r - mt * w);
    const int per = ((rows + nt - 1) / nt + 15) & ~15;  // equal tiles: at most bn, none empty
    t.e = lo;
    t.mt = mt;
    t.row0 = s.off[lo] + ti * per;
    t.n = min(per, rows - ti * per);
    t.n16 = (t.n + 15) & ~15;
    return true;
}

__device__ __forceinline__ bool lin_wait(uint64_t *bar, uint32_t parity, const LinArgs &a,
                                         volatile int *abort) {
    bool ok = mbar_try_wait(bar, parity);
    if (!ok) {
        const uint64_t t0 = globaltimer_ns();
        for (uint32_t it = 1; !ok; ++it) {
            ok = mbar_try_wait(bar, parity);
            if (!ok && (it & 15u) == 0) {
                if (*abort) break;
                if (globaltimer_ns() - t0 > a.wait_ns) {
                    atomicOr(a.err, RB_LIN_ERR_WAIT);
                    *abort = 1;
                    break;
                }
            }
        }
    }
    return __all_sync(0xffffffffu, ok);  // the warp goes one way
}

// 16 consecutive columns of this thread's lane.
__device__ __forceinline__ void lin_ld16(uint32_t taddr, float (&v)[16]) {
    tmem_ld16(taddr, reinterpret_cast<int(&)[16]>(v), 0);
}
// Wait for it; the values are not used before.
__device__ __forceinline__ void lin_ld_done(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]),
                   "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]),
                   "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}

__device__ __forceinline__ float lin_silu(float g) { return g / (1.f + expf(-g)); }

__device__ __forceinline__ void lin_store(const LinArgs &a, int64_t at, float v) {
    if (a.out_dtype == RABBIT_CUDA_F32) static_cast<float *>(a.y)[at] = v;
    else if (a.out_dtype == RABBIT_CUDA_F16) static_cast<__half *>(a.y)[at] = from_f32<__half>(v);
    else static_cast<__nv_bfloat16 *>(a.y)[at] = from_f32<__nv_bfloat16>(v);
}

// Which of 32 tokens of a tile, from c on, are written: bit j for token c + j.
__device__ __forceinline__ uint32_t lin_written(const LinArgs &a, const LinTile &t, int c, int lane) {
    bool w = c + lane < t.n;
    if (w && a.rows) {
        const int r = __ldg(a.rows + t.row0 + c + lane);
        w = r >= 0 && r < a.x_rows;
    }
    return __ballot_sync(0xffffffffu, w);
}

__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Word at `p` (this CTA's shared memory) of the cluster's CTA `rank`.
__device__ __forceinline__ float cluster_ld(const float *p, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

template <bool F8, bool GATED>
__global__ void __launch_bounds__(kLinThreads, 1)
    k_linear(const __grid_constant__ LinArgs a, const __grid_constant__ CUtensorMap mw,
             const __grid_constant__ CUtensorMap mx) {
    extern __shared__ uint8_t lin_raw[];
    uint8_t *ring = lin_raw + ((1024u - (smem_u32(lin_raw) & 1023u)) & 1023u);
    constexpr int G = GATED ? 2 : 1;
    const uint32_t stage_bytes = lin_stage_bytes(GATED, a.bn);
    LinShared &s = *reinterpret_cast<LinShared *>(ring + (size_t)a.stages * stage_bytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int width = G * a.bn;                       // columns of a buffer
    const int bufs = min(512 / width, kLinBufs);
    volatile int *abort = &s.abort;

    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < bufs; ++i) {
            mbar_init(&s.dfull[i], 1);
            mbar_init(&s.sfull[i], 1);
            mbar_init(&s.dempty[i], 8);
        }
        mbar_init(&s.mdone, 1);
        s.abort = 0;
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc(&s.tmem, 512);
    launch_dependents();
    wait_prerequisite();
    // The experts' rows; with offsets out of order or range the call has none at all (tiles
    // of ranges that overlap could be more than the launch was made for).
    bool bad = false;
    for (int e = threadIdx.x; e < a.E; e += kLinThreads) {
        int lo = 0, hi = a.R;
        if (a.offsets) {
            lo = a.offsets[e];
            hi = a.offsets[e + 1];
            bad |= lo < 0 || hi < lo || hi > a.R;
        }
        s.off[e] = lo;
        s.cnt[e] = hi - lo;
    }
    bad = __syncthreads_or(bad);
    if (bad && threadIdx.x == 0) atomicOr(a.err, RB_LIN_ERR_OFFSETS);
    if (warp == 0) {
        int before = 0;
        for (int e0 = 0; e0 < a.E; e0 += 32) {
            int n = e0 + lane < a.E && !bad ? (s.cnt[e0 + lane] + a.bn - 1) / a.bn : 0;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int m = __shfl_up_sync(0xffffffffu, n, d);
                if (lane >= d) n += m;
            }
            if (e0 + lane < a.E) s.pre[e0 + lane + 1] = before + n;
            before += __shfl_sync(0xffffffffu, n, 31);
        }
        if (lane == 0) s.pre[0] = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    const uint32_t rank = a.split > 1 ? cluster_rank() : 0;
    // a cluster has one tile; a CTA by itself each gridDim.x-th
    const int first = blockIdx.x / a.split, stride = a.split > 1 ? 1 << 30 : gridDim.x;
    const int k0 = (int)((int64_t)a.steps * rank / a.split);
    const int k1 = (int)((int64_t)a.steps * (rank + 1) / a.split);
    LinTile t;

    if (warp == 0) {  // ------------------------------------------------ TMA
        const uint64_t keep = policy_evict_last(), once = policy_evict_first();
        int it = 0;
        bool ok = true;
        for (int i = first; ok && lin_tile(a, s, i, t); i += stride) {
            int src[2][4];  // with a list: the rows of x of quads lane and lane + 32
            if (a.rows) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int c = (lane + 32 * h) * 4 + j;
                        int r = c < t.n ? __ldg(a.rows + t.row0 + c) : 0;
                        if (r < 0 || r >= a.x_rows) {
                            atomicOr(a.err, RB_LIN_ERR_ROWS);
                            r = 0;  // read for nothing: lin_written leaves the row out
                        }
                        src[h][j] = r;
                    }
            }
            const int boxes = (t.n16 + a.box - 1) / a.box;
            const uint32_t bytes = G * kLinTile + (a.rows ? t.n16 : boxes * a.box) * 128;
            // weights that no other tile of tokens reads leave the L2 first
            const uint64_t pol = s.pre[t.e + 1] - s.pre[t.e] > 1 ? keep : once;
            for (int k = k0; k < k1; ++k, ++it) {
                const int st = it % a.stages;
                if (!(ok = lin_wait(&s.empty[st], ((it / a.stages) & 1) ^ 1, a, abort))) break;
                uint8_t *base = ring + (size_t)st * stage_bytes, *xb = base + G * kLinTile;
                const int c0 = k * (F8 ? 128 : 64);
                if (lane == 0) {
                    mbar_arrive_expect_tx(&s.full[st], bytes);
#pragma unroll
                    for (int g = 0; g < G; ++g)
                        tma_load_4d(base + g * kLinTile, &mw, c0, t.mt * 128, g, t.e, &s.full[st],
                                    pol);
                }
                __syncwarp();
                if (a.rows) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int q = lane + 32 * h;
                        if (4 * q < t.n16)
                            tma_gather4(xb + q * 512, &mx, c0, src[h][0], src[h][1], src[h][2],
                                        src[h][3], &s.full[st]);
                    }
                } else if (lane < boxes) {
                    tma_load_2d(xb + lane * a.box * 128, &mx, c0, t.row0 + lane * a.box,
                                &s.full[st]);
                }
            }
        }
        if (!ok)  // copies under way end before the block does
            for (int j = max(0, it - a.stages); j < it; ++j)
                if (lane == 0) mbar_wait(&s.full[j % a.stages], (j / a.stages) & 1, a.wait_ns, nullptr, 0);
    } else if (warp == 1) {  // ------------------------------------------ MMA
        int it = 0, db = 0;
        bool ok = true;
        for (int i = first; ok && lin_tile(a, s, i, t); i += stride) {
            const uint32_t idesc = float_idesc(a.format, t.n16);
            for (int k = k0; k < k1; ++k, ++it) {
                const int st = it % a.stages, buf = db % bufs;
                if (F8 || k == k0)
                    if (!(ok = lin_wait(&s.dempty[buf], ((db / bufs) & 1) ^ 1, a, abort))) break;
                if (!(ok = lin_wait(&s.full[st], (it / a.stages) & 1, a, abort))) break;
                tc_fence_after();
                if (lane == 0) {
                    uint8_t *base = ring + (size_t)st * stage_bytes;
                    const uint64_t xd = swizzled_desc(smem_u32(base + G * kLinTile));
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const uint64_t wd = swizzled_desc(smem_u32(base + g * kLinTile));
                        const uint32_t d = tmem + buf * width + g * a.bn;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mma_float_ss<F8>(d, wd + 2 * j, xd + 2 * j, idesc,
                                             j > 0 || (!F8 && k > k0));
                    }
                    mma_commit(&s.empty[st]);
                    if (F8 || k == k1 - 1) mma_commit(&s.dfull[buf]);
                }
                __syncwarp();
                if (F8 || k == k1 - 1) ++db;
            }
        }
        if (!ok && lane == 0) {  // products under way end before their memory is given back
            mma_commit(&s.mdone);
            mbar_wait(&s.mdone, 0, a.wait_ns, nullptr, 0);
        }
        __syncwarp();
    } else if (F8 && warp == 2) {  // --------------------------------- scales
        constexpr int NT = GATED ? 4 : 8;  // tokens of a lane
        const int nb = a.mt;               // rows of scale blocks of a matrix
        int db = 0;
        bool ok = true;
        for (int i = first; ok && lin_tile(a, s, i, t); i += stride) {
            const float *xs[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int c = lane + 32 * j;
                int64_t r = t.row0 + c;
                if (c < t.n && a.rows) {
                    r = __ldg(a.rows + r);
                    if (r < 0 || r >= a.x_rows) r = 0;
                }
                xs[j] = c < t.n ? a.xs + r * a.xs_stride : nullptr;
            }
            const float *ws = a.ws + ((int64_t)t.e * G * nb + t.mt) * a.steps;
            float v[NT], w[G];
            auto fetch = [&](int k) {
#pragma unroll
                for (int j = 0; j < NT; ++j) v[j] = xs[j] ? __ldg(xs[j] + k) : 0.f;
#pragma unroll
                for (int g = 0; g < G; ++g) w[g] = __ldg(ws + (int64_t)g * nb * a.steps + k);
            };
            fetch(k0);
            for (int k = k0; k < k1; ++k, ++db) {
                const int buf = db % bufs;
                if (!(ok = lin_wait(&s.dempty[buf], ((db / bufs) & 1) ^ 1, a, abort))) break;
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        if (lane + 32 * j < t.n16) s.sc[buf][g * a.bn + lane + 32 * j] = v[j] * w[g];
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.sfull[buf]);
                if (k + 1 < k1) fetch(k + 1);
            }
        }
    } else if (warp >= 4) {  // ------------------------------------- readout
        const int q = warp & 3, h = (warp - 4) >> 2;
        const int nl = q * 32 + lane;  // output of the tile
        float *part = reinterpret_cast<float *>(ring);
        int db = 0;
        bool ok = true;
        for (int i = first; ok && lin_tile(a, s, i, t); i += stride) {
            const int n = t.mt * 128 + nl;
            const int64_t y0 = (int64_t)t.row0 * a.y_stride + n;
            // values of the 16 tokens from c on (gated: gate's and up's): to y, or to the
            // cluster's sum
            auto put = [&](int c, const float (&v)[16], const float (&u)[16]) {
                if (a.split > 1) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        part[(c + j) * 128 + nl] = v[j];
                        if (GATED) part[(a.bn + c + j) * 128 + nl] = u[j];
                    }
                    return;
                }
                uint32_t to = lin_written(a, t, c, lane);
                if (n >= a.N) to = 0;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (to >> j & 1)
                        lin_store(a, y0 + (c + j) * a.y_stride,
                                  GATED ? lin_silu(v[j]) * u[j] : v[j]);
                __syncwarp();
            };
            if constexpr (F8) {
                constexpr int NC = GATED ? 4 : 8;  // blocks of 16 tokens
                float acc[G][NC][16];
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[g][c][j] = 0.f;
                for (int k = k0; k < k1; ++k, ++db) {
                    const int buf = db % bufs, ph = (db / bufs) & 1;
                    if (!(ok = lin_wait(&s.sfull[buf], ph, a, abort))) break;
                    if (!(ok = lin_wait(&s.dfull[buf], ph, a, abort))) break;
                    tc_fence_after();
                    const uint32_t d = tmem + ((uint32_t)(q * 32) << 16) + buf * width;
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            const int col = (2 * c + h) * 16;
                            if (col >= t.n16) break;
                            float v[16];
                            lin_ld16(d + g * a.bn + col, v);
                            const float4 *sc = reinterpret_cast<const float4 *>(&s.sc[buf][g * a.bn + col]);
                            float4 f[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) f[j] = sc[j];
                            lin_ld_done(v);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                acc[g][c][4 * j] = fmaf(v[4 * j], f[j].x, acc[g][c][4 * j]);
                                acc[g][c][4 * j + 1] = fmaf(v[4 * j + 1], f[j].y, acc[g][c][4 * j + 1]);
                                acc[g][c][4 * j + 2] = fmaf(v[4 * j + 2], f[j].z, acc[g][c][4 * j + 2]);
                                acc[g][c][4 * j + 3] = fmaf(v[4 * j + 3], f[j].w, acc[g][c][4 * j + 3]);
                            }
                        }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s.dempty[buf]);
                }
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    if ((2 * c + h) * 16 < t.n16)
                        put((2 * c + h) * 16, acc[0][c], acc[G - 1][c]);
            } else {
                const int buf = db % bufs;
                if (!(ok = lin_wait(&s.dfull[buf], (db / bufs) & 1, a, abort))) break;
                tc_fence_after();
                const uint32_t d = tmem + ((uint32_t)(q * 32) << 16) + buf * width;
                for (int c = 16 * h; c < t.n16; c += 32) {
                    float v[16], u[16];
                    lin_ld16(d + c, v);
                    if (GATED) lin_ld16(d + a.bn + c, u);
                    lin_ld_done(v);
                    if (GATED) lin_ld_done(u);
                    put(c, v, GATED ? u : v);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.dempty[buf]);
                ++db;
            }
        }
    }
    __syncwarp();
    if (a.split > 1) {  // one tile a cluster: its parts summed in the order of the ranks
        cluster_arrive();
        cluster_wait();
        if (warp >= 4 && !*abort && lin_tile(a, s, first, t)) {
            const int nl = (warp & 3) * 32 + lane, h = (warp - 4) >> 2;
            const int n = t.mt * 128 + nl;
            const float *part = reinterpret_cast<const float *>(ring);
            for (int c = 0; c < t.n; c += 32) {
                const uint32_t to = lin_written(a, t, c, lane);
                for (int j = 0; j < 32; ++j) {
                    const int tok = c + j, turn = tok / a.split;
                    if (!(to >> j & 1) || tok - turn * a.split != (int)rank || (turn & 1) != h) continue;
                    float v = 0.f, u = 0.f;
                    for (int r = 0; r < a.split; ++r) {
                        v += cluster_ld(part + tok * 128 + nl, r);
                        if (GATED) u += cluster_ld(part + (a.bn + tok) * 128 + nl, r);
                    }
                    if (n < a.N)
                        lin_store(a, (int64_t)(t.row0 + tok) * a.y_stride + n,
                                  GATED ? lin_silu(v) * u : v);
                }
            }
        }
        cluster_arrive();  // nobody leaves while its part is read
        cluster_wait();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
}

}  // namespace rb
