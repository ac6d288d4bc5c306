// rb_linear_rows.cuh -- e4m3 products of many tokens: the tokens are the MMA's rows.
//
// Each step's product of 256 tokens x 256 weight rows is read out of tensor memory and added to
// 32-bit registers times sx[token] sw[block] (rb_linear.cuh, kLinF8). With the tokens on the
// lanes a thread has one token, its scales are two numbers a step, and an element is one fma; with
// the weights on the lanes each column has a scale of its own, and reading those from shared
// memory (32 broadcasts of 16 bytes a warp and step) held the readout to 650 cycles a step
// where these take 335 and the MMAs 512. 8191 x 4096 x 28672: 1.13 ms in a long run (1.7 PFLOP/s, at the
// power limit) and 1.07 in one of 20 calls, where that way took 2.5 and copies without MMAs and readout
// 0.67: what is left is bound by the L2.
//
// A pair of CTAs has a tile of 256 tokens and 256 weight rows (gated: 128 of the gate, 128 of
// the up matrix): CTA r brings tokens 128 r .. and the r-th half of the weight rows, and
// CTA 0 issues MMAs of M = 256, N = 256 for both. Roles: warp 0 TMA, warp 1 MMA, warps 4..11
// readout (warp w: tokens 32 (w % 4) .., the even or odd blocks of 16 columns), warps 12..15
// gather the token rows of a list.
#pragma once
#include "rb_linear.cuh"

namespace rb {

constexpr uint32_t kRowsStage = 2 * kLinTile;
constexpr uint32_t kRowsPitch = 128 + 16;          // bytes of a token's outputs on their way
constexpr uint32_t kRowsOut = 128 * kRowsPitch;
__host__ __device__ constexpr size_t lin_rows_fixed(int E) {
    return 1024 + kRowsOut + sizeof(LinShared) + 8 * (size_t)(E + 1);
}

template <bool GATED, typename OUT>
__global__ void __launch_bounds__(kLinThreads, 1)
    k_linear_rows(const __grid_constant__ LinArgs a, const __grid_constant__ CUtensorMap mw,
                  const __grid_constant__ CUtensorMap mx) {
    extern __shared__ uint8_t lin_raw[];
    uint8_t *ring = lin_raw + ((1024u - (smem_u32(lin_raw) & 1023u)) & 1023u);
    uint8_t *outs = ring + (size_t)a.stages * kRowsStage;
    LinShared &s = *reinterpret_cast<LinShared *>(outs + kRowsOut);
    int *off = reinterpret_cast<int *>(&s + 1), *pre = off + a.E + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort = &s.abort;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
            mbar_init(&s.rows[i], 128);
            mbar_init(&s.told[i], 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.dfull[i], 1);
            mbar_init(&s.mfree[i], 16);
        }
        mbar_init(&s.mdone, 1);
        s.abort = 0;
        s.issued = s.stepped = s.filled = s.ended = 0;
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc_pair(&s.tmem, 512);
    launch_dependents();
    wait_prerequisite();
    lin_experts(a, off, pre, 256);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers are ready
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    const int first = blockIdx.x / 2, stride = gridDim.x / 2;
    LinTile t;

    // Registers: 512 x 128 at the launch (linear_create checks it); 128 x 72 + 128 x 56 +
    // 256 x 192 from here.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0) {  // -------------------------------------------- TMA
            if (elect_one()) {
                const uint64_t keep = policy_evict_last();
                LinRing st;
                int issued = 0;
                bool ok = true;
                const uint32_t bytes = 2 * (kLinTile + (a.rows ? 0 : kLinTile));
                const int held = a.withhold >> rank & 1;
                for (int i = first; ok && lin_tile(a, off, pre, i, t); i += a.withhold ? 1 << 30 : stride) {
                    const int n0 = GATED ? t.mt * 128 : t.mt * 256 + rank * 128;
                    const int r0 = t.row0 + rank * 128;
                    for (int k = 0; k < a.steps - held; ++k, ++issued) {
                        if (!(ok = lin_wait1(&s.empty[st.at], st.phase ^ 1, a, abort))) break;
                        uint8_t *base = ring + (size_t)st.at * kRowsStage;
                        const uint32_t bar = cluster_addr(&s.full[st.at], 0);
                        s.bytes[st.at] = bytes / 2;
                        if (leader) mbar_arrive_expect_tx(&s.full[st.at], bytes);
                        for (int b = 0; b < 128; b += GATED ? 64 : 128)  // (the map's boxes)
                            tma_load_4d_pair(base + kLinTile + b * 128, &mw, k * 128, n0 + b, GATED ? rank : 0,
                                             t.e, bar, keep);
                        if (!a.rows) tma_load_2d_pair(base, &mx, k * 128, r0, bar);
                        st.next(a.stages);
                    }
                }
                if (ok) lin_emptied(a, s, issued, abort);
                s.issued = issued;
            }
            __syncwarp();
        } else if (warp == 1) {  // -------------------------------------- MMA
            if (leader) {
                if (elect_one()) {
                    LinRing st, db;
                    bool ok = true;
                    int stepped = 0;
                    const uint64_t xd0 = swizzled_desc(smem_u32(ring)), wd0 = swizzled_desc(smem_u32(ring + kLinTile));
                    const uint32_t idesc = float_idesc(a.format, 256, 256);
                    for (int i = first; ok && lin_tile(a, off, pre, i, t); i += stride)
                        for (int k = 0; k < a.steps; ++k) {
                            if (!(ok = lin_wait1<true>(&s.full[st.at], st.phase, a, abort))) break;
                            if (a.rows && !(ok = lin_wait1<true>(&s.told[st.at], st.phase, a, abort))) break;
                            cluster_acquire_shared();
                            if (!(ok = lin_wait1<true>(&s.mfree[db.at], db.phase ^ 1, a, abort))) break;
                            tc_fence_after();
                            const uint64_t step = (uint64_t)(st.at * kRowsStage) >> 4;
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                mma_float_ss<true, true>(tmem + db.at * 256, xd0 + step + 2 * j, wd0 + step + 2 * j,
                                                         idesc, j > 0);
                            mma_commit_pair(&s.dfull[db.at]);
                            mma_commit_pair(&s.empty[st.at]);
                            ++stepped;
                            st.next(a.stages);
                            db.next(2);
                        }
                    if (!ok) mma_commit_pair(&s.mdone);  // lin_settle waits for it
                    s.stepped = s.filled = stepped;
                    s.ended = !ok;
                }
            }
            __syncwarp();
        } else if (warp == 2 && a.rows) {  // ------------- word of gathered rows
            if (elect_one())
                lin_tell<true>(a, s, off, pre, first, stride, 0, a.steps, abort);
            __syncwarp();
        }
    } else if (warp >= 12) {  // ------------------------------------- gather
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (a.rows) {
            LinRing st;
            bool ok = true;
            for (int i = first; ok && lin_tile(a, off, pre, i, t); i += stride)
                ok = lin_gather<8>(a, s, smem_u32(ring), kRowsStage, t, rank * 128, 128, 0, a.steps, st, abort);
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {  // ---------------------------------------------------- readout
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int q = warp & 3, h = (warp - 4) >> 2, tid = threadIdx.x - 128;
        const int mine = q * 32 + lane;  // this thread's token of the CTA's 128
        const int nb = (a.N + 127) / 128;
        const uint32_t lanes = (uint32_t)(q * 32) << 16, mfree = cluster_addr(&s.mfree[0], 0);
        constexpr int AHEAD = 4;  // steps whose scales are on their way
        LinRing db;
        bool ok = true;
        uint32_t tile = 0;
        const float *xs, *w0, *w1;  // scales of this thread's token and of columns 0..127, 128..255
        float sx[AHEAD], s0[AHEAD], s1[AHEAD];
        auto fetch = [&](int k, int j) {
            if (k >= a.steps) return;
            sx[j] = __ldg(xs + k);
            s0[j] = __ldg(w0 + k);
            s1[j] = __ldg(w1 + k);
        };
        auto begin = [&](const LinTile &t) {  // a tile's scales and the first of them
            const int c = rank * 128 + mine;
            int r = t.row0 + c;
            if (c < t.n && a.rows) {
                r = __ldg(a.rows + r);
                if (r >= a.x_rows) r = -1;
            }
            if (c >= t.n) r = -1;
            // (the tile before the last is behind every warp, by the barrier)
            const uint32_t w = __ballot_sync(0xffffffffu, r >= 0);
            if (h == 0 && lane == 0) s.written[(tile + 1) & 1][q] = w;
            xs = a.xs + (uint64_t)max(r, 0) * a.xs_stride;
            const int b0 = GATED ? t.mt : 2 * t.mt, b1 = GATED ? nb + t.mt : min(2 * t.mt + 1, nb - 1);
            w0 = a.ws + ((int64_t)t.e * (1 + GATED) * nb + b0) * a.steps;
            w1 = w0 + (int64_t)(b1 - b0) * a.steps;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) fetch(j, j);
        };
        LinTile next;
        bool more = lin_tile(a, off, pre, first, next);
        if (more) begin(next);
        for (int i = first; ok && more; i += stride) {
            t = next;
            ++tile;
            float acc[8][16];  // block 2 j + h
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int l = 0; l < 16; ++l) acc[j][l] = 0.f;
            for (int k = 0; ok && k < a.steps; k += AHEAD) {
#pragma unroll
                for (int p = 0; p < AHEAD; ++p) {
                    if (k + p >= a.steps) break;
                    const float f0 = sx[p] * s0[p], f1 = sx[p] * s1[p];
                    fetch(k + p + AHEAD, p);
                    if (!(ok = lin_wait(&s.dfull[db.at], db.phase, a, abort))) break;
                    tc_fence_after();
                    const uint32_t d = tmem + lanes + db.at * 256 + 16 * h;
                    float v[2][16];
                    lin_ld16(d, v[0]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        lin_ld_done(v[j & 1]);
                        if (j < 7) {
                            lin_ld16(d + 32 * (j + 1), v[(j + 1) & 1]);
                        } else {  // all is in registers
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) cluster_bar_arrive(mfree + db.at * 8);
                            db.next(2);
                        }
                        const float f = j < 4 ? f0 : f1;
#pragma unroll
                        for (int l = 0; l < 16; ++l) acc[j][l] = fmaf(v[j & 1][l], f, acc[j][l]);
                    }
                }
            }
            // (a wait that ran out ends it for every warp of the block before a barrier among them)
            ok = named_all(1, kLinReaders, ok);
            if (!ok) break;
            // the next tile's first scales come while this one's outputs leave
            more = lin_tile(a, off, pre, i + stride, next);
            if (more) begin(next);
            // Out in rows: W columns of the 128 tokens at a time, through shared memory
            constexpr int W = 128 / (int)sizeof(OUT), NB = W / 32;  // columns, a thread's blocks of 16
            const int n0 = t.mt * (GATED ? 128 : 256);
#pragma unroll
            for (int o = 0; o < (GATED ? 4 : 8) / NB; ++o) {
                if (n0 + o * W >= a.N) break;
                named_sync(1, kLinReaders);  // the outputs before have left
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float(&g)[16] = acc[o * NB + b];
#pragma unroll
                    for (int l = 0; l < 16; l += 8) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            v[e] = GATED ? lin_silu<OUT>(g[l + e]) * acc[(o * NB + b + 4) & 7][l + e] : g[l + e];
                        store8<true>(reinterpret_cast<OUT *>(outs + mine * kRowsPitch) + (2 * b + h) * 16 + l, v);
                    }
                }
                named_sync(1, kLinReaders);
                const int col = n0 + o * W, piece = tid & 7;
                constexpr int V = 16 / (int)sizeof(OUT);
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const int tok = p * 32 + (tid >> 3);
                    if (!(s.written[tile & 1][p] >> (tid >> 3) & 1)) continue;
                    const uint8_t *row = outs + tok * kRowsPitch;
                    OUT *y = static_cast<OUT *>(a.y) + (int64_t)(t.row0 + rank * 128 + tok) * a.y_stride + col;
                    if (a.vec && col + (piece + 1) * V <= a.N) {
                        reinterpret_cast<uint4 *>(y)[piece] = reinterpret_cast<const uint4 *>(row)[piece];
                        continue;
                    }
                    // rows that do not lie on 16 bytes, or the last columns: 4 bytes at a time, the
                    // eight threads' side by side (without them: this thread's piece)
#pragma unroll 1
                    for (int e = 0; e < 4; ++e) {
                        const int w = a.vec ? 4 * piece + e : 8 * e + piece, c = w * (4 / (int)sizeof(OUT));
                        const uint32_t v = reinterpret_cast<const uint32_t *>(row)[w];
                        if (sizeof(OUT) == 4 || (a.pairs && col + c + 2 <= a.N)) {
                            if (col + c < a.N) *reinterpret_cast<uint32_t *>(y + c) = v;
                        } else {
                            const OUT *two = reinterpret_cast<const OUT *>(&v);
                            if (col + c < a.N) y[c] = two[0];
                            if (col + c + 1 < a.N) y[c + 1] = two[1];
                        }
                    }
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // both have read their products
    if (*abort) lin_settle<true>(a, s, 2);
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
    cluster_sync_all();
}

}  // namespace rb
