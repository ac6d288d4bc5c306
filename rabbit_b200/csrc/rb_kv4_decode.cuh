// rb_kv4_decode.cuh -- attention over the 4-bit cache for few query rows a
// sequence (decoding, drafted tokens): every KV head's rows at once against a
// stream of granules.
//
// A CTA walks an equal run of the batch's granules (kv4_cut), whatever
// sequences they belong to: one warp fetches granules into a ring in shared
// memory (one bulk copy each), W warps take them in turn. A warp keeps the
// query rows' operands and its own running (maximum, sum, output) in registers;
// at the end of an item the warps merge in shared memory. An item that a run's
// border cuts is merged from the runs' partial results by whichever CTA
// arrives last, in the order of the runs, so results do not depend on timing.
//
// The arithmetic of a granule, on m16n8k16 fp16 instructions with fp32 sums:
//  * S = Q K^T: rows are query rows, columns 8 tokens. K's nibbles u = code + 8
//    go in as the fp16 numbers u 2^-24 (a nibble in the low mantissa bits is
//    one: no conversion) and 16 u 2^-24 (the next nibble, one mask; those
//    channels of Q are a sixteenth). The accumulator starts at -8 2^-24 sum Q,
//    which takes the bias off, and each group's sum is scaled in fp32.
//    Q is scaled by a power of two per row into fp16's upper range: exact for
//    16-bit queries; fp32 queries (SPLIT) go in two terms of 11 bits, the
//    second in the instruction's other 8 rows.
//  * O^T = V^T P^T: rows are channels, columns query rows. S's registers are
//    already the operand's layout. Each group's weights are p s, s the value
//    scale, rounded to fp16 (fp32 queries: two terms).
//  * p = 2^(t - M) with M a running reference >= max_j (t_j + log2 s_j) - 14, so
//    every weight is at most 2^14 in fp16 and the largest are far above its
//    subnormals. M is raised only when a weight would pass 2^14, to weights of
//    at most 2^6: with a first tile's maximum as a guide that is rare, and the
//    output is rescaled only then.
#pragma once
#include "rb_device.cuh"
#include "rb_kv4_attn.cuh"
#include "rb_types.cuh"

namespace rb {

constexpr float kNoRef = -3e38f;  // M before any visible token

template <int NG, int RB, bool SPLIT>
struct DecodeCfg {
    static constexpr int W = 7;                      // consumer warps; with the producer 8, two a sub-partition
    static constexpr int kThreads = 32 * (W + 1);
    static constexpr int kRows = 8 * RB;
    static constexpr int kCtas = RB == 1 && NG <= 4 ? 2 : 1;  // per SM
    static constexpr int S = 3 * W;                  // ring slots (at least 16: the producer's step is 8)
    static constexpr int kCh = 32 * NG;
    static constexpr int kStride = kCh + 4;          // merge rows: spreads a quarter warp over the banks
    static constexpr int NB = RB * (SPLIT ? 2 : 1);  // 8-row operand blocks
    static constexpr int MT = (NB + 1) / 2;          // 16-row tiles
    static constexpr size_t kRing = (size_t)S * kv4_bytes(NG);
    static constexpr size_t kMerge = sizeof(float) * (size_t)W * kRows * kStride;
    static constexpr size_t kSmem = kRing + kMerge;
};

// Block-wide helpers over the CTA's threads.
template <int NT>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *warp_sums, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += up;
    }
    __syncthreads();  // warp_sums may still be read from an earlier call
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        const int64_t t = warp_sums[w];
        if (w < warp) before += t;
        total += t;
    }
    return before + s - v;  // exclusive
}

__device__ __forceinline__ Kv4Seq load_seq(const Kv4AttnArgs &a, int i, int *bad = nullptr) {
    Kv4Seq s;
    const int s0 = a.q_start ? a.q_start[i] : i, s1 = a.q_start ? a.q_start[i + 1] : i + 1;
    const int e = kv4_seq(s0, s1, a.kv_len[i], a.T, a.max_q, (int64_t)a.max_pages * a.c.page, a.window, s);
    if (bad) *bad = e;
    return s;
}

// A position in the batch's units: sequence, item of it, unit of the item.
struct Kv4Walk {
    Kv4Seq s;
    int seq, sub, off;
};

// Store 4 consecutive channels of a row.
__device__ __forceinline__ void store4(const Kv4AttnArgs &a, int64_t at, const float (&v)[4], int n) {
    if (a.dtype == RABBIT_CUDA_F32) {
        float *o = static_cast<float *>(a.out) + at;
        if (a.vec) {
            *reinterpret_cast<float4 *>(o) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            for (int i = 0; i < n; ++i) o[i] = v[i];
        }
        return;
    }
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = a.dtype == RABBIT_CUDA_F16 ? __half_as_ushort(__float2half_rn(v[i]))
                                          : __bfloat16_as_ushort(__float2bfloat16_rn(v[i]));
    uint16_t *o = static_cast<uint16_t *>(a.out) + at;
    if (a.vec) {
        *reinterpret_cast<uint2 *>(o) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    } else {
        for (int i = 0; i < n; ++i) o[i] = h[i];
    }
}

// 8 channels of a query row as fp32.
__device__ __forceinline__ void load_q8(const Kv4AttnArgs &a, int64_t at, float (&v)[8]) {
    if (a.dtype == RABBIT_CUDA_F32) {
        const float *p = static_cast<const float *>(a.q) + at;
        if (a.vec) load8<true>(v, p);
        else load8<false>(v, p);
    } else if (a.dtype == RABBIT_CUDA_F16) {
        const __half *p = static_cast<const __half *>(a.q) + at;
        if (a.vec) load8<true>(v, p);
        else load8<false>(v, p);
    } else {
        const __nv_bfloat16 *p = static_cast<const __nv_bfloat16 *>(a.q) + at;
        if (a.vec) load8<true>(v, p);
        else load8<false>(v, p);
    }
}

template <int NG, int RB, bool SPLIT>
__global__ void __launch_bounds__(DecodeCfg<NG, RB, SPLIT>::kThreads, DecodeCfg<NG, RB, SPLIT>::kCtas)
    k_kv4_decode(const __grid_constant__ Kv4AttnArgs a) {
    using C = DecodeCfg<NG, RB, SPLIT>;
    constexpr int W = C::W, S = C::S, NB = C::NB;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[S], empty[S];
    __shared__ uint8_t valid[S];
    __shared__ int64_t warp_sums[C::kThreads / 32];
    __shared__ int64_t found_before;
    __shared__ int found_seq;
    __shared__ float wm[W][C::kRows], wl[W][C::kRows];
    __shared__ float fac[W][C::kRows], suml[C::kRows];
    __shared__ bool last_in;
    float *mo = reinterpret_cast<float *>(smem + C::kRing);  // [W][rows][kStride]
    launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init_fence();
    }
    wait_prerequisite();
    const Kv4View &c = a.c;
    const int G = a.nh / c.nkv;

    // ---- this CTA's run of units
    int64_t mine = 0;
    for (int i = tid; i < a.n_seqs; i += C::kThreads) {
        int bad;
        const Kv4Seq s = load_seq(a, i, &bad);
        if (bad && blockIdx.x == 0) atomicOr(c.err, bad);
        mine += kv4_items(s, G, C::kRows, c.nkv) * kv4_units(s);
    }
    int64_t total, excl = block_scan<C::kThreads>(mine, warp_sums, total);
    if (total == 0) return;
    // a run shorter than two granules a warp is not worth its merge
    const int64_t most = (total + 2 * W - 1) / (2 * W);
    const int64_t parts = most < gridDim.x ? most : gridDim.x;
    if (blockIdx.x >= parts) return;
    const int64_t u0 = kv4_cut(blockIdx.x, total, parts), u1 = kv4_cut(blockIdx.x + 1, total, parts);
    if (a.n_seqs <= C::kThreads) {
        if (mine > 0 && excl <= u0 && u0 < excl + mine) {
            found_seq = tid;
            found_before = excl;
        }
    } else {
        int64_t base = 0;
        for (int i0 = 0; i0 < a.n_seqs && base <= u0; i0 += C::kThreads) {
            const int i = i0 + tid;
            int64_t cost = 0, all;
            if (i < a.n_seqs) {
                const Kv4Seq s = load_seq(a, i);
                cost = kv4_items(s, G, C::kRows, c.nkv) * kv4_units(s);
            }
            const int64_t before = base + block_scan<C::kThreads>(cost, warp_sums, all);
            if (cost > 0 && before <= u0 && u0 < before + cost) {
                found_seq = i;
                found_before = before;
            }
            base += all;
        }
    }
    __syncthreads();
    Kv4Walk w;
    w.seq = found_seq;
    w.s = load_seq(a, w.seq);
    {
        const int64_t r = u0 - found_before;
        w.sub = (int)(r / kv4_units(w.s));
        w.off = (int)(r % kv4_units(w.s));
    }
    // to the next item; true while the run goes on
    auto advance = [&](int64_t &u, int took) {
        u += took;
        w.off = 0;
        if (u >= u1) return false;
        if (++w.sub >= kv4_items(w.s, G, C::kRows, c.nkv)) {
            w.sub = 0;
            do w.s = load_seq(a, ++w.seq);
            while (w.s.nq == 0);
        }
        return true;
    };

    if (warp == W) {
        // ---- producer: granules of the run into the ring, 8 lanes at a time
        const uint64_t policy = policy_evict_first();
        uint32_t ring = 0;
        bool ok = true, more = true;
        for (int64_t u = u0; more && ok;) {
            const int take = (int)min((int64_t)(kv4_units(w.s) - w.off), u1 - u);
            const int real = w.s.n > 0 ? take : 0, head = w.sub % c.nkv;
            for (int k0 = 0; k0 < real && ok; k0 += 32) {
                const int k = k0 + lane;
                int page = -1, r = 0;
                if (k < real) {
                    const int pos = (w.s.g0 + w.off + k) * kKv4Granule, pi = pos / c.page;
                    r = pos - pi * c.page;
                    page = a.table[(int64_t)w.seq * a.max_pages + pi];
                    if (page < 0 || page >= c.n_pages) {
                        atomicOr(c.err, RB_KV4_ERR_PAGE);
                        page = -1;
                    }
                }
                for (int g8 = 0; g8 < 4 && k0 + 8 * g8 < real; ++g8) {
                    if ((lane >> 3) == g8 && k < real) {
                        const uint32_t at = ring + k, slot = at % S, gen = at / S;
                        if (gen > 0) ok = mbar_wait(&empty[slot], (gen - 1) & 1, a.wait_ns, c.err, 0);
                        if (ok) {
                            valid[slot] = page >= 0;
                            if (page >= 0) {
                                mbar_arrive_expect_tx(&full[slot], kv4_bytes(NG));
                                bulk_g2s(smem + slot * kv4_bytes(NG),
                                         c.base + (size_t)page * c.page_bytes() +
                                             (size_t)head * c.head_bytes() +
                                             (size_t)(r / kKv4Granule) * kv4_bytes(NG),
                                         kv4_bytes(NG), &full[slot], policy);
                            } else {
                                mbar_arrive(&full[slot]);
                            }
                        }
                    }
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
            }
            ring += real;
            more = advance(u, take);
        }
        // copies in flight end before the CTA does, also after a wait ran out
        if (!ok) {
            for (int i = lane; i < S; i += 32)
                for (int ph = 0; ph < 2; ++ph) mbar_wait(&full[i], ph, a.wait_ns, nullptr, 0);
        }
        return;
    }

    // ---- consumers
    const int g = lane >> 2, t = lane & 3;
    uint32_t ring = 0;
    bool ok = true, more = true;
    for (int64_t u = u0; more;) {
        const int units = kv4_units(w.s), take = (int)min((int64_t)(units - w.off), u1 - u);
        const int real = w.s.n > 0 ? take : 0;
        const int kvh = w.sub % c.nkv, rho0 = (w.sub / c.nkv) * C::kRows, R = min(C::kRows, w.s.nq * G - rho0);
        const int at_lo = w.s.len - w.s.nq + rho0 / G, at_hi = w.s.len - w.s.nq + (rho0 + R - 1) / G;

        // query operands of this item
        uint32_t qf[NB][2 * NG][2];
        float qs[NB][NG], cs[RB];
        int at[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int rho = rho0 + 8 * rb + g;
            const bool in = 8 * rb + g < R;
            const int qi = rho / G;
            at[rb] = in ? w.s.len - w.s.nq + qi : -1;
            const int64_t base = (int64_t)(w.s.row0 + qi) * a.qs + (int64_t)(kvh * G + rho % G) * c.hd;
            float q[NG][8], top = 0.f;
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
#pragma unroll
                for (int i = 0; i < 8; ++i) q[grp][i] = 0.f;
                if (in && 32 * grp + 8 * t < c.hd) load_q8(a, base + 32 * grp + 8 * t, q[grp]);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(q[grp][i]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^(14 - e), 2^e <= top: the largest goes to [2^14, 2^15)
            int e = (int)(__float_as_uint(top) >> 23) - 127;
            e = max(e, -100);
            const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
            const float down = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
            cs[rb] = a.scale * 16777216.0f * down;
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
#pragma unroll
                for (int part = 0; part < (SPLIT ? 2 : 1); ++part) {
                    const int b = SPLIT ? 2 * rb + part : rb;
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {  // step: even nibbles, then odd ones (16 u)
                        const float f = i ? 0.0625f : 1.0f, f1 = i ? 16.f : 1.0f;
                        float v[4] = {q[grp][i], q[grp][i + 4], q[grp][i + 2], q[grp][i + 6]};
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] *= part == 0 ? up * f : f;
                        const uint32_t x0 = pack_f16(v[0], v[1]), x1 = pack_f16(v[2], v[3]);
                        qf[b][2 * grp + i][0] = x0;
                        qf[b][2 * grp + i][1] = x1;
                        const float2 r0 = __half22float2(*reinterpret_cast<const __half2 *>(&x0));
                        const float2 r1 = __half22float2(*reinterpret_cast<const __half2 *>(&x1));
                        sum += ((r0.x + r0.y) + (r1.x + r1.y)) * f1;
                        if (SPLIT && part == 0) {  // what the first term leaves, in units of `up`
                            q[grp][i] = (v[0] - r0.x) * f1;
                            q[grp][i + 4] = (v[1] - r0.y) * f1;
                            q[grp][i + 2] = (v[2] - r1.x) * f1;
                            q[grp][i + 6] = (v[3] - r1.y) * f1;
                        }
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    qs[b][grp] = sum * (-8.0f / 16777216.0f);
                }
            }
        }

        float M[RB], l[RB], o[RB][NG][2][4];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            M[rb] = kNoRef;
            l[rb] = 0.f;
#pragma unroll
            for (int grp = 0; grp < NG; ++grp)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[rb][grp][m][i] = 0.f;
        }

        for (int k = (int)((warp + W - ring % W) % W); k < real; k += W) {
            const uint32_t n = ring + k, slot = n % S, gen = n / S;
            if (ok) ok = mbar_wait(&full[slot], gen & 1, a.wait_ns, c.err);
            const uint8_t *gr = smem + slot * kv4_bytes(NG);
            int p0 = (w.s.g0 + w.off + k) * kKv4Granule;
            const bool seen = ok && valid[slot];
            if (!seen) p0 = 0x40000000;  // nothing of it is visible
            const bool edge = p0 + 15 > at_lo || (a.window > 0 && p0 <= at_hi - a.window);

            // scores
            float sc[RB][4];
#pragma unroll
            for (int n8 = 0; n8 < 2; ++n8) {
                uint32_t kw[NG], k0[(NG + 1) / 2], k1[(NG + 1) / 2];
                load_piece<4 * NG>(kw, gr + (8 * n8 + kv4_token(g)) * kv4_row(NG) + t * 4 * NG);
                load_piece<2 * NG>(k0, gr + kv4_ks(NG) + (8 * n8 + t) * 2 * NG);
                load_piece<2 * NG>(k1, gr + kv4_ks(NG) + (8 * n8 + 4 + (t ^ 1)) * 2 * NG);
                float s0[RB], s1[RB];
#pragma unroll
                for (int grp = 0; grp < NG; ++grp) {
                    const uint32_t x = kw[grp], y = x >> 8;
                    const float f0 = piece_bf16(k0, grp), f1 = piece_bf16(k1, grp);
#pragma unroll
                    for (int m = 0; m < C::MT; ++m) {
                        const int b0 = 2 * m, b1 = 2 * m + 1;
                        const bool two = b1 < NB;
                        float d[4];
                        const float c1 = two ? qs[two ? b1 : b0][grp] : 0.f;
                        mma_f16(d, qf[b0][2 * grp][0], two ? qf[two ? b1 : b0][2 * grp][0] : 0u,
                                qf[b0][2 * grp][1], two ? qf[two ? b1 : b0][2 * grp][1] : 0u,
                                x & 0x000f000fu, y & 0x000f000fu, qs[b0][grp], qs[b0][grp], c1, c1);
                        mma_f16(d, qf[b0][2 * grp + 1][0], two ? qf[two ? b1 : b0][2 * grp + 1][0] : 0u,
                                qf[b0][2 * grp + 1][1], two ? qf[two ? b1 : b0][2 * grp + 1][1] : 0u,
                                x & 0x00f000f0u, y & 0x00f000f0u, d[0], d[1], d[2], d[3]);
                        if (SPLIT) {
                            s0[m] = grp ? fmaf(d[0] + d[2], f0, s0[m]) : (d[0] + d[2]) * f0;
                            s1[m] = grp ? fmaf(d[1] + d[3], f1, s1[m]) : (d[1] + d[3]) * f1;
                        } else {
                            s0[0] = grp ? fmaf(d[0], f0, s0[0]) : d[0] * f0;
                            s1[0] = grp ? fmaf(d[1], f1, s1[0]) : d[1] * f1;
                            if (RB == 2) {
                                s0[RB - 1] = grp ? fmaf(d[2], f0, s0[RB - 1]) : d[2] * f0;
                                s1[RB - 1] = grp ? fmaf(d[3], f1, s1[RB - 1]) : d[3] * f1;
                            }
                        }
                    }
                }
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    sc[rb][2 * n8] = s0[rb] * cs[rb];
                    sc[rb][2 * n8 + 1] = s1[rb] * cs[rb];
                }
            }

            // value scales of the lane's four tokens, and what they add to the reference
            uint32_t vs[4][(NG + 1) / 2];
            float ls[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                load_piece<2 * NG>(vs[j], gr + kv4_vs(NG) + (8 * (j >> 1) + (j & 1 ? 4 + (t ^ 1) : t)) * 2 * NG);
                float top = piece_bf16(vs[j], 0);
#pragma unroll
                for (int grp = 1; grp < NG; ++grp) top = fmaxf(top, piece_bf16(vs[j], grp));
                ls[j] = fmaxf(log2_fast(top), -100.f);
            }
            if (edge) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int p = p0 + 8 * (j >> 1) + (j & 1 ? 4 + (t ^ 1) : t);
                    bool any = false;
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        const bool vis = p <= at[rb] && (a.window == 0 || p > at[rb] - a.window);
                        if (!vis) sc[rb][j] = -INFINITY;
                        any |= vis;
                    }
                    if (!any) {
                        ls[j] = 0.f;
#pragma unroll
                        for (int i = 0; i < (NG + 1) / 2; ++i) vs[j][i] = 0u;
                    }
                }
            }
            // raise the reference where a weight would pass 2^14
            bool raise = false;
            float cand[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                cand[rb] = fmaxf(fmaxf(sc[rb][0] + ls[0], sc[rb][1] + ls[1]),
                                 fmaxf(sc[rb][2] + ls[2], sc[rb][3] + ls[3]));
                raise |= cand[rb] > M[rb] + 14.f;
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    float cd = cand[rb];
                    cd = fmaxf(cd, __shfl_xor_sync(0xffffffffu, cd, 1));
                    cd = fmaxf(cd, __shfl_xor_sync(0xffffffffu, cd, 2));
                    const float mn = cd > M[rb] + 14.f ? cd - 6.f : M[rb];
                    const float f = exp2_fast(M[rb] - mn);
                    M[rb] = mn;
                    l[rb] *= f;
                    const float fa = __shfl_sync(0xffffffffu, f, 8 * t), fb = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
                    for (int grp = 0; grp < NG; ++grp)
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            o[rb][grp][m][0] *= fa;
                            o[rb][grp][m][1] *= fb;
                            o[rb][grp][m][2] *= fa;
                            o[rb][grp][m][3] *= fb;
                        }
                }
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[rb][j] = exp2_fast(sc[rb][j] - M[rb]);
                l[rb] += (sc[rb][0] + sc[rb][1]) + (sc[rb][2] + sc[rb][3]);
            }

            // values
            uint32_t vw[4][(NG + 1) / 2];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                load_piece<2 * NG>(vw[j], gr + kv4_v(NG) + (8 * (j >> 1) + (j & 1 ? 4 + (t ^ 1) : t)) * kv4_row(NG) +
                                              (g ^ ((t & 2) << 1)) * 2 * NG);
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[slot]);
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
                uint32_t e0[4], e1[4];
                value_codes(e0, vw[0], vw[1], grp);
                value_codes(e1, vw[2], vw[3], grp);
                const float f[4] = {piece_bf16(vs[0], grp), piece_bf16(vs[1], grp), piece_bf16(vs[2], grp),
                                    piece_bf16(vs[3], grp)};
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    float p[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        p[j] = sc[rb][j] * f[j];
                        // the other row block may see a value that is not finite
                        if (RB > 1 && sc[rb][j] == 0.f) p[j] = 0.f;
                    }
                    const uint32_t h0 = pack_f16(p[0], p[1]), h1 = pack_f16(p[2], p[3]);
                    float *o0 = o[rb][grp][0], *o1 = o[rb][grp][1];
                    mma_f16(o[rb][grp][0], e0[0], e0[2], e1[0], e1[2], h0, h1, o0[0], o0[1], o0[2], o0[3]);
                    mma_f16(o[rb][grp][1], e0[1], e0[3], e1[1], e1[3], h0, h1, o1[0], o1[1], o1[2], o1[3]);
                    if (SPLIT) {
                        const float2 r0 = __half22float2(*reinterpret_cast<const __half2 *>(&h0));
                        const float2 r1 = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
                        const uint32_t x0 = pack_f16(p[0] - r0.x, p[1] - r0.y);
                        const uint32_t x1 = pack_f16(p[2] - r1.x, p[3] - r1.y);
                        mma_f16(o[rb][grp][0], e0[0], e0[2], e1[0], e1[2], x0, x1, o0[0], o0[1], o0[2], o0[3]);
                        mma_f16(o[rb][grp][1], e0[1], e0[3], e1[1], e1[3], x0, x1, o1[0], o1[1], o1[2], o1[3]);
                    }
                }
            }
        }
        ring += real;

        // ---- the item's end: merge the warps
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            l[rb] += __shfl_xor_sync(0xffffffffu, l[rb], 1);
            l[rb] += __shfl_xor_sync(0xffffffffu, l[rb], 2);
            if (t == 0) {
                wm[warp][8 * rb + g] = M[rb];
                wl[warp][8 * rb + g] = l[rb];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float *row = mo + (warp * C::kRows + 8 * rb + 2 * t + i) * C::kStride + 4 * g;
#pragma unroll
                for (int grp = 0; grp < NG; ++grp)
                    *reinterpret_cast<float4 *>(row + 32 * grp) =
                        make_float4(o[rb][grp][0][i], o[rb][grp][1][i], o[rb][grp][0][2 + i], o[rb][grp][1][2 + i]);
            }
        }
        named_sync(1, 32 * W);
        const bool begins = w.off == 0, ends = w.off + take == units;
        const bool whole = begins && ends;
        const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
        if (tid < C::kRows) {
            float mx = kNoRef, L = 0.f;
            for (int x = 0; x < W; ++x) mx = fmaxf(mx, wm[x][tid]);
            for (int x = 0; x < W; ++x) {
                const float f = exp2_fast(wm[x][tid] - mx);
                fac[x][tid] = f;
                L += f * wl[x][tid];
            }
            suml[tid] = L;
            if (!whole) {
                float *st = a.part + (size_t)2 * gridDim.x * C::kRows * C::kCh + (size_t)(slot * C::kRows + tid) * 2;
                st[0] = mx;
                st[1] = L;
            }
        }
        named_sync(1, 32 * W);
        auto row_at = [&](int r) {
            const int rho = rho0 + r;
            return (int64_t)(w.s.row0 + rho / G) * a.os + (int64_t)(kvh * G + rho % G) * c.hd;
        };
        for (int i = tid; i < R * (C::kCh / 4); i += 32 * W) {
            const int r = i / (C::kCh / 4), ch = 4 * (i % (C::kCh / 4));
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < W; ++x) {
                const float4 p = *reinterpret_cast<const float4 *>(mo + (x * C::kRows + r) * C::kStride + ch);
                const float f = fac[x][r];
                v[0] = fmaf(p.x, f, v[0]);
                v[1] = fmaf(p.y, f, v[1]);
                v[2] = fmaf(p.z, f, v[2]);
                v[3] = fmaf(p.w, f, v[3]);
            }
            if (!whole) {
                __stcg(reinterpret_cast<float4 *>(a.part + ((size_t)slot * C::kRows + r) * C::kCh + ch),
                       make_float4(v[0], v[1], v[2], v[3]));
            } else if (ch < c.hd) {
                const float inv = suml[r] != 0.f ? 1.0f / suml[r] : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] *= inv;
                store4(a, row_at(r) + ch, v, min(4, c.hd - ch));
            }
        }
        if (!whole) {
            // the runs of this item: `first` begins it, the others continue it
            const int64_t start = u - w.off;
            const int first = kv4_run_of(start, total, parts), final = kv4_run_of(start + units - 1, total, parts);
            __threadfence();
            named_sync(1, 32 * W);
            if (tid == 0) {
                const unsigned n = atomicAdd(a.count + first, 1u);
                last_in = n == (unsigned)(final - first);
                if (last_in) a.count[first] = 0u;  // ready for the next call
            }
            named_sync(1, 32 * W);
            if (last_in) {
                __threadfence();
                const float *stats = a.part + (size_t)2 * gridDim.x * C::kRows * C::kCh;
                for (int i = tid; i < R * (C::kCh / 4); i += 32 * W) {
                    const int r = i / (C::kCh / 4), ch = 4 * (i % (C::kCh / 4));
                    float mx = kNoRef, L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                    for (int b = first; b <= final; ++b)
                        mx = fmaxf(mx, __ldcg(stats + (size_t)((2 * b + (b == first)) * C::kRows + r) * 2));
#pragma unroll 4
                    for (int b = first; b <= final; ++b) {
                        const size_t s = (size_t)(2 * b + (b == first)) * C::kRows + r;
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(stats + 2 * s));
                        const float4 p = __ldcg(reinterpret_cast<const float4 *>(a.part + s * C::kCh + ch));
                        const float f = exp2_fast(ml.x - mx);
                        L = fmaf(ml.y, f, L);
                        v[0] = fmaf(p.x, f, v[0]);
                        v[1] = fmaf(p.y, f, v[1]);
                        v[2] = fmaf(p.z, f, v[2]);
                        v[3] = fmaf(p.w, f, v[3]);
                    }
                    if (ch < c.hd) {
                        const float inv = L != 0.f ? 1.0f / L : 0.f;
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] *= inv;
                        store4(a, row_at(r) + ch, v, min(4, c.hd - ch));
                    }
                }
            }
        }
        named_sync(1, 32 * W);  // the merge buffers may be written again
        more = advance(u, take);
    }
}

}  // namespace rb
