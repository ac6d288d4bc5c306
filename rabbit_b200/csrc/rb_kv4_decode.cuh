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
// The arithmetic of a granule, on m16n8k16 fp16 instructions with fp32 sums.
// Lane (g, t):
//  * S^T = K Q^T: rows are the granule's 16 tokens, columns 8 query rows. K's
//    nibbles u = code + 8 go in as the fp16 numbers u 2^-24 (a nibble in the low
//    mantissa bits is one: a mask, no conversion) and 16 u 2^-24 (the next
//    nibble; those channels of Q are a sixteenth). Each group's sum has its
//    bias, 8 2^-24 sum Q, taken off and is scaled in fp32. Q is scaled by a
//    power of two per row into fp16's upper range: exact for 16-bit queries.
//    fp32 queries (SPLIT) go in two terms of 11 bits, with K's codes signed: the
//    instruction truncates its sums, and without the bias they are smaller.
//  * O^T = V^T P^T: rows are channels, columns query rows. Each group's weights
//    are p s, s the value scale, rounded to fp16 (SPLIT: two terms) and turned
//    from S^T's layout into the operand's by a transpose per 8 x 8 pairs.
//  * p = 2^(x - M) with M a running reference of the row such that every weight is
//    at most 2^14 in fp16 and the largest are far above its subnormals. M is
//    raised only when a weight would pass 2^14, to weights of at most 2^6: after
//    the first granules that is rare, and the output is rescaled only then.
#pragma once
#include "rb_device.cuh"
#include "rb_kv4_attn.cuh"
#include "rb_types.cuh"

namespace rb {

constexpr int kDecodeMaxGrid = 320;  // CTAs of a launch at most
constexpr float kNoRef = -3e38f;  // M before any visible token

template <int NG, int RB, bool SPLIT>
struct DecodeCfg {
    // CTAs per SM, and consumer warps: with the producer two CTAs of 8 warps of
    // 128 registers a thread, or where the output takes more one of 12 of 168, or
    // of 8 of 255
    static constexpr int kCtas = NG * RB <= 4 ? 2 : 1;
    static constexpr int W = kCtas == 1 && NG <= 4 ? 11 : 7;
    static constexpr int D = 4;                      // ring slots of a warp
    static constexpr int kThreads = 32 * (W + 1);
    static constexpr int kRows = 8 * RB;
    static constexpr int kCh = 32 * NG;
    static constexpr int kStride = kCh + 4;          // merge rows: spreads a quarter warp over the banks
    static constexpr int NT = SPLIT ? 2 : 1;         // terms of a query
    static constexpr size_t kRing = (size_t)W * D * kv4_bytes(NG);
    // merge rows of the warps; also (factor, sum) pairs of an item's pieces, one a run
    static constexpr size_t kPairs = sizeof(float2) * (size_t)kRows * kDecodeMaxGrid;
    static constexpr size_t kRows32 = sizeof(float) * (size_t)W * kRows * kStride;
    static constexpr size_t kMerge = kRows32 > kPairs ? kRows32 : kPairs;
    static constexpr size_t kQuery = 16 * (size_t)RB * NG * (32 * NT + 4);  // operands, bias
    static constexpr size_t kSmem = kRing + kMerge + kQuery;
};

// A run's share of one item, from the producer to the consumers.
struct DecodeStep {
    int granules;             // real ones of the share
    int p0;                   // position of the first
    int rho0, rows, kvh;      // row tile, KV head
    int row0, at0;            // sequence's first query row, and its position
    int from, whole, slot;    // place of a partial result
    int first, last, more;
};
constexpr int kSteps = 4;

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

// Barrier among `threads` threads; whether `ok` held for all of them.
__device__ __forceinline__ bool named_all(int id, int threads, bool ok) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)ok), "r"(id), "r"(threads)
        : "memory");
    return r != 0;
}

__device__ __forceinline__ Kv4Seq load_seq(const Kv4AttnArgs &a, int i, int *bad = nullptr) {
    Kv4Seq s;
    const int s0 = a.q_start ? a.q_start[i] : i, s1 = a.q_start ? a.q_start[i + 1] : i + 1;
    const int e = kv4_seq(s0, s1, a.kv_len[i], a.T, a.max_q, (int64_t)a.max_pages * a.c.page, a.window, s);
    if (bad) *bad = e;
    return s;
}

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
    constexpr int W = C::W, D = C::D, NT = C::NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[W * D], empty[W * D], step_full[kSteps], step_empty[kSteps];
    __shared__ uint8_t valid[W * D];
    __shared__ DecodeStep steps[kSteps];
    __shared__ int64_t warp_sums[C::kThreads / 32];
    __shared__ int64_t found_before;
    __shared__ int found_seq;
    __shared__ float wm[W][C::kRows], wl[W][C::kRows];
    __shared__ float fac[W][C::kRows], suml[C::kRows];
    __shared__ bool last_in;
    launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < W * D; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < kSteps; ++i) {
            mbar_init(&step_full[i], 1);
            mbar_init(&step_empty[i], W);
        }
        mbar_init_fence();
    }
    wait_prerequisite();
    const Kv4View &c = a.c;
    const int G = a.nh / c.nkv;

    // ---- this CTA's run of units
    int64_t mine = 0, total;
    for (int i = tid; i < a.n_seqs; i += C::kThreads) {
        int bad;
        const Kv4Seq s = load_seq(a, i, &bad);
        if (bad && blockIdx.x == 0) atomicOr(c.err, bad);
        mine += kv4_cost(s, G, C::kRows, c.nkv);
    }
    const int64_t excl = block_scan<C::kThreads>(mine, warp_sums, total);
    if (total == 0) return;
    const int64_t parts = kv4_parts(total, gridDim.x);
    if (blockIdx.x >= parts) return;
    const int64_t u0 = kv4_cut(blockIdx.x, total, parts);
    if (a.n_seqs <= C::kThreads) {
        if (mine > 0 && excl <= u0 && u0 < excl + mine) {
            found_seq = tid;
            found_before = excl;
        }
    } else {
        int64_t base = 0;
        for (int i0 = 0; i0 < a.n_seqs && base <= u0; i0 += C::kThreads) {
            const int i = i0 + tid;
            const int64_t cost = i < a.n_seqs ? kv4_cost(load_seq(a, i), G, C::kRows, c.nkv) : 0;
            int64_t all;
            const int64_t before = base + block_scan<C::kThreads>(cost, warp_sums, all);
            if (cost > 0 && before <= u0 && u0 < before + cost) {
                found_seq = i;
                found_before = before;
            }
            base += all;
        }
    }
    __syncthreads();

    if (warp == W) {
        // ---- producer: the run's steps, and their granules into the warps' rings
        const uint64_t policy = policy_evict_first();
        const int64_t u1 = kv4_cut(blockIdx.x + 1, total, parts);
        int seq = found_seq;
        Kv4Seq s = load_seq(a, seq);
        int64_t u = u0;
        int item = kv4_granules(s) + kKv4Fixed, sub = (int)((u0 - found_before) / item),
            off = (int)((u0 - found_before) % item);
        int ring = 0;  // warp that takes the step's first granule
        int issued = 0, slot = 0, phase = 0;  // lane w: granules issued (D at most), warp w's next slot, its round
        bool ok = true, more = true;
        for (int step = 0; more && ok;) {
            const Kv4Share sh = kv4_share(s, off, u, u1, total, parts);
            const Kv4Seq now = s;
            const int now_seq = seq, now_sub = sub;
            u += item - off;
            off = 0;
            more = u < u1;
            if (more && ++sub >= kv4_items(s, G, C::kRows, c.nkv)) {
                sub = 0;
                do s = load_seq(a, ++seq);
                while (s.nq == 0);
                item = kv4_granules(s) + kKv4Fixed;
            }
            // the item that a run ends in may have no share of it
            if (more && u1 - u <= kKv4Fixed) more = false;
            if (sh.take == 0) continue;
            const int real = now.n > 0 ? sh.take : 0, head = now_sub % c.nkv;
            const int d = step % kSteps;
            if (step >= kSteps) ok = mbar_wait(&step_empty[d], (step / kSteps - 1) & 1, a.wait_ns, c.err, 0);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (lane == 0) {
                DecodeStep &t = steps[d];
                t.granules = real;
                t.p0 = (now.g0 + sh.from) * kKv4Granule;
                t.rho0 = now_sub / c.nkv * C::kRows;
                t.rows = min(C::kRows, now.nq * G - t.rho0);
                t.kvh = head;
                t.row0 = now.row0;
                t.at0 = now.len - now.nq;
                t.from = sh.from;
                t.whole = sh.begins && sh.ends;
                t.slot = 2 * blockIdx.x + (sh.begins ? 1 : 0);
                t.first = sh.first;
                t.last = sh.last;
                t.more = more;
                mbar_arrive(&step_full[d]);
            }
            ++step;
            // lane w serves consumer warp w, whenever a slot of that warp is free
            int k = lane < W ? (lane + W - ring) % W : real;
            const uint8_t *from = nullptr;
            auto look_up = [&]() {
                from = nullptr;
                if (k >= real) return;
                const int pos = (now.g0 + sh.from + k) * kKv4Granule, pi = pos / c.page;
                const int page = a.table[(int64_t)now_seq * a.max_pages + pi];
                if (page >= 0 && page < c.n_pages)
                    from = c.base + (size_t)page * c.page_bytes() + (size_t)head * c.head_bytes() +
                           (size_t)((pos - pi * c.page) / kKv4Granule) * kv4_bytes(NG);
                else
                    atomicOr(c.err, RB_KV4_ERR_PAGE);
            };
            look_up();
            for (uint64_t t0 = 0;;) {
                const bool ready = k < real && (issued < D || mbar_test(&empty[lane * D + slot], (phase ^ 1) & 1));
                if (ready) {
                    const int at = lane * D + slot;
                    valid[at] = from != nullptr;
                    if (from) {
                        mbar_arrive_expect_tx(&full[at], kv4_bytes(NG));
                        bulk_g2s(smem + at * kv4_bytes(NG), from, kv4_bytes(NG), &full[at], policy);
                    } else {
                        mbar_arrive(&full[at]);
                    }
                    if (issued < D) ++issued;
                    if (++slot == D) {
                        slot = 0;
                        phase ^= 1;
                    }
                    k += W;
                    look_up();
                }
                if (!__any_sync(0xffffffffu, k < real)) break;
                if (__any_sync(0xffffffffu, ready)) {
                    t0 = 0;
                } else {
                    if (t0 == 0) t0 = globaltimer_ns();
                    __nanosleep(100);
                    if (globaltimer_ns() - t0 > a.wait_ns) {
                        if (lane == 0) set_error(c.err, RB_ERR_TIMEOUT);
                        ok = false;
                        break;
                    }
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            ring = (ring + real) % W;
        }
        // after a wait that ran out: copies in flight end before the CTA does
        if (!ok)
            for (int i = lane; i < W * D; i += 32)
                for (int ph = 0; ph < 2; ++ph) mbar_wait(&full[i], ph, a.wait_ns, nullptr, 0);
        return;
    }

    // ---- consumers
    const int g = lane >> 2, t = lane & 3;
    float *mo = reinterpret_cast<float *>(smem + C::kRing);  // [W][rows][kStride]
    uint4 *qop = reinterpret_cast<uint4 *>(smem + C::kRing + C::kMerge);  // [RB][NT][NG][32 lanes]
    float4 *bias = reinterpret_cast<float4 *>(qop + RB * NT * NG * 32);   // [RB][NG][4 t]
    const uint8_t *own = smem + warp * D * kv4_bytes(NG);  // this warp's slots
    int next = warp;        // granules of the coming steps before this warp's next one
    int j = 0, phase = 0;   // its slot
    bool ok = true;
    for (int step = 0;; ++step) {
        const DecodeStep &st = steps[step % kSteps];
        if (ok) ok = mbar_wait(&step_full[step % kSteps], (step / kSteps) & 1, a.wait_ns, c.err);
        if (!named_all(2, 32 * W, ok)) break;  // a wait ran out: all warps leave together
        const int real = st.granules, R = st.rows, rho0 = st.rho0, kvh = st.kvh;
        const int at_lo = st.at0 + rho0 / G, at_hi = st.at0 + (rho0 + R - 1) / G;

        // The item's query operands, a group a warp, into shared memory: for lane
        // (g, t) row g's channels (nibbles 0, 4 | 2, 6 | 1, 5 | 3, 7 of word t of the
        // group); for rows 2 t, 2 t + 1 the bias their columns start from. In
        // registers stays what turns those columns' sums into powers of two.
        float cs[RB][2];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int rho = rho0 + 8 * rb + g, qi = rho / G;
            const bool in = 8 * rb + g < R;
            const int64_t base = (int64_t)(st.row0 + qi) * a.qs + (int64_t)(kvh * G + rho - qi * G) * c.hd;
            float top = 0.f;
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
                float q[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (in && 32 * grp + 8 * t < c.hd) load_q8(a, base + 32 * grp + 8 * t, q);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(q[i]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^(14 - e), 2^e <= top: the largest goes to [2^14, 2^15)
            const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100);
            const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
            const float down = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
            const float sup = a.scale < 0.f ? -up : up;
            const float c1 = fabsf(a.scale) * down * (SPLIT ? 1.0f : 16777216.0f);
            cs[rb][0] = __shfl_sync(0xffffffffu, c1, 8 * t);
            cs[rb][1] = __shfl_sync(0xffffffffu, c1, 8 * t + 4);
            for (int grp = warp; grp < NG; grp += W) {
                float q[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
                if (in && 32 * grp + 8 * t < c.hd) load_q8(a, base + 32 * grp + 8 * t, q);
                uint32_t f[NT][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {  // the instruction's two steps
                    const float by = !SPLIT && i ? 0.0625f : 1.0f, back = !SPLIT && i ? 16.f : 1.0f;
                    float v[4] = {q[i], q[i + 4], q[i + 2], q[i + 6]};
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] *= sup * by;
#pragma unroll
                    for (int term = 0; term < NT; ++term) {
                        const uint32_t x0 = pack_f16(v[0], v[1]), x1 = pack_f16(v[2], v[3]);
                        f[term][2 * i] = x0;
                        f[term][2 * i + 1] = x1;
                        const float2 r0 = __half22float2(*reinterpret_cast<const __half2 *>(&x0));
                        const float2 r1 = __half22float2(*reinterpret_cast<const __half2 *>(&x1));
                        sum += ((r0.x + r0.y) + (r1.x + r1.y)) * back;
                        v[0] -= r0.x;  // what this term leaves to the next
                        v[1] -= r0.y;
                        v[2] -= r1.x;
                        v[3] -= r1.y;
                    }
                }
#pragma unroll
                for (int term = 0; term < NT; ++term)
                    qop[((rb * NT + term) * NG + grp) * 32 + lane] =
                        make_uint4(f[term][0], f[term][1], f[term][2], f[term][3]);
                if constexpr (!SPLIT) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    sum *= -8.0f / 16777216.0f;
                    const float s0 = __shfl_sync(0xffffffffu, sum, 8 * t), s1 = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
                    if (g == 0) bias[(rb * NG + grp) * 4 + t] = make_float4(s0, s1, s0, s1);
                }
            }
        }
        named_sync(1, 32 * W);

        float M[RB][2], l[RB][2], o[RB][NG][2][4];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            M[rb][0] = M[rb][1] = kNoRef;
            l[rb][0] = l[rb][1] = 0.f;
#pragma unroll
            for (int grp = 0; grp < NG; ++grp)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[rb][grp][m][i] = 0.f;
        }

        // Two granules are under way in a warp: the scores of one and the output of
        // the one before it are independent, in one stretch of code without a
        // branch, so one's instructions fill the other's waits.
        const int tok = kv4_token(g);
        constexpr int NW = (NG + 1) / 2;
        struct Scores {
            float sc[RB][4];           // tokens tok, tok + 8; query rows 2 t, 2 t + 1
            uint32_t v0[NW], v1[NW];   // the tokens' value scales
        };
        // the granule in slot j, when it is there; its validity
        auto arrived = [&]() -> bool {
            if (ok) ok = mbar_wait(&full[warp * D + j], phase, a.wait_ns, c.err);
            return ok && valid[warp * D + j];
        };
        auto score = [&](const uint8_t *gr, Scores &s) {
            uint32_t k0[NG], k1[NG], s0[NW], s1[NW];
            load_piece<4 * NG>(k0, gr + tok * kv4_row(NG) + t * 4 * NG);
            load_piece<4 * NG>(k1, gr + (tok + 8) * kv4_row(NG) + t * 4 * NG);
            load_piece<2 * NG>(s0, gr + kv4_ks(NG) + tok * 2 * NG);
            load_piece<2 * NG>(s1, gr + kv4_ks(NG) + (tok + 8) * 2 * NG);
            load_piece<2 * NG>(s.v0, gr + kv4_vs(NG) + tok * 2 * NG);
            load_piece<2 * NG>(s.v1, gr + kv4_vs(NG) + (tok + 8) * 2 * NG);
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
                uint32_t e0[4], e1[4];
                key_codes<SPLIT>(e0, k0[grp]);
                key_codes<SPLIT>(e1, k1[grp]);
                const float f0 = piece_bf16(s0, grp), f1 = piece_bf16(s1, grp);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    float d[4];
#pragma unroll
                    for (int term = NT - 1; term >= 0; --term) {  // the small term first
                        const uint4 b = qop[((rb * NT + term) * NG + grp) * 32 + lane];
                        if (SPLIT && term == NT - 1) {
                            mma_f16(d, e0[0], e1[0], e0[1], e1[1], b.x, b.y, 0.f, 0.f, 0.f, 0.f);
                        } else if (!SPLIT) {
                            const float4 c0 = bias[(rb * NG + grp) * 4 + t];
                            mma_f16(d, e0[0], e1[0], e0[1], e1[1], b.x, b.y, c0.x, c0.y, c0.z, c0.w);
                        } else {
                            mma_f16(d, e0[0], e1[0], e0[1], e1[1], b.x, b.y, d[0], d[1], d[2], d[3]);
                        }
                        mma_f16(d, e0[2], e1[2], e0[3], e1[3], b.z, b.w, d[0], d[1], d[2], d[3]);
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float f = x < 2 ? f0 : f1;
                        s.sc[rb][x] = grp ? fmaf(d[x], f, s.sc[rb][x]) : d[x] * f;
                    }
                }
            }
        };
        // what only some granules need: masks at the ends of what a row sees, and a
        // higher reference
        auto settle = [&](Scores &s, int p0, bool there) {
            const bool edge = !there || p0 + kKv4Granule - 1 > at_lo || (a.window > 0 && p0 <= at_hi - a.window);
            // the lane's largest value scale, in a half each (positive: in order as integers)
            uint32_t vmax = 0;
#pragma unroll
            for (int i = 0; i < NW; ++i) vmax = __vmaxu2(vmax, __vmaxu2(s.v0[i], s.v1[i]));
            vmax = max(vmax << 16, vmax & 0xffff0000u);
            // a bound with it first, each token's own scale only where that one fails
            const float vtop = fmaxf(log2_fast(__uint_as_float(vmax)), -100.f);
            bool odd = edge || vmax >= 0x7f800000u;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    odd |= fmaf(fmaxf(s.sc[rb][i], s.sc[rb][2 + i]), cs[rb][i], vtop) > M[rb][i] + 14.f;
            if (!__any_sync(0xffffffffu, odd)) return;
            if (edge) {
                auto sees = [&](int r, int p) {  // tile row r, position p
                    const int at = st.at0 + (rho0 + r) / G;
                    return there && r < R && p <= at && (a.window == 0 || p > at - a.window);
                };
                // Value scales of tokens that no row sees may be anything, and one that
                // only some rows see may be NaN: it makes those rows' channels NaN and
                // has no part in the products.
                if (__any_sync(0xffffffffu, vmax >= 0x7f800000u))
#pragma unroll 1
                    for (int x = 0; x < kKv4Granule; ++x)
#pragma unroll
                        for (int grp = 0; grp < NG; ++grp) {
                            const uint32_t own16 = (x < 8 ? s.v0[grp >> 1] : s.v1[grp >> 1]) >> (16 * (grp & 1)) & 0xffffu;
                            if (__shfl_sync(0xffffffffu, own16, 4 * (x & 7)) < 0x7f80u) continue;
                            const int p = p0 + kv4_token(x & 7) + (x & 8);
#pragma unroll
                            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                                for (int i = 0; i < 2; ++i)
                                    if (sees(8 * rb + 2 * t + i, p))
#pragma unroll
                                        for (int m = 0; m < 2; ++m)
                                            o[rb][grp][m][i] = o[rb][grp][m][2 + i] = __uint_as_float(0x7fc00000u);
                            if (g == (x & 7)) {
                                const uint32_t keep = grp & 1 ? 0xffffu : 0xffff0000u;
                                if (x < 8) s.v0[grp >> 1] &= keep;
                                else s.v1[grp >> 1] &= keep;
                            }
                        }
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
                        if (!sees(8 * rb + 2 * t + (x & 1), p0 + tok + 8 * (x >> 1))) s.sc[rb][x] = -INFINITY;
            }
            float top0 = piece_bf16(s.v0, 0), top1 = piece_bf16(s.v1, 0);
#pragma unroll
            for (int grp = 1; grp < NG; ++grp) {
                top0 = fmaxf(top0, piece_bf16(s.v0, grp));
                top1 = fmaxf(top1, piece_bf16(s.v1, grp));
            }
            top0 = fmaxf(log2_fast(top0), -100.f);
            top1 = fmaxf(log2_fast(top1), -100.f);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float cd = fmaxf(fmaf(s.sc[rb][i], cs[rb][i], top0), fmaf(s.sc[rb][2 + i], cs[rb][i], top1));
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) cd = fmaxf(cd, __shfl_xor_sync(0xffffffffu, cd, x));
                    const float mn = cd > M[rb][i] + 14.f ? cd - 6.f : M[rb][i];
                    const float f = exp2_fast(M[rb][i] - mn);
                    M[rb][i] = mn;
                    l[rb][i] *= f;
#pragma unroll
                    for (int grp = 0; grp < NG; ++grp)
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            o[rb][grp][m][i] *= f;
                            o[rb][grp][m][2 + i] *= f;
                        }
                }
        };
        auto output = [&](const uint8_t *gr, Scores &s, int slot) {
            // values: tokens 2 t, 2 t + 1 of the tile's order, channels 4 g .. 4 g + 3
            uint32_t vw[4][NW];
#pragma unroll
            for (int x = 0; x < 4; ++x)
                load_piece<2 * NG>(vw[x], gr + kv4_v(NG) + (8 * (x >> 1) + (x & 1 ? 4 + (t ^ 1) : t)) * kv4_row(NG) +
                                              (g ^ ((t & 2) << 1)) * 2 * NG);
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[slot]);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    s.sc[rb][x] = exp2_fast(fmaf(s.sc[rb][x], cs[rb][x & 1], -M[rb][x & 1]));
                l[rb][0] += s.sc[rb][0] + s.sc[rb][2];
                l[rb][1] += s.sc[rb][1] + s.sc[rb][3];
            }
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
                uint32_t e0[4], e1[4];
                value_codes(e0, vw[0], vw[1], grp);
                value_codes(e1, vw[2], vw[3], grp);
                const float f[2] = {piece_bf16(s.v0, grp), piece_bf16(s.v1, grp)};
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    // weights, turned into the operand of rows g: tokens 2 t, 2 t + 1
                    uint32_t h[2 * NT];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float u = s.sc[rb][2 * n] * f[n], v = s.sc[rb][2 * n + 1] * f[n];
                        const uint32_t w = pack_f16(u, v);
                        h[n] = transpose8(w);
                        if constexpr (SPLIT) {
                            const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&w));
                            h[2 + n] = transpose8(pack_f16(u - r.x, v - r.y));
                        }
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        float *acc = o[rb][grp][m];
                        if constexpr (SPLIT) {
                            // the sum in fp32 outside: the instruction truncates what it adds to
                            float d[4];
                            mma_f16(d, e0[m], e0[m + 2], e1[m], e1[m + 2], h[2], h[3], 0.f, 0.f, 0.f, 0.f);
                            mma_f16(d, e0[m], e0[m + 2], e1[m], e1[m + 2], h[0], h[1], d[0], d[1], d[2], d[3]);
#pragma unroll
                            for (int x = 0; x < 4; ++x) acc[x] += d[x];
                        } else {
                            mma_f16(o[rb][grp][m], e0[m], e0[m + 2], e1[m], e1[m + 2], h[0], h[1], acc[0], acc[1],
                                    acc[2], acc[3]);
                        }
                    }
                }
            }
        };
        auto to_next_slot = [&]() {
            if (++j == D) {
                j = 0;
                phase ^= 1;
            }
        };
        if (next < real) {
            Scores cur;
            const bool there = arrived();
            score(own + j * kv4_bytes(NG), cur);
            settle(cur, st.p0 + next * kKv4Granule, there);
            for (next += W; next < real; next += W) {
                const int before = j;
                to_next_slot();
                const bool it_there = arrived();
                Scores nxt;
                score(own + j * kv4_bytes(NG), nxt);
                output(own + before * kv4_bytes(NG), cur, warp * D + before);
                settle(nxt, st.p0 + next * kKv4Granule, it_there);
                cur = nxt;
            }
            output(own + j * kv4_bytes(NG), cur, warp * D + j);
            to_next_slot();
        }
        next -= real;

        // ---- the share's end: merge the warps
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int s = 4; s < 32; s <<= 1) l[rb][i] += __shfl_xor_sync(0xffffffffu, l[rb][i], s);
                if (g == 0) {
                    wm[warp][8 * rb + 2 * t + i] = M[rb][i];
                    wl[warp][8 * rb + 2 * t + i] = l[rb][i];
                }
                float *row = mo + (warp * C::kRows + 8 * rb + 2 * t + i) * C::kStride + 4 * g;
#pragma unroll
                for (int grp = 0; grp < NG; ++grp)
                    *reinterpret_cast<float4 *>(row + 32 * grp) =
                        make_float4(o[rb][grp][0][i], o[rb][grp][1][i], o[rb][grp][0][2 + i], o[rb][grp][1][2 + i]);
            }
        named_sync(1, 32 * W);
        const bool whole = st.whole;
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
                float *p = a.part + (size_t)2 * gridDim.x * C::kRows * C::kCh + (size_t)(st.slot * C::kRows + tid) * 2;
                p[0] = mx;
                p[1] = L;
            }
        }
        named_sync(1, 32 * W);
        auto row_at = [&](int r) {
            const int rho = rho0 + r, qi = rho / G;
            return (int64_t)(st.row0 + qi) * a.os + (int64_t)(kvh * G + rho - qi * G) * c.hd;
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
                __stcg(reinterpret_cast<float4 *>(a.part + ((size_t)st.slot * C::kRows + r) * C::kCh + ch),
                       make_float4(v[0], v[1], v[2], v[3]));
            } else if (ch < c.hd) {
                const float inv = suml[r] != 0.f ? 1.0f / suml[r] : 0.f;
#pragma unroll
                for (int x = 0; x < 4; ++x) v[x] *= inv;
                store4(a, row_at(r) + ch, v, min(4, c.hd - ch));
            }
        }
        if (!whole) {
            __threadfence();
            named_sync(1, 32 * W);
            if (tid == 0) {
                const unsigned n = atomicAdd(a.count + st.first, 1u);
                last_in = n == (unsigned)(st.last - st.first);
                if (last_in) a.count[st.first] = 0u;  // ready for the next call
            }
            named_sync(1, 32 * W);
            if (last_in) {
                __threadfence();
                // the pieces' factors into shared memory (the merge rows are free),
                // then their outputs, eight loads in flight a thread
                const float *stats = a.part + (size_t)2 * gridDim.x * C::kRows * C::kCh;
                const int np = st.last - st.first + 1;
                const int first = st.first;
                auto piece = [&](int b, int r) { return (size_t)(2 * (first + b) + (b == 0)) * C::kRows + r; };
                float2 *pf = reinterpret_cast<float2 *>(mo);  // [rows][np]
                for (int i = tid; i < R * np; i += 32 * W) {
                    const int r = i / np;
                    pf[i] = __ldcg(reinterpret_cast<const float2 *>(stats) + piece(i - r * np, r));
                }
                named_sync(1, 32 * W);
                for (int r = warp; r < R; r += W) {
                    float mx = kNoRef, L = 0.f;
                    for (int b = lane; b < np; b += 32) mx = fmaxf(mx, pf[r * np + b].x);
#pragma unroll
                    for (int s = 16; s; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
                    for (int b = lane; b < np; b += 32) {
                        const float f = exp2_fast(pf[r * np + b].x - mx);
                        L = fmaf(pf[r * np + b].y, f, L);
                        pf[r * np + b].x = f;
                    }
#pragma unroll
                    for (int s = 16; s; s >>= 1) L += __shfl_xor_sync(0xffffffffu, L, s);
                    if (lane == 0) suml[r] = L;
                }
                named_sync(1, 32 * W);
                for (int i = tid; i < R * (C::kCh / 4); i += 32 * W) {
                    const int r = i / (C::kCh / 4), ch = 4 * (i % (C::kCh / 4));
                    float v[4] = {0.f, 0.f, 0.f, 0.f};
                    for (int b0 = 0; b0 < np; b0 += 8) {
                        float4 p[8];
#pragma unroll
                        for (int b = 0; b < 8; ++b)
                            if (b0 + b < np)
                                p[b] = __ldcg(reinterpret_cast<const float4 *>(a.part + piece(b0 + b, r) * C::kCh + ch));
#pragma unroll
                        for (int b = 0; b < 8; ++b)
                            if (b0 + b < np) {
                                const float f = pf[r * np + b0 + b].x;
                                v[0] = fmaf(p[b].x, f, v[0]);
                                v[1] = fmaf(p[b].y, f, v[1]);
                                v[2] = fmaf(p[b].z, f, v[2]);
                                v[3] = fmaf(p[b].w, f, v[3]);
                            }
                    }
                    if (ch < c.hd) {
                        const float inv = suml[r] != 0.f ? 1.0f / suml[r] : 0.f;
#pragma unroll
                        for (int x = 0; x < 4; ++x) v[x] *= inv;
                        store4(a, row_at(r) + ch, v, min(4, c.hd - ch));
                    }
                }
            }
        }
        const bool more = st.more;
        named_sync(1, 32 * W);  // the merge buffers may be written again
        if (lane == 0) mbar_arrive(&step_empty[step % kSteps]);
        if (!more) break;
    }
}

}  // namespace rb
