// rb_kv4_decode.cuh -- attention over the 4-bit cache for few query rows a
// sequence (decoding, drafted tokens): every KV head's rows at once against a
// stream of granules.
//
// A CTA per SM walks an equal run of the batch's granules (kv4_cut), whatever
// sequences they belong to, item after item ("steps"):
//  * one warp fetches the granules into a ring in shared memory, a bulk copy
//    each, as far ahead as the ring holds, across steps;
//  * one warp makes the query operands of the next step, and merges the one
//    before;
//  * W warps take the granules in turn, with a running (reference, sum, output)
//    of the step's query rows in registers, which they leave in shared memory
//    at the step's end. The hardware favours older warps; that all share one
//    ring keeps them together, since none can be further ahead than it holds.
// An item that a run's border cuts is merged from the runs' partial results by
// whichever CTA arrives last, in the order of the runs.
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
//  * p = 2^((x - M) - D) with a running reference of the row in two parts, a score M
//    and an exponent D of values, such that every weight is at most 2^14 in fp16 and
//    the largest are far above its subnormals. It is raised only when a weight
//    would pass 2^14, to weights of at most 2^6: after the first granules that is
//    rare, and the output is rescaled only then. (In one number a score past 2^24
//    would leave no room for D. x is rounded to fp32 before M is taken off, so that
//    equal scores stay equal to their reference.)
//
// Bound by its instructions, 376 for each further granule (2304 bytes at 128 channels;
// 16-bit queries), 46 % of a launch's issue slots with its start and merge: 49 us for 1 x
// 131072 positions of 8 KV heads (3.06 TB/s, 0.47 of the measured copy rate), 61 us
// for 64 x 4096 (0.44), 195 us for 128 x 8192 (0.56). fp32 queries take two terms: 68
// us for 16 sequences of 4 rows, 6 query heads a KV head, and 2048 positions; with 16 rows
// a tile they spill 60 / 96 bytes of stores / loads at 168 registers.
//
// Range: bf16 has fp32's exponents and a query operand fp16's, so channels more than 2^24
// below their row's largest lose bits. A value's weight p s is rounded to fp16, which
// keeps its bits down to 2^-20 of the row's largest weight and is zero from 2^-31.
#pragma once
#include "rb_device.cuh"
#include "rb_kv4_attn.cuh"
#include "rb_types.cuh"

namespace rb {

constexpr int kDecodeMaxGrid = 320;  // CTAs of a launch at most
constexpr float kNoRef = -3e38f;  // M before any visible token
// A token whose value scales are below 2^-80, or all 0, counts as one of 2^-80: its weight
// p s is at most 2^14, so p at most 2^94, and 2^30 positions of such p have a finite sum.
constexpr float kLeastScale = -80.f;

template <int NG, int RB, bool SPLIT>
struct DecodeCfg {
    // W warps that compute, and two more: 16 of 128 registers a thread, or where
    // the output takes more 12 of 168 or 8 of 255
    static constexpr int W = NG * RB <= 4 ? 14 : NG <= 4 ? 10 : 6;
    static constexpr int kThreads = 32 * (W + 2);
    // ring slots, SL for each lane of the fetching warp: a warp holds two while it
    // works, the others are on their way
    static constexpr int SL = W == 14 ? 2 : 1, S = 32 * SL;
    static constexpr int K = NG > 4 ? 2 : RB == 1 && !SPLIT ? 6 : 4;  // steps whose operands are held
    static constexpr int kRows = 8 * RB;
    static constexpr int kCh = 32 * NG;
    static constexpr int kStride = kCh + 4;          // merge rows: spreads a quarter warp over the banks
    static constexpr int NT = SPLIT ? 2 : 1;         // terms of a query
    static constexpr size_t kRing = (size_t)S * kv4_bytes(NG);
    // a step's outputs, a row each of every warp; at the run's end also what the
    // threads make of an item's pieces, 6 values each
    static constexpr size_t kOut = sizeof(float) * (size_t)W * kRows * kStride;
    static constexpr size_t kPieces = sizeof(float) * 6 * kThreads;
    static constexpr size_t kMerge = kOut > kPieces ? kOut : kPieces;
    static constexpr size_t kQuery = 16 * (size_t)RB * NG * (32 * NT + 4);  // operands, bias
    static constexpr size_t kSmem = kRing + kMerge + K * kQuery;
};

// A run's share of one item.
struct DecodeStep {
    int base, granules;        // of the run's granules: [base, base + granules)
    int p0;                    // position of the first
    int rho0, rows, kvh;       // row tile, KV head
    int row0, at0;             // sequence's first query row, and its position
    int whole, slot, n;        // of its output: the item's granules,
    int64_t start;             // and the unit of the first
    int owner;                 // the warp that takes all of a short whole item; -1: in turn
    int more;
};
constexpr int kShort = 6;  // granules of a short item

// The walk over a run's steps, the same in every warp that makes it.
struct DecodeWalk {
    Kv4Seq s;
    int64_t u, u1;
    int seq, sub, off, item, base, shorts;
    bool more;
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

// The next step of the walk that has granules of the run in it; false at the
// end. now / seq: the step's sequence.
__device__ __forceinline__ bool next_step(const Kv4AttnArgs &a, int G, int rows, int warps, DecodeWalk &w, DecodeStep &d,
                                          Kv4Seq &now, int &seq) {
    while (w.more) {
        const Kv4Share sh = kv4_share(w.s, w.off, w.u, w.u1);
        now = w.s;
        seq = w.seq;
        const int sub = w.sub;
        w.u += w.item - w.off;
        w.off = 0;
        // the item that a run ends in may have no share of it
        w.more = w.u1 - w.u > kKv4Fixed;
        if (w.more && ++w.sub >= kv4_items(w.s, G, rows, a.c.nkv)) {
            w.sub = 0;
            do w.s = load_seq(a, ++w.seq);
            while (kv4_items(w.s, G, rows, a.c.nkv) == 0);
            w.item = w.s.n + kKv4Fixed;
        }
        if (sh.take == 0) continue;
        d.base = w.base;
        d.granules = sh.take;
        d.p0 = (now.g0 + sh.from) * kKv4Granule;
        d.rho0 = sub / a.c.nkv * rows;
        d.kvh = sub % a.c.nkv;
        d.rows = min(rows, now.nq * G - d.rho0);
        d.row0 = now.row0;
        d.at0 = now.len - now.nq;
        d.whole = sh.begins && sh.ends;
        d.slot = 2 * blockIdx.x + (sh.begins ? 1 : 0);
        d.n = now.n;
        d.start = sh.start;
        d.owner = d.whole && sh.take <= kShort ? w.shorts++ % warps : -1;
        d.more = w.more;
        w.base += d.granules;
        return true;
    }
    return false;
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

// 8 channels of a query row as they lie (NV vectors of 16 bytes), and as fp32:
// apart, so that the loads of several pieces are under way at once.
template <int NV>
__device__ __forceinline__ void load_q8(const Kv4AttnArgs &a, int64_t at, uint4 (&w)[NV]) {
    if (a.vec) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const char *>(a.q) + at * (2 * NV));
#pragma unroll
        for (int i = 0; i < NV; ++i) w[i] = p[i];
    } else if constexpr (NV == 2) {
        const uint32_t *p = static_cast<const uint32_t *>(a.q) + at;
        w[0] = make_uint4(p[0], p[1], p[2], p[3]);
        w[1] = make_uint4(p[4], p[5], p[6], p[7]);
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(a.q) + at;
        w[0] = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16,
                          p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
    }
}
template <int NV>
__device__ __forceinline__ void q8_f32(const uint4 (&w)[NV], bool bf16, float (&v)[8]) {
    const uint32_t *x = &w[0].x;
    if constexpr (NV == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __uint_as_float((&w[0].x)[i]);
            v[4 + i] = __uint_as_float((&w[1].x)[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(x + i));
            v[2 * i] = bf16 ? __uint_as_float(x[i] << 16) : h.x;
            v[2 * i + 1] = bf16 ? __uint_as_float(x[i] & 0xffff0000u) : h.y;
        }
    }
}

// A warp loads a step's query rows: lane (g, t) the channels of words t of row g.
template <int NG, int RB, bool SPLIT>
__device__ __forceinline__ void load_rows(const Kv4AttnArgs &a, const DecodeStep &d, int G,
                                          uint4 (&x8)[RB][NG][SPLIT ? 2 : 1]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int rho = d.rho0 + 8 * rb + g, qi = rho / G;
        const bool in = 8 * rb + g < d.rows;
        const int64_t base = (int64_t)(d.row0 + qi) * a.qs + (int64_t)(d.kvh * G + rho - qi * G) * a.c.hd;
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
#pragma unroll
            for (int i = 0; i < (SPLIT ? 2 : 1); ++i) x8[rb][grp][i] = make_uint4(0, 0, 0, 0);
            if (in && 32 * grp + 8 * t < a.c.hd) load_q8(a, base + 32 * grp + 8 * t, x8[rb][grp]);
        }
    }
}

// and makes them the step's operands, for lane (g, t): row g's channels (nibbles
// 0, 4 | 2, 6 | 1, 5 | 3, 7 of word t of a group); for rows 2 t, 2 t + 1 the bias
// their columns start from; a row's unit: one of its scores as a power of two.
template <int NG, int RB, bool SPLIT>
__device__ __forceinline__ void make_operands(const Kv4AttnArgs &a, uint8_t *query, float *unit,
                                              const uint4 (&x8)[RB][NG][SPLIT ? 2 : 1]) {
    constexpr int NT = SPLIT ? 2 : 1;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const bool bf16 = a.dtype == RABBIT_CUDA_BF16;
    uint4 *q = reinterpret_cast<uint4 *>(query);
    float4 *c0 = reinterpret_cast<float4 *>(q + RB * NT * NG * 32);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        float top = 0.f;
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
            float v[8];
            q8_f32(x8[rb][grp], bf16, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(14 - e), 2^e <= top: the largest goes to [2^14, 2^15)
        const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100);
        const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        const float down = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
        const float sup = a.scale < 0.f ? -up : up;
        if (t == 0) unit[8 * rb + g] = fabsf(a.scale) * (down * 16777216.0f);
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
            float sum = 0.f, y[8];
            q8_f32(x8[rb][grp], bf16, y);
            uint32_t f[NT][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // the instruction's two steps
                const float by = !SPLIT && i ? 0.0625f : 1.0f, back = !SPLIT && i ? 16.f : 1.0f;
                float v[4] = {y[i], y[i + 4], y[i + 2], y[i + 6]};
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
                q[((rb * NT + term) * NG + grp) * 32 + lane] =
                    make_uint4(f[term][0], f[term][1], f[term][2], f[term][3]);
            if constexpr (!SPLIT) {
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum *= -8.0f / 16777216.0f;
                const float s0 = __shfl_sync(0xffffffffu, sum, 8 * t);
                const float s1 = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
                if (g == 0) c0[(rb * NG + grp) * 4 + t] = make_float4(s0, s1, s0, s1);
            }
        }
    }
}

template <int NG, int RB, bool SPLIT>
__global__ void __launch_bounds__(DecodeCfg<NG, RB, SPLIT>::kThreads, 1)
    k_kv4_decode(const __grid_constant__ Kv4AttnArgs a) {
    using C = DecodeCfg<NG, RB, SPLIT>;
    constexpr int W = C::W, S = C::S, NT = C::NT, K = C::K;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[S], empty[S];            // granules
    __shared__ __align__(8) uint64_t asked[K], done[K];            // steps: operands made; done with
    __shared__ __align__(8) uint64_t left, merged;                 // outputs written; merged
    __shared__ int tag[S];                   // a slot's last granule: 2 x its round + whether it is there
    __shared__ DecodeStep steps[K];
    __shared__ __align__(8) float unit[K][C::kRows];      // a step's rows: one of their scores, as a power of two
    __shared__ int pending, pend[2][6];      // items whose last piece came from here
    __shared__ int64_t warp_sums[C::kThreads / 32];
    __shared__ int64_t found_before;
    __shared__ int found_seq;
    __shared__ Kv4Seq found;
    __shared__ float wm[W][C::kRows], wl[W][C::kRows];
    __shared__ float suml[C::kRows];
    launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < S) {
        tag[tid] = -2;  // no round
        mbar_init(&full[tid], 1);
        mbar_init(&empty[tid], 1);
        if (tid < K) {
            mbar_init(&asked[tid], 1);
            mbar_init(&done[tid], W);
        }
        if (tid == 0) {
            mbar_init(&left, W);
            mbar_init(&merged, 1);
        }
        mbar_init_fence();
    }
    if (tid == 0) {
        pending = 0;
    }
    wait_prerequisite();
    const Kv4View &c = a.c;
    const int G = a.nh / c.nkv;

    // ---- this CTA's run of units
    int64_t mine = 0, total;
    Kv4Seq s = {};
    for (int i = tid; i < a.n_seqs; i += C::kThreads) {
        int bad;
        s = load_seq(a, i, &bad);
        if (bad && blockIdx.x == 0) atomicOr(c.err, bad);
        mine += kv4_cost(s, G, C::kRows, c.nkv);
    }
    const int64_t excl = block_scan<C::kThreads>(mine, warp_sums, total);
    // rows of sequences that see nothing: zeros
    for (int i = blockIdx.x; i < a.n_seqs; i += gridDim.x) {
        const Kv4Seq s = load_seq(a, i);
        if (s.n > 0) continue;
        const int row4 = a.nh * (c.hd / 4);
        for (int64_t x = tid; x < (int64_t)s.nq * row4; x += C::kThreads) {
            const float zero[4] = {0.f, 0.f, 0.f, 0.f};
            const int64_t r = x / row4;
            store4(a, (s.row0 + r) * a.os + 4 * (x - r * row4), zero, 4);
        }
    }
    if (total == 0) return;
    const int64_t parts = kv4_parts(total, gridDim.x);
    if (blockIdx.x >= parts) return;
    const int64_t u0 = kv4_cut(blockIdx.x, total, parts);
    if (a.n_seqs <= C::kThreads) {
        if (mine > 0 && excl <= u0 && u0 < excl + mine) {
            found = s;
            found_seq = tid;
            found_before = excl;
        }
    } else {
        int64_t base = 0;
        for (int i0 = 0; i0 < a.n_seqs && base <= u0; i0 += C::kThreads) {
            const int i = i0 + tid;
            int64_t all, cost = 0;
            if (i < a.n_seqs) {
                s = load_seq(a, i);
                cost = kv4_cost(s, G, C::kRows, c.nkv);
            }
            const int64_t before = base + block_scan<C::kThreads>(cost, warp_sums, all);
            if (cost > 0 && before <= u0 && u0 < before + cost) {
                found = s;
                found_seq = i;
                found_before = before;
            }
            base += all;
        }
    }
    __syncthreads();
    auto start_walk = [&](DecodeWalk &w) {
        w.seq = found_seq;
        w.s = found;
        w.u = u0;
        w.u1 = kv4_cut(blockIdx.x + 1, total, parts);
        w.item = w.s.n + kKv4Fixed;
        const int64_t r = u0 - found_before;
        w.sub = r >> 31 ? (int)(r / w.item) : (int)r / w.item;
        w.off = (int)(r - (int64_t)w.sub * w.item);
        w.base = 0;
        w.shorts = 0;
        w.more = true;
    };
    float *mo = reinterpret_cast<float *>(smem + C::kRing);  // [W][rows][kStride]
    // operands [K][RB][NT][NG][32 lanes], each followed by the bias [RB][NG][4 t]
    uint8_t *queries = smem + C::kRing + C::kMerge;
    const float *stats = a.part + (size_t)2 * gridDim.x * C::kRows * C::kCh;  // pieces' (reference, sum)
    auto row_at = [&](int row0, int kvh, int rho) {
        const int qi = rho / G;
        return (int64_t)(row0 + qi) * a.os + (int64_t)(kvh * G + rho - qi * G) * c.hd;
    };
    bool ok = true;

    if (warp == W) {
        // ---- the run's granules into the ring; a lane serves a slot, whenever it is free
        const uint64_t policy = policy_evict_first();
        DecodeWalk w;
        DecodeStep d;
        Kv4Seq now;
        int seq, issued = 0;  // granules this lane has issued: every 32nd of the run
        start_walk(w);
        while (ok && next_step(a, G, C::kRows, W, w, d, now, seq)) {
            int k = (lane - d.base) & 31;
            const uint8_t *from = nullptr;
            auto look_up = [&]() {
                from = nullptr;
                if (k >= d.granules) return;
                const int pos = d.p0 + k * kKv4Granule, pi = pos / c.page;
                const int page = a.table[(int64_t)seq * a.max_pages + pi];
                if (page >= 0 && page < c.n_pages)
                    from = c.base + (size_t)page * c.page_bytes() + (size_t)d.kvh * c.head_bytes() +
                           (size_t)((pos - pi * c.page) / kKv4Granule) * kv4_bytes(NG);
                else
                    atomicOr(c.err, RB_KV4_ERR_PAGE);
            };
            look_up();
            for (uint64_t t0 = 0;;) {
                const int slot = lane + 32 * (issued % C::SL), round = issued / C::SL;
                const bool ready = k < d.granules && (round == 0 || mbar_test(&empty[slot], (round - 1) & 1));
                if (ready) {
                    *static_cast<volatile int *>(&tag[slot]) = 2 * round + (from != nullptr);
                    if (from) {
                        mbar_arrive_expect_tx(&full[slot], kv4_bytes(NG));
                        bulk_g2s(smem + slot * kv4_bytes(NG), from, kv4_bytes(NG), &full[slot], policy);
                    } else {
                        mbar_arrive(&full[slot]);
                    }
                    ++issued;
                    k += 32;
                    look_up();
                }
                if (!__any_sync(0xffffffffu, k < d.granules)) break;
                if (__any_sync(0xffffffffu, ready)) {
                    t0 = 0;
                } else {
                    if (t0 == 0) t0 = globaltimer_ns();
                    __nanosleep(100);
                    if (globaltimer_ns() - t0 > a.wait_ns) {
                        if (lane == 0) atomicOr(c.err, RB_KV4_ERR_WAIT);
                        ok = false;
                    }
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
            }
        }
        // copies in flight end before the CTA does, also where a wait ran out
        for (int i = max(0, issued - C::SL); i < issued; ++i)
            mbar_wait(&full[lane + 32 * (i % C::SL)], (i / C::SL) & 1, kKv4DrainNs, nullptr, 0);
    } else if (warp == W + 1) {
        // ---- operands of the coming steps, as far ahead as there is room, and merges
        DecodeWalk w;
        DecodeStep d;
        Kv4Seq now;
        int seq;
        uint4 x8[RB][NG][NT];  // the next step's query rows, loaded ahead
        start_walk(w);
        bool has = next_step(a, G, C::kRows, W, w, d, now, seq);
        if (has && d.owner < 0) load_rows<NG, RB, SPLIT>(a, d, G, x8);
        int asked_n = 0, seen_n = 0, merged_n = 0;  // steps made; steps looked at for a merge; merges
        // A barrier may have turned for one lane's test and not yet for another's: the
        // shuffles, votes and counters behind a test need one answer for the warp.
        auto turned = [](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test(bar, parity)); };
        for (uint64_t t0 = 0; has || seen_n < asked_n;) {
            bool did = false;
            // Step asked_n, once its buffer's last step is done with (and merged)
            const int buf = asked_n % K;
            if (has && asked_n - seen_n < K &&
                (asked_n < K || turned(&done[buf], (asked_n / K - 1) & 1))) {
                did = true;
                if (d.owner < 0)
                    make_operands<NG, RB, SPLIT>(a, queries + buf * C::kQuery, unit[buf], x8);
                if (lane == 0) steps[buf] = d;
                __syncwarp();
                if (lane == 0 && !(a.withhold && blockIdx.x == 0 && asked_n == 0)) mbar_arrive(&asked[buf]);
                ++asked_n;
                has = next_step(a, G, C::kRows, W, w, d, now, seq);
                if (has && d.owner < 0) load_rows<NG, RB, SPLIT>(a, d, G, x8);
            }
            if (seen_n < asked_n) {
                const DecodeStep &st = steps[seen_n % K];
                if (st.owner >= 0) {
                    ++seen_n;
                    did = true;
                } else if (turned(&left, merged_n & 1)) {
                    // the warps' outputs, in their order; lane r has row r's factors
                    did = true;
                    const DecodeStep m = st;
                    float mx = kNoRef, L = 0.f, f[W];
                    const int r0 = lane < C::kRows ? lane : 0;
#pragma unroll
                    for (int x = 0; x < W; ++x) {
                        f[x] = wm[x][r0];
                        mx = fmaxf(mx, f[x]);
                    }
#pragma unroll
                    for (int x = 0; x < W; ++x) {
                        const float l = wl[x][r0];
                        f[x] = l == 0.f ? 0.f : exp2_fast(f[x] - mx);
                        L = fmaf(f[x], l, L);
                        if (lane < C::kRows) wm[x][r0] = f[x];
                    }
                    if (lane < C::kRows) suml[lane] = L;
                    if (!m.whole && lane < m.rows) {
                        float *p = const_cast<float *>(stats) + (size_t)(m.slot * C::kRows + lane) * 2;
                        p[0] = mx;
                        p[1] = L;
                    }
                    __syncwarp();
                    for (int i = lane; i < m.rows * (C::kCh / 4); i += 32) {
                        const int r = i / (C::kCh / 4), ch = 4 * (i % (C::kCh / 4));
                        float v[4] = {0.f, 0.f, 0.f, 0.f};
                        const float *p = mo + r * C::kStride + ch;
#pragma unroll
                        for (int x = 0; x < W; ++x) {
                            const float4 y = *reinterpret_cast<const float4 *>(p + x * C::kRows * C::kStride);
                            const float fx = wm[x][r];
                            v[0] = fmaf(y.x, fx, v[0]);
                            v[1] = fmaf(y.y, fx, v[1]);
                            v[2] = fmaf(y.z, fx, v[2]);
                            v[3] = fmaf(y.w, fx, v[3]);
                        }
                        if (!m.whole) {
                            __stcg(reinterpret_cast<float4 *>(a.part + ((size_t)m.slot * C::kRows + r) * C::kCh + ch),
                                   make_float4(v[0], v[1], v[2], v[3]));
                        } else if (ch < c.hd) {
                            const float s = suml[r] != 0.f ? 1.0f / suml[r] : 0.f;
#pragma unroll
                            for (int x = 0; x < 4; ++x) v[x] *= s;
                            store4(a, row_at(m.row0, m.kvh, m.rho0 + r) + ch, v, min(4, c.hd - ch));
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&merged);
                    if (!m.whole) {
                        __threadfence();
                        __syncwarp();
                        if (lane == 0) {
                            // the runs that have a share of the item
                            const int first = kv4_run_of(m.start, total, parts);
                            const int last = kv4_run_of(m.start + m.n - 1, total, parts);
                            const unsigned before = atomicAdd(a.count + first, 1u);
                            if (before == (unsigned)(last - first)) {
                                a.count[first] = 0u;  // ready for the next call
                                int *p = pend[pending++];
                                p[0] = first;
                                p[1] = last;
                                p[2] = m.rows;
                                p[3] = m.row0;
                                p[4] = m.kvh;
                                p[5] = m.rho0;
                            }
                        }
                        __syncwarp();
                    }
                    ++merged_n;
                    ++seen_n;
                }
            }
            if (did) {
                t0 = 0;
            } else {
                if (t0 == 0) t0 = globaltimer_ns();
                __nanosleep(64);
                if (__any_sync(0xffffffffu, globaltimer_ns() - t0 > a.wait_ns)) {
                    if (lane == 0) atomicOr(c.err, RB_KV4_ERR_WAIT);
                    break;
                }
            }
        }
    } else {
        // ---- scores and outputs
        const int g = lane >> 2, t = lane & 3, tok = kv4_token(g);
        constexpr int NW = (NG + 1) / 2;
        struct Scores {
            float sc[RB][4];           // tokens tok, tok + 8; query rows 2 t, 2 t + 1
            uint32_t v0[NW], v1[NW];   // the tokens' value scales
        };
        int merges = 0;
        for (int step = 0;; ++step) {
            const int buf = step % K;
            if (ok) ok = kv4_wait(&asked[buf], (step / K) & 1, a);
            if (!__all_sync(0xffffffffu, ok)) break;
            const DecodeStep &st = steps[buf];
            const int end = st.base + st.granules, owner = st.owner, by = owner < 0 ? W : 1;
            const bool more = st.more;
            // this warp's first granule of the step: every W-th of the run, or all
            int n = owner < 0 ? st.base + (warp + W - st.base % W) % W : owner == warp ? st.base : end;
            const bool some = n < end;
            if (!some && owner >= 0) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&done[buf]);
                if (!more) break;
                continue;
            }
            const int R = st.rows, rho0 = st.rho0, kvh = st.kvh, p00 = st.p0 - kKv4Granule * st.base;
            if (owner >= 0) {  // a short item's warp makes its operands itself
                uint4 x8[RB][NG][NT];
                load_rows<NG, RB, SPLIT>(a, st, G, x8);
                make_operands<NG, RB, SPLIT>(a, queries + buf * C::kQuery, unit[buf], x8);
                __syncwarp();
            }
            const int at_lo = st.at0 + rho0 / G, at_hi = st.at0 + (rho0 + R - 1) / G;
            const uint4 *q = reinterpret_cast<const uint4 *>(queries + buf * C::kQuery);
            const float4 *c0 = reinterpret_cast<const float4 *>(q + RB * NT * NG * 32);
            float M[RB][2], D[RB][2], l[RB][2], o[RB][NG][2][4];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    M[rb][i] = kNoRef;
                    D[rb][i] = l[rb][i] = 0.f;
                }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int grp = 0; grp < NG; ++grp)
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[rb][grp][m][i] = 0.f;

            // Two granules are under way in a warp: the scores of one and the output of
            // the one before it are independent, in one stretch of code without a
            // branch, so one's instructions fill the other's waits.
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
                    // signed codes are whole numbers: 2^-24 goes into their scale, so that sums with
                    // the largest keys stay finite
                    const float by = SPLIT ? 1.0f / 16777216.0f : 1.0f;
                    const float f0 = piece_bf16(s0, grp) * by, f1 = piece_bf16(s1, grp) * by;
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        float d[4];
#pragma unroll
                        for (int term = NT - 1; term >= 0; --term) {  // the small term first
                            const uint4 b = q[((rb * NT + term) * NG + grp) * 32 + lane];
                            if (SPLIT && term == NT - 1) {
                                mma_f16(d, e0[0], e1[0], e0[1], e1[1], b.x, b.y, 0.f, 0.f, 0.f, 0.f);
                            } else if (!SPLIT) {
                                const float4 c = c0[(rb * NG + grp) * 4 + t];
                                mma_f16(d, e0[0], e1[0], e0[1], e1[1], b.x, b.y, c.x, c.y, c.z, c.w);
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
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const float2 cs = *reinterpret_cast<const float2 *>(&unit[buf][8 * rb + 2 * t]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) s.sc[rb][x] = __fmul_rn(s.sc[rb][x], x & 1 ? cs.y : cs.x);
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
                const float vtop = fmaxf(log2_fast(__uint_as_float(vmax)), kLeastScale);
                bool odd = edge || vmax >= 0x7f800000u;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        odd |= (fmaxf(s.sc[rb][i], s.sc[rb][2 + i]) - M[rb][i]) + vtop > D[rb][i] + 14.f;
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
                top0 = fmaxf(log2_fast(top0), kLeastScale);
                top1 = fmaxf(log2_fast(top1), kLeastScale);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float mn = fmaxf(M[rb][i], fmaxf(s.sc[rb][i], s.sc[rb][2 + i]));
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
                        float cd = fmaxf((s.sc[rb][i] - mn) + top0, (s.sc[rb][2 + i] - mn) + top1);
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) cd = fmaxf(cd, __shfl_xor_sync(0xffffffffu, cd, x));
                        const float was = (M[rb][i] - mn) + D[rb][i];
                        const bool raise = cd > was + 14.f;
                        const float f = raise ? exp2_fast(was - (cd - 6.f)) : 1.f;
                        if (raise) {
                            M[rb][i] = mn;
                            D[rb][i] = cd - 6.f;
                        }
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
            auto output = [&](const uint8_t *gr, Scores &s, uint64_t *release) {
                // values: tokens 2 t, 2 t + 1 of the tile's order, channels 4 g .. 4 g + 3
                uint32_t vw[4][NW];
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    load_piece<2 * NG>(vw[x], gr + kv4_v(NG) + (8 * (x >> 1) + (x & 1 ? 4 + (t ^ 1) : t)) * kv4_row(NG) +
                                                  (g ^ ((t & 2) << 1)) * 2 * NG);
                __syncwarp();
                if (lane == 0) mbar_arrive(release);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        s.sc[rb][x] = exp2_fast((s.sc[rb][x] - M[rb][x & 1]) - D[rb][x & 1]);
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

            // The granule, when it is there; its validity. A slot's granules go to one
            // warp after another, and a barrier tells only a phase from the next: a warp
            // ahead of the slot's earlier granules would take an older phase for its own.
            // So it looks for its round's tag first, which is written once the round
            // before is over. The lanes leave with one answer: after a wait that ran out
            // all of them have ok false.
            auto arrived = [&](int n) -> bool {
                const volatile int *at = &tag[n % S];
                int v = *at;
                if (v >> 1 != n / S) {
                    const uint64_t t0 = globaltimer_ns();
                    while (ok && (v = *at) >> 1 != n / S) {
                        __nanosleep(64);
                        if (globaltimer_ns() - t0 > a.wait_ns) {
                            atomicOr(c.err, RB_KV4_ERR_WAIT);
                            ok = false;
                        }
                    }
                }
                if (ok) ok = kv4_wait(&full[n % S], (n / S) & 1, a);
                ok = __all_sync(0xffffffffu, ok);
                return v & 1;
            };
            // (A warp that holds a granule's slot waits only for one less than S after it:
            // the first granule that is waited for and not yet fetched never waits for a
            // slot whose holder waits itself.)
            static_assert(W < S, "a granule and the next one of its warp in the ring");
            if (some) {
                Scores cur;
                {
                    const bool there = arrived(n);
                    if (!ok) break;
                    score(smem + n % S * kv4_bytes(NG), cur);
                    settle(cur, p00 + n * kKv4Granule, there);
                }
                for (int nx = n + by; nx < end; nx += by) {
                    const bool there = arrived(nx);
                    if (!ok) break;
                    Scores nxt;
                    score(smem + nx % S * kv4_bytes(NG), nxt);
                    output(smem + n % S * kv4_bytes(NG), cur, &empty[n % S]);
                    settle(nxt, p00 + nx * kKv4Granule, there);
                    cur = nxt;
                    n = nx;
                }
                if (!ok) break;
                output(smem + n % S * kv4_bytes(NG), cur, &empty[n % S]);
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int s = 4; s < 32; s <<= 1) l[rb][i] += __shfl_xor_sync(0xffffffffu, l[rb][i], s);

            if (owner >= 0) {
                // ---- a short item's end: its rows, from here
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = 8 * rb + 2 * t + i;
                        const float s = l[rb][i] != 0.f ? 1.0f / l[rb][i] : 0.f;
#pragma unroll
                        for (int grp = 0; grp < NG; ++grp) {
                            const float v[4] = {o[rb][grp][0][i] * s, o[rb][grp][1][i] * s, o[rb][grp][0][2 + i] * s,
                                                o[rb][grp][1][2 + i] * s};
                            const int ch = 32 * grp + 4 * g;
                            if (r < R && ch < c.hd) store4(a, row_at(st.row0, kvh, rho0 + r) + ch, v, min(4, c.hd - ch));
                        }
                    }
                __syncwarp();
                if (lane == 0) mbar_arrive(&done[buf]);
                if (!more) break;
                continue;
            }
            // ---- the step's end: this warp's output (a warp without a granule of the
            // step has only zeros, as its factors are)
            __syncwarp();
            if (lane == 0) mbar_arrive(&done[buf]);
            if (merges > 0 && ok) ok = kv4_wait(&merged, (merges - 1) & 1, a);
            if (!__all_sync(0xffffffffu, ok)) break;
            ++merges;
            float *out = mo + (size_t)warp * C::kRows * C::kStride;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    // the reference in one number again: M + D, or M where D would be lost in it
                    const float ref = fabsf(M[rb][i]) < 1048576.f ? M[rb][i] + D[rb][i] : M[rb][i];
                    const float f = exp2_fast((M[rb][i] - ref) + D[rb][i]);
                    if (g == 0) {
                        wm[warp][8 * rb + 2 * t + i] = ref;
                        wl[warp][8 * rb + 2 * t + i] = l[rb][i] * f;
                    }
                    float *row = out + (8 * rb + 2 * t + i) * C::kStride + 4 * g;
#pragma unroll
                    for (int grp = 0; grp < NG; ++grp)
                        *reinterpret_cast<float4 *>(row + 32 * grp) =
                            make_float4(o[rb][grp][0][i] * f, o[rb][grp][1][i] * f, o[rb][grp][0][2 + i] * f,
                                        o[rb][grp][1][2 + i] * f);
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(&left);
            if (!more) break;
        }
    }

    // ---- items whose last piece came from this run: merged by the whole CTA, in
    // the pieces' order. A thread takes 4 channels of a row and every `ways`-th
    // run of pieces, then the ways are merged (in shared memory: all else in it
    // is done with).
    __syncthreads();
    for (int x = 0; x < pending; ++x) {
        __threadfence();
        const int first = pend[x][0], np = pend[x][1] - first + 1, R = pend[x][2], n4 = R * (C::kCh / 4);
        const int ways = max(1, min(8, C::kThreads / n4)), each = (np + ways - 1) / ways;
        float *part = mo;  // [ways][6][n4]
        auto fold = [](float &mx, float &L, float (&v)[4], float m, float l, const float4 &y) {
            const float up = fmaxf(mx, m), f = exp2_fast(mx - up), h = exp2_fast(m - up);
            mx = up;
            L = fmaf(L, f, l * h);
            v[0] = fmaf(v[0], f, y.x * h);
            v[1] = fmaf(v[1], f, y.y * h);
            v[2] = fmaf(v[2], f, y.z * h);
            v[3] = fmaf(v[3], f, y.w * h);
        };
        for (int i0 = 0; i0 < n4; i0 += C::kThreads) {
            const int way = ways > 1 ? tid / n4 : 0, i = ways > 1 ? tid - way * n4 : i0 + tid;
            const int r = i / (C::kCh / 4), ch = 4 * (i % (C::kCh / 4));
            float mx = kNoRef, L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
            if (way < ways && i < n4) {
                const int end = min(np, (way + 1) * each);
                for (int b0 = way * each; b0 < end; b0 += 8) {
                    float4 y[8];
                    float2 ml[8];
#pragma unroll
                    for (int b = 0; b < 8; ++b)
                        if (b0 + b < end) {
                            const size_t s = (size_t)(2 * (first + b0 + b) + (b0 + b == 0)) * C::kRows + r;
                            ml[b] = __ldcg(reinterpret_cast<const float2 *>(stats) + s);
                            y[b] = __ldcg(reinterpret_cast<const float4 *>(a.part + s * C::kCh + ch));
                        }
#pragma unroll
                    for (int b = 0; b < 8; ++b)
                        if (b0 + b < end) fold(mx, L, v, ml[b].x, ml[b].y, y[b]);
                }
                if (way > 0) {
                    float *p = part + (size_t)way * 6 * n4 + i;
                    p[0] = mx;
                    p[n4] = L;
#pragma unroll
                    for (int k = 0; k < 4; ++k) p[(2 + k) * n4] = v[k];
                }
            }
            __syncthreads();
            if (way == 0 && i < n4 && ch < c.hd) {
                for (int k = 1; k < ways; ++k) {
                    const float *p = part + (size_t)k * 6 * n4 + i;
                    fold(mx, L, v, p[0], p[n4], make_float4(p[2 * n4], p[3 * n4], p[4 * n4], p[5 * n4]));
                }
                const float inv = L != 0.f ? 1.0f / L : 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] *= inv;
                store4(a, row_at(pend[x][3], pend[x][4], pend[x][5] + r) + ch, v, min(4, c.hd - ch));
            }
            __syncthreads();
        }
    }
}

}  // namespace rb
