// rb_kv4_chunk.cuh -- attention over the 4-bit cache for many query rows a
// sequence (prefill chunks) of 16-bit types: the codes of a tile of positions
// are made fp16 once in shared memory for 64 query rows of a KV head.
//
// A CTA has 8 warps that make fp16 tiles (64 positions; four warps take the even
// ones, four the odd ones) and 8 that multiply (16 query rows and every other tile each, m16n8k16 with fp32
// sums; scores, softmax and output stay in their registers), so tiles are made
// while those before are multiplied. Raw granules come by bulk copies four tiles ahead.
//
// Exactness: a code has 3 bits and a scale 8, so code * scale has 11, as an fp16
// number has. Each token has a power of two of its own, 2^ek for its keys (put back on
// its scores) and 2^ev for its values (put into its weights: p = 2^((x - M) - D) is summed
// up, p 2^ev multiplies the values, with the reference M, D as in rb_kv4_decode.cuh),
// that brings its largest scale to [2^12, 2^13). So what a row does not see, of whatever
// size, has no part in it. Of one token the channel groups whose scale is at least
// 2^-29 of its largest are exact; below 2^-37 they are zero. Query channels 2^22 below
// their row's largest lose bits. The weights are rounded to fp16 (2^-11).
//
// Bound by the latency of the two kinds of warps, not yet by the matrix
// instructions (tensor pipe 39 %, issue slots 50 %): 64 rows x 64 positions x 128 channels
// are 512 of those, 1024 cycles of the four sub-partitions; a tile takes some 2700.
// 256 rows x 4 heads a KV head over 4352 positions of 8 KV heads, bf16, 128 CTAs: 97 us,
// 183 TFLOP/s, 0.11 of the measured cuBLAS bf16 rate. Of the splits, measured with one
// exponent a granule: 4 warps of either kind 119 us, 8 making 130 us (the others then spilled),
// 8 multiplying 122 us, 8 of either 91 us; the tokens' own exponents take 4 us more,
// the reference in two parts 2.
#pragma once
#include <type_traits>

#include "rb_device.cuh"
#include "rb_kv4_decode.cuh"

namespace rb {

template <int NG>
struct ChunkCfg {
    static constexpr int kRows = 64, kTile = 64;     // query rows, positions
    static constexpr int kMul = 8, kThreads = 32 * (kMul + 8);  // warps that multiply, two for each 16 rows; that make tiles
    static constexpr int kCh = 32 * NG;
    static constexpr int kStride = 2 * kCh + 16;     // bytes of a tile's row: 8 rows in different banks
    static constexpr int kRaw = 4, kMade = 4;        // stages of raw granules, of fp16 tiles
    static constexpr size_t kRawBytes = 4 * (size_t)kv4_bytes(NG);
    static constexpr size_t kMadeBytes = 2 * (size_t)kTile * kStride;  // keys, then values
    static constexpr size_t kQuery = 16 * 4 * 2 * NG * 32;  // operands of 4 x 16 rows
    static constexpr size_t kSmem = kRaw * kRawBytes + kMade * kMadeBytes + kQuery;
    // at the end the second warps' (reference, sum) and outputs, over the fp16 tiles
    static_assert(4 * 32 * 4 * (6 + 16 * NG) <= kMade * kMadeBytes, "room for the merge");
};

struct ChunkGranule {  // of a tile, beside its fp16 values
    float ev;          // the largest of its tokens'
    int there, odd;    // it was read; some value scale is not finite
};

// Exponents of tokens' scales go from 2^-64 on (a scale below that, and 0, count as
// that). A weight is at most 2^14 as its value is multiplied by it, so at most 2^90 in
// the sum, which 2^30 positions do not overflow.
constexpr int kChunkLeast = -64, kChunkLift = 12;

// A token's exponent: of the largest finite one of its scales; and which of them
// are not finite. (Scales are not below zero: in order as integers.)
template <int NW>
__device__ __forceinline__ int token_exponent(const uint32_t (&sc)[NW], int &odd) {
    uint32_t top = sc[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) top = __vmaxu2(top, sc[i]);
    top = max(top & 0xffffu, top >> 16);
    odd = 0;
    if (top >= 0x7f80u) {
        top = 0;
#pragma unroll
        for (int i = 0; i < 2 * NW; ++i) {
            const uint32_t x = sc[i >> 1] >> (16 * (i & 1)) & 0xffffu;
            if (x >= 0x7f80u) odd |= 1 << i;
            else top = max(top, x);
        }
    }
    return max((int)(top >> 7) - 127, kChunkLeast);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ uint32_t mul_f16(uint32_t a, __half2 s) {
    const __half2 h = __hmul2(*reinterpret_cast<const __half2 *>(&a), s);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <int NG>
__global__ void __launch_bounds__(ChunkCfg<NG>::kThreads, 1) k_kv4_chunk(const __grid_constant__ Kv4AttnArgs a) {
    using C = ChunkCfg<NG>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t raw_full[C::kRaw], made[C::kMade], used[C::kMade];
    __shared__ ChunkGranule meta[C::kMade][4];
    __shared__ __align__(8) float kback[C::kMade][C::kTile], vback[C::kMade][C::kTile];  // 2^(ek - lift), 2^(ev - lift) of each token
    __shared__ uint8_t vbad[C::kMade][C::kTile];  // groups of a position whose value scale is not finite
    __shared__ int raw_there[C::kRaw];
    launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < C::kRaw; ++i) mbar_init(&raw_full[i], 1);
        for (int i = 0; i < C::kMade; ++i) {
            mbar_init(&made[i], 4);
            mbar_init(&used[i], 4);
        }
        mbar_init_fence();
    }
    wait_prerequisite();
    const Kv4View &c = a.c;
    const int G = a.nh / c.nkv, seq = blockIdx.z, kvh = blockIdx.y;
    int bad;
    const Kv4Seq s = load_seq(a, seq, &bad);
    if (bad && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) atomicOr(c.err, bad);
    // the last rows see most: they come first
    const int rho0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * C::kRows, R = min(C::kRows, s.nq * G - rho0);
    if (R <= 0) return;
    const int at0 = s.len - s.nq;
    const int at_lo = at0 + rho0 / G, at_hi = at0 + (rho0 + R - 1) / G;
    const int lo = a.window > 0 && at_lo >= a.window ? at_lo - a.window + 1 : 0;
    const int g0 = lo / kKv4Granule, ng = at_hi >= lo ? at_hi / kKv4Granule + 1 - g0 : 0;
    const int tiles = (ng + 3) / 4;
    __syncthreads();
    bool ok = true;

    if (warp >= C::kMul) {
        // ---- raw granules into fp16 tiles: four warps the even ones, four the odd ones,
        // warp w granule w of each
        const int w = warp & 3, turn = (warp - C::kMul) >> 2;
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const uint64_t policy = policy_evict_last();  // the other row tiles read them too
        // lanes 0..3 of the first of these warps have a granule each of a tile: its page,
        // looked up a tile before it is needed
        int page = -1;
        auto look_up = [&](int tile) {
            const int k = 4 * tile + lane;
            page = -1;
            if (lane < 4 && k < ng)
                page = a.table[(int64_t)seq * a.max_pages + (g0 + k) * kKv4Granule / c.page];
        };
        auto fetch = [&](int tile) {
            const int st = tile % C::kRaw, k = 4 * tile + lane;
            const uint8_t *from = nullptr;
            if (lane < 4 && k < ng) {
                if (page >= 0 && page < c.n_pages)
                    from = c.base + (size_t)page * c.page_bytes() + (size_t)kvh * c.head_bytes() +
                           (size_t)((g0 + k) % (c.page / kKv4Granule)) * kv4_bytes(NG);
                else
                    atomicOr(c.err, RB_KV4_ERR_PAGE);
            }
            const unsigned there = __ballot_sync(0xffffffffu, from != nullptr);
            if (lane == 0) {
                raw_there[st] = there;
                if (there) mbar_arrive_expect_tx(&raw_full[st], __popc(there) * kv4_bytes(NG));
                else mbar_arrive(&raw_full[st]);
            }
            __syncwarp();
            if (from) bulk_g2s(smem + st * C::kRawBytes + lane * kv4_bytes(NG), from, kv4_bytes(NG), &raw_full[st], policy);
            look_up(tile + 2);
        };
        if (w == 0) {
            look_up(turn);
            for (int i = turn; i < min(C::kRaw, tiles); i += 2) fetch(i);
        }
        for (int tile = turn; tile < tiles; tile += 2) {
            const int st = tile % C::kRaw, mt = tile % C::kMade;
            ok = kv4_wait(&raw_full[st], (tile / C::kRaw) & 1, a, 64);
            if (tile >= C::kMade && ok) ok = kv4_wait(&used[mt], (tile / C::kMade - 1) & 1, a, 64);
            ok = __all_sync(0xffffffffu, ok);
            const bool there = raw_there[st] >> w & 1;
            const uint8_t *gr = smem + st * C::kRawBytes + w * kv4_bytes(NG);
            uint8_t *kt = smem + C::kRaw * C::kRawBytes + mt * C::kMadeBytes + (size_t)w * 16 * C::kStride;
            uint8_t *vt = kt + C::kTile * C::kStride;
            constexpr int NW = (NG + 1) / 2;
            auto make = [&](auto part) {
                constexpr bool values = decltype(part)::value;
                const uint16_t *scales = reinterpret_cast<const uint16_t *>(gr + (values ? kv4_vs(NG) : kv4_ks(NG)));
                if constexpr (!values) {
                    if (lane == 0) meta[mt][w].there = there;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {  // word t of a token's groups
                        const int j = (lane >> 2) + 8 * x, t = lane & 3;
                        uint32_t kw[NG], sc[NW];
                        load_piece<4 * NG>(kw, gr + j * kv4_row(NG) + t * 4 * NG);
                        load_piece<2 * NG>(sc, scales + j * NG);
                        int mask;
                        const int e = token_exponent(sc, mask);
                        const float down = pow2(kChunkLift - e);
                        if (t == 0) kback[mt][16 * w + j] = pow2(e - kChunkLift);
#pragma unroll
                        for (int grp = 0; grp < NG; ++grp) {
                            uint32_t y[4];
                            key_codes<true>(y, kw[grp]);  // nibbles (0, 4), (2, 6), (1, 5), (3, 7)
                            const __half2 f = __float2half2_rn(piece_bf16(sc, grp) * down);
                            *reinterpret_cast<uint4 *>(kt + j * C::kStride + 2 * (32 * grp + 8 * t)) =
                                there ? make_uint4(mul_f16(y[0], f), mul_f16(y[2], f), mul_f16(y[1], f), mul_f16(y[3], f))
                                      : make_uint4(0, 0, 0, 0);
                        }
                    }
                } else {
                    int most = kChunkLeast, any = 0;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {  // word g of a token's groups
                        const int j = (lane >> 3) + 4 * x, g = lane & 7;
                        uint32_t vw[NW], sc[NW];
                        load_piece<2 * NG>(vw, gr + kv4_v(NG) + j * kv4_row(NG) + kv4_vplace(j, g) * 2 * NG);
                        load_piece<2 * NG>(sc, scales + j * NG);
                        int mask;
                        const int e = token_exponent(sc, mask);
                        const float down = pow2(kChunkLift - e);
                        most = max(most, e);
                        any |= mask;
                        if (g == 0) {
                            vback[mt][16 * w + j] = pow2(e - kChunkLift);
                            vbad[mt][16 * w + j] = (uint8_t)mask;
                        }
#pragma unroll
                        for (int i = 0; i < NW; ++i) {  // two groups at a time, one in each half of a pair
                            const uint32_t h = vw[i], h8 = h >> 8;
                            // (a value that is not finite is put into the output by itself)
                            const float s0 = piece_bf16(sc, 2 * i), s1 = 2 * i + 1 < NG ? piece_bf16(sc, 2 * i + 1) : 0.f;
                            const __half2 f = __floats2half2_rn(s0 < INFINITY ? s0 * down : 0.f, s1 < INFINITY ? s1 * down : 0.f);
                            uint32_t y[4];
                            signed_codes(y[0], y[1], h);
                            signed_codes(y[2], y[3], h8);
#pragma unroll
                            for (int k = 0; k < 4; ++k) y[k] = there ? mul_f16(y[k], f) : 0u;
                            uint8_t *to = vt + j * C::kStride + 2 * (64 * i + 4 * g);
                            *reinterpret_cast<uint2 *>(to) =
                                make_uint2(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410));
                            if (2 * i + 1 < NG)
                                *reinterpret_cast<uint2 *>(to + 64) =
                                    make_uint2(__byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632));
                        }
                    }
                    const bool odd = __any_sync(0xffffffffu, any);
                    most = __reduce_max_sync(0xffffffffu, most);
                    if (lane == 0) {
                        meta[mt][w].ev = (float)(most - kChunkLift);
                        meta[mt][w].odd = odd;
                    }
                }
            };
            if (ok) {
                make(std::false_type());
                make(std::true_type());
                __syncwarp();
                if (lane == 0 && !(a.withhold && tile == 0 && w == 0)) mbar_arrive(&made[mt]);
            }
            // the raw stage is read, by all four warps, or one's wait ran out
            ok = named_all(3 + turn, 128, ok);
            if (!ok) {
                if (w == 0)  // the copies of this tile and those fetched ahead of it
                    for (int i = tile; i < min(tile + C::kRaw, tiles); i += 2)
                        mbar_wait(&raw_full[i % C::kRaw], (i / C::kRaw) & 1, kKv4DrainNs, nullptr, 0);
                return;
            }
            if (w == 0 && tile + C::kRaw < tiles) fetch(tile + C::kRaw);
        }
        return;
    }

    // ---- rows 16 wr + g and + 8 of the tile; one warp takes its even tiles, another the
    // odd ones, so one's instructions fill the other's waits
    const int g = lane >> 2, t = lane & 3, wr = warp & 3, turn = warp >> 2;
    // (registers: 8 x 32 x (72 + 168) of the 65536 that 512 threads of 128 begin with)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    uint4 *qs = reinterpret_cast<uint4 *>(smem + C::kRaw * C::kRawBytes + C::kMade * C::kMadeBytes) + wr * 2 * NG * 32 + lane;
    float cs[2];
    int at[2];
    const bool bf16 = a.dtype == RABBIT_CUDA_BF16;
    const uint16_t *qp[2];
    bool in[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 16 * wr + g + 8 * i, rho = rho0 + r, qi = rho / G;
        in[i] = r < R;
        at[i] = in[i] ? at0 + qi : -1;
        qp[i] = static_cast<const uint16_t *>(a.q) + (int64_t)(s.row0 + qi) * a.qs + (int64_t)(kvh * G + rho - qi * G) * c.hd;
        // channels t and t + 4 of every 8: the order in which the tile holds them
        float x[4 * NG][2], top = 0.f;
#pragma unroll
        for (int b = 0; b < 4 * NG; ++b)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t h = in[i] && 8 * b < c.hd ? qp[i][8 * b + t + 4 * k] : 0u;
                x[b][k] = bf16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
                top = fmaxf(top, fabsf(x[b][k]));
            }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100);
        // to [2^8, 2^9): the products with keys of at most 14 stay far inside fp32
        const float up = __uint_as_float((uint32_t)(127 + 8 - e) << 23);
        cs[i] = a.scale * __uint_as_float((uint32_t)(127 - 8 + e) << 23);
        if (turn == 0) {
#pragma unroll
            for (int ks = 0; ks < 2 * NG; ++ks) {
                uint32_t *y = &qs[ks * 32].x;
                y[i] = pack_f16(x[2 * ks][0] * up, x[2 * ks][1] * up);
                y[2 + i] = pack_f16(x[2 * ks + 1][0] * up, x[2 * ks + 1][1] * up);
            }
        }
    }
    named_sync(2, 32 * C::kMul);
    float M[2] = {kNoRef, kNoRef}, D[2] = {0.f, 0.f}, l[2] = {0.f, 0.f}, o[4 * NG][4];
#pragma unroll
    for (int b = 0; b < 4 * NG; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[b][i] = 0.f;
    const uint32_t tiles_at = smem_u32(smem) + (uint32_t)(C::kRaw * C::kRawBytes);
    // row addresses of the loads: keys, matrices (8 positions x 8 channels) in the order
    // (0, 0), (0, 8), (8, 0), (8, 8); values (0, 0), (8, 0), (0, 8), (8, 8)
    const uint32_t kat = ((lane & 7) + (lane >> 4) * 8) * C::kStride + ((lane >> 3) & 1) * 16;
    const uint32_t vat = ((lane & 7) + ((lane >> 3) & 1) * 8) * C::kStride + (lane >> 4) * 16;
    for (int tile = turn; tile < tiles; tile += 2) {
        const int mt = tile % C::kMade, p0 = (g0 + 4 * tile) * kKv4Granule;
        ok = __all_sync(0xffffffffu, kv4_wait(&made[mt], (tile / C::kMade) & 1, a, 64));
        if (!ok) break;
        const uint32_t kt = tiles_at + mt * (uint32_t)C::kMadeBytes, vt = kt + C::kTile * C::kStride;
        float sc[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[n][i] = 0.f;
        // channels outside, positions inside: eight sums that do not wait for one another
#pragma unroll
        for (int ks = 0; ks < 2 * NG; ++ks) {
            uint32_t b[4][4];
            const uint4 q = qs[ks * 32];
#pragma unroll
            for (int j = 0; j < 4; ++j) ldmatrix4(b[j], kt + kat + j * 16 * C::kStride + ks * 32);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float *s0 = sc[2 * j], *s1 = sc[2 * j + 1];
                mma_f16(sc[2 * j], q.x, q.y, q.z, q.w, b[j][0], b[j][1], s0[0], s0[1], s0[2], s0[3]);
                mma_f16(sc[2 * j + 1], q.x, q.y, q.z, q.w, b[j][2], b[j][3], s1[0], s1[1], s1[2], s1[3]);
            }
        }
        // scores as powers of two; masks where some row does not see all of the tile
        ChunkGranule m[4];
        int all = 1, odd = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] = meta[mt][j];
            all &= m[j].there;
            odd |= m[j].there & m[j].odd;
        }
        const bool edge = !all || p0 + C::kTile - 1 > at_lo || (a.window > 0 && p0 <= at_hi - a.window);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const float2 k = *reinterpret_cast<const float2 *>(&kback[mt][8 * n + 2 * t]);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[n][i] = __fmul_rn(sc[n][i], cs[i >> 1] * (i & 1 ? k.y : k.x));
        }
        if (edge) {
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int p = p0 + 8 * n + 2 * t + (i & 1), r = at[i >> 1];
                    if (!m[n >> 1].there || p > r || (a.window > 0 && p <= r - a.window)) sc[n][i] = -INFINITY;
                }
        }
        // a bound with the largest score and ev first, each token's own only where that fails
        const float ev = fmaxf(fmaxf(m[0].ev, m[1].ev), fmaxf(m[2].ev, m[3].ev));
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) mx[i] = fmaxf(mx[i], fmaxf(sc[n][2 * i], sc[n][2 * i + 1]));
        if (__any_sync(0xffffffffu, (mx[0] - M[0]) + ev > D[0] + 14.f || (mx[1] - M[1]) + ev > D[1] + 14.f)) {
            float cand[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                mx[i] = fmaxf(mx[i], M[i]);
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const float2 v = *reinterpret_cast<const float2 *>(&vback[mt][8 * n + 2 * t]);
                const float e0 = log2_fast(v.x), e1 = log2_fast(v.y);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    cand[i] = fmaxf(cand[i], fmaxf((sc[n][2 * i] - mx[i]) + e0, (sc[n][2 * i + 1] - mx[i]) + e1));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float cd = fmaxf(cand[i], __shfl_xor_sync(0xffffffffu, cand[i], 1));
                cd = fmaxf(cd, __shfl_xor_sync(0xffffffffu, cd, 2));
                const float was = (M[i] - mx[i]) + D[i];
                const bool raise = cd > was + 14.f;
                const float f = raise ? exp2_fast(was - (cd - 6.f)) : 1.f;
                if (raise) {
                    M[i] = mx[i];
                    D[i] = cd - 6.f;
                }
                l[i] *= f;
#pragma unroll
                for (int b = 0; b < 4 * NG; ++b) {
                    o[b][2 * i] *= f;
                    o[b][2 * i + 1] *= f;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float *x = sc[2 * j + n];
                const float2 v = *reinterpret_cast<const float2 *>(&vback[mt][16 * j + 8 * n + 2 * t]);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = exp2_fast((x[i] - M[i >> 1]) - D[i >> 1]);
                l[0] += x[0] + x[1];
                l[1] += x[2] + x[3];
                w[2 * n] = pack_f16(x[0] * v.x, x[1] * v.y);
                w[2 * n + 1] = pack_f16(x[2] * v.x, x[3] * v.y);
            }
#pragma unroll
            for (int b = 0; b < 4 * NG; b += 2) {
                uint32_t v[4];
                ldmatrix4_t(v, vt + vat + j * 16 * C::kStride + b * 16);
                float *o0 = o[b], *o1 = o[b + 1];
                mma_f16(o[b], w[0], w[1], w[2], w[3], v[0], v[1], o0[0], o0[1], o0[2], o0[3]);
                mma_f16(o[b + 1], w[0], w[1], w[2], w[3], v[2], v[3], o1[0], o1[1], o1[2], o1[3]);
            }
        }
        if (odd) {  // values that are not finite: NaN for the rows that see them
            for (int x = 0; x < C::kTile; ++x) {
                if (!(meta[mt][x >> 4].there & meta[mt][x >> 4].odd)) continue;
                const int mask = vbad[mt][x], p = p0 + x;
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (mask && p <= at[i] && (a.window == 0 || p > at[i] - a.window))
#pragma unroll
                        for (int b = 0; b < 4 * NG; ++b)
                            if (mask >> (b / 4) & 1) o[b][2 * i] = o[b][2 * i + 1] = __uint_as_float(0x7fc00000u);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&used[mt]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    // the odd tiles' part joins the even tiles'
    if (!named_all(2, 32 * C::kMul, ok)) return;  // all fp16 tiles are read, or a wait ran out
    float *part = reinterpret_cast<float *>(smem + C::kRaw * C::kRawBytes) + wr * 32 * (6 + 16 * NG) + lane;
    if (turn == 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            part[32 * i] = M[i];
            part[32 * (2 + i)] = D[i];
            part[32 * (4 + i)] = l[i];
        }
#pragma unroll
        for (int b = 0; b < 4 * NG; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[32 * (6 + 4 * b + i)] = o[b][i];
    }
    named_sync(2, 32 * C::kMul);
    if (turn == 1) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float l1 = part[32 * (4 + i)], more = (part[32 * i] - M[i]) + (part[32 * (2 + i)] - D[i]);
        const float f0 = exp2_fast(fminf(-more, 0.f)), f1 = exp2_fast(fminf(more, 0.f));
        l[i] = fmaf(l[i], f0, l1 * f1);
#pragma unroll
        for (int b = 0; b < 4 * NG; ++b)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                o[b][2 * i + k] = fmaf(o[b][2 * i + k], f0, part[32 * (6 + 4 * b + 2 * i + k)] * f1);
        if (!in[i]) continue;
        const float inv = l[i] != 0.f ? 1.0f / l[i] : 0.f;
        const int rho = rho0 + 16 * wr + g + 8 * i, qi = rho / G;
        uint16_t *out = static_cast<uint16_t *>(a.out) + (int64_t)(s.row0 + qi) * a.os + (int64_t)(kvh * G + rho - qi * G) * c.hd;
#pragma unroll
        for (int b = 0; b < 4 * NG; ++b) {
            if (8 * b >= c.hd) continue;
            const float x = o[b][2 * i] * inv, y = o[b][2 * i + 1] * inv;
            const uint16_t hx = bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
            const uint16_t hy = bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(y)) : __half_as_ushort(__float2half_rn(y));
            if (a.vec) {
                *reinterpret_cast<uint32_t *>(out + 8 * b + 2 * t) = hx | (uint32_t)hy << 16;
            } else {
                out[8 * b + 2 * t] = hx;
                out[8 * b + 2 * t + 1] = hy;
            }
        }
    }
}

}  // namespace rb
