// rb_f8.cu -- C ABI: rows and blocks as e4m3 codes with a scale for each 128
// columns.
//
// Bound by memory: x is read and its codes are written once. The codes are those of the
// exact quotient x / s, without a division for each value, from r within 2^-22 of 1 / s:
//  * fp32: |x| r (1 - 2^-21) <= |x| / s <= |x| r (1 + 2^-21) holds for the computed products
//    (they round by 2^-24 each). Rounding to e4m3 is monotone, so where both ends give one
//    code it is the quotient's. Where they give two neighbours, the sign of x - m s, m the middle
//    between them, decides; one fma has it exactly.
//  * 16 bits: x, the block's largest value t and a middle m have at most 11, 11 and 5
//    bits, so 448 x / t and m are 2^-16 apart or equal; x / s differs from 448 x / t by s's rounding
//    alone. So x / s is on the side of m on which 448 x / t is or, where that equals m (such x are
//    not rare: x = 3/4 t is one), on the side that the sign of t - 448 s tells, one for the
//    block: the product with r (1 +- 2^-20) has the quotient's code. With 448 s = t the quotient itself is
//    made exact by a correction, and a tie goes to the even code.
// Each rounding and tie is equal to the 64-bit oracle's. 16384 rows of 4096 bf16 took 124 us with the ends
// of the interval and a call for each value between them.
#include <cuda_fp8.h>

#include "rb_device.cuh"
#include "rb_launch.h"
#include "rb_runtime.h"
#include "rb_types.cuh"

namespace rb {

struct F8Args {
    const void *x;
    int64_t xs;
    const int *rows;  // [n_rows] or NULL
    int x_rows;
    uint8_t *q;
    int64_t qs;
    float *scale;
    int n_rows, n_cols, nb;  // nb: blocks of 128 columns
    uint32_t magic;          // i / nb = umulhi(i, magic) >> shift for i below 2^31
    int shift;
};

constexpr int kF8Threads = 256, kF8Resident = 4;  // CTAs of an SM
constexpr uint32_t kInfBits = 0x7F800000u;

// e4m3 codes of two values, to nearest even, held at +-448 (a in the low byte).
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float e4m3_value(uint32_t code) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
}

// A block's scale from the bits of its largest |x|, and what its codes are made with.
struct F8Scale {
    float s, r, lo, hi;  // s, near 1 / s; fp32: the interval's ends; 16 bits: lo, towards the block's side
    bool even;           // 448 s is the block's largest value
    bool rare;           // s is zero, NaN, or below kF8Tiny
};
constexpr float kF8Tiny = 0x1p-60f, kF8Grow = 0x1p64f;
template <bool SHORT>
__device__ __forceinline__ F8Scale f8_scale(uint32_t top) {
    F8Scale f;
    // top / 448 to nearest: a product and one correction (equal to the division for every
    // mantissa while nothing falls below fp32's normal numbers)
    const float t = __uint_as_float(top), q = t * (1.f / 448.f);
    f.s = fmaf(fmaf(-q, 448.f, t), 1.f / 448.f, q);
    f.rare = !(f.s >= kF8Tiny) || top >= kInfBits;
    f.r = __fdividef(1.f, f.s);
    if constexpr (SHORT) {
        const float rest = fmaf(-f.s, 448.f, t);
        f.even = rest == 0.f;
        f.lo = f.r * (rest > 0.f ? 1.f + 0x1p-20f : 1.f - 0x1p-20f);
    } else {
        f.lo = f.r * (1.f - 0x1p-21f);
        f.hi = f.r * (1.f + 0x1p-21f);
    }
    if (f.rare) f.s = top >= kInfBits ? __uint_as_float(0x7FC00000u) : __fdiv_rn(t, 448.f);
    return f;
}

// Code of v where the ends of its quotient's interval give c and c + 1.
__device__ __forceinline__ uint32_t f8_between(float v, float s, uint32_t c) {
    const float m = 0.5f * (fabsf(e4m3_value(c)) + fabsf(e4m3_value(c + 1)));
    const float r = fmaf(-m, s, fabsf(v));
    return r > 0.f || (r == 0.f && (c & 1)) ? c + 1 : c;
}
// Codes of a block without a number (NaN), of zeros, or with a scale below kF8Tiny: x and s are
// multiplied by 2^64, where 1 / s and the remainders are far from fp32's smallest numbers.
__device__ __noinline__ uint32_t f8_rare(float v, float s) {
    if (!(s > 0.f)) return s == 0.f ? 0u : 0x7Fu;
    s *= kF8Grow;
    v *= kF8Grow;
    const float r = __fdividef(1.f, s);
    const uint32_t ab = e4m3x2(v * (r * (1.f - 0x1p-21f)), v * (r * (1.f + 0x1p-21f)));
    const uint32_t a = ab & 255, b = ab >> 8 & 255;
    return a == b ? a : f8_between(v, s, a);
}

// Codes of eight values, the first in the low byte. SHORT: they have at most 11 significant
// bits.
template <bool SHORT>
__device__ __forceinline__ uint2 f8_codes(const float (&x)[8], const F8Scale &f) {
    uint32_t a[2];
    if constexpr (SHORT) {
        float t[8];
        if (f.even) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                t[i] = x[i] * f.r;
                t[i] = fmaf(-fmaf(t[i], f.s, -x[i]), f.r, t[i]);  // (a zero keeps its sign)
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = x[i] * f.lo;
        }
        a[0] = e4m3x2(t[0], t[1]) | e4m3x2(t[2], t[3]) << 16;
        a[1] = e4m3x2(t[4], t[5]) | e4m3x2(t[6], t[7]) << 16;
    } else {
        uint32_t m[2];  // 1 in the bytes whose upper end has the next code
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float *v = x + 4 * i;
            a[i] = e4m3x2(v[0] * f.lo, v[1] * f.lo) | e4m3x2(v[2] * f.lo, v[3] * f.lo) << 16;
            m[i] = (e4m3x2(v[0] * f.hi, v[1] * f.hi) | e4m3x2(v[2] * f.hi, v[3] * f.hi) << 16) - a[i];
        }
        if (m[0] | m[1]) {
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
                const int sh = 8 * (i & 3);
                if (((i < 4 ? m[0] : m[1]) >> sh & 1) == 0) continue;
                float v = x[0];
#pragma unroll
                for (int j = 1; j < 8; ++j) v = i == j ? x[j] : v;
                const uint32_t c = (i < 4 ? a[0] : a[1]) >> sh & 255;
                const uint32_t up = (f8_between(v, f.s, c) - c) << sh;
                if (i < 4) a[0] += up;
                else a[1] += up;
            }
        }
    }
    return make_uint2(a[0], a[1]);
}

// Eight values of a row as they lie in memory, S columns apart; past the row zeros. S = 1: 16 bytes
// at a time. Rows that do not lie on 16 bytes are read one value at a time, and there a block's
// lanes have neighbouring columns (8192 rows of 4100 f16: 43 us; with eight columns in a row each, 70).
template <typename T>
struct F8Raw {
    uint4 w[sizeof(T) / 2];
};
template <typename T, int S>
__device__ __forceinline__ F8Raw<T> f8_load(const T *at, int left) {  // `left` columns from there on
    F8Raw<T> d;
    if (S == 1 && left >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) d.w[i] = reinterpret_cast<const uint4 *>(at)[i];
    } else {
        T *e = reinterpret_cast<T *>(&d);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i * S < left ? at[i * S] : from_f32<T>(0.f);
    }
    return d;
}
template <typename T>
__device__ __forceinline__ void f8_values(const F8Raw<T> &d, float (&v)[8]) {
    const T *e = reinterpret_cast<const T *>(&d);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
}
// The largest |value|'s bits, in T's own format (they order as the values do, infinity and
// NaN above); two 16-bit numbers at a time.
template <typename T>
__device__ __forceinline__ uint32_t f8_top(const F8Raw<T> &d) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&d);
    if constexpr (sizeof(T) == 2) {
        uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
        for (int i = 1; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        return max(m & 0xFFFFu, m >> 16);
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
        return m;
    }
}
template <typename T>
__device__ __forceinline__ uint32_t f8_top_f32(uint32_t top) {
    if constexpr (sizeof(T) == 2) {
        const unsigned short h = (unsigned short)top;
        return __float_as_uint(to_f32(*reinterpret_cast<const T *>(&h)));
    } else {
        return top;
    }
}
// The codes of eight values to q, `left` columns from there on.
template <typename T, int S>
__device__ __forceinline__ void f8_store(uint8_t *q, int left, const F8Raw<T> &d, const F8Scale &f) {
    float v[8];
    f8_values(d, v);
    if (!f.rare) {
        const uint2 w = f8_codes<sizeof(T) == 2>(v, f);
        if (S == 1 && left >= 8) {
            *reinterpret_cast<uint2 *>(q) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i * S < left) q[i * S] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i * S < left) q[i * S] = (uint8_t)f8_rare(v[i], f.s);
    }
}

// One scale for each row's block: eight lanes hold a block, a lane columns 8 l .. (scalar
// form: l, l + 8, ..) of each half of it; BATCH blocks of each eight lanes are in flight.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kF8Threads, kF8Resident) k_f8_rows(const __grid_constant__ F8Args a) {
    constexpr int BATCH = 2, S = VEC ? 1 : 8;
    launch_dependents();
    wait_prerequisite();
    const uint32_t items = (uint32_t)a.n_rows * a.nb, teams = gridDim.x * (kF8Threads / 8);
    const int lane = threadIdx.x & 7;
    for (uint32_t i0 = (blockIdx.x * kF8Threads + threadIdx.x) / 32 * 4; i0 < items; i0 += teams * BATCH) {
        F8Raw<T> d[BATCH][2];
        int row[BATCH], block[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {  // a warp's four blocks side by side, then `teams` on
            const uint32_t i = i0 + (threadIdx.x >> 3 & 3) + b * teams;
            row[b] = -1;
            if (i < items) {
                int r = a.nb == 1 ? i : __umulhi(i, a.magic) >> a.shift;
                block[b] = i - r * a.nb;
                row[b] = r;
                if (a.rows) {
                    r = __ldg(a.rows + r);
                    if (r < 0 || r >= a.x_rows) row[b] = -1;
                }
                if (row[b] >= 0) {
                    const int c = block[b] * 128 + lane * (8 / S);
                    const T *x = static_cast<const T *>(a.x) + r * a.xs + c;
                    d[b][0] = f8_load<T, S>(x, a.n_cols - c);
                    d[b][1] = f8_load<T, S>(x + 64, a.n_cols - c - 64);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            uint32_t top = row[b] >= 0 ? max(f8_top(d[b][0]), f8_top(d[b][1])) : 0u;
#pragma unroll
            for (int m = 4; m; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
            if (row[b] < 0) continue;
            const F8Scale f = f8_scale<sizeof(T) == 2>(f8_top_f32<T>(top));
            const int c = block[b] * 128 + lane * (8 / S);
            uint8_t *q = a.q + row[b] * a.qs + c;
            f8_store<T, S>(q, a.n_cols - c, d[b][0], f);
            f8_store<T, S>(q + 64, a.n_cols - c - 64, d[b][1], f);
            if (lane == 0) a.scale[(int64_t)row[b] * a.nb + block[b]] = f.s;
        }
    }
}

// One scale for each 128 rows x 128 columns: a CTA holds the block in registers, reads it whole and then
// writes it whole. 14336 x 4096: f32 103 us (2.9 TB/s), bf16 69 us (2.6 TB/s); it runs once for each matrix.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kF8Threads) k_f8_blocks(const __grid_constant__ F8Args a) {
    __shared__ uint32_t warp_top[kF8Threads / 32];
    launch_dependents();
    wait_prerequisite();
    constexpr int S = VEC ? 1 : 16;
    const int r0 = blockIdx.x * 128, c = blockIdx.y * 128 + (threadIdx.x & 15) * (VEC ? 8 : 1);
    F8Raw<T> d[8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = r0 + (threadIdx.x >> 4) + 16 * i;
        if (r < a.n_rows) {
            d[i] = f8_load<T, S>(static_cast<const T *>(a.x) + r * a.xs + c, a.n_cols - c);
            top = max(top, f8_top(d[i]));
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kF8Threads / 32; ++i) top = max(top, warp_top[i]);
    const F8Scale f = f8_scale<sizeof(T) == 2>(f8_top_f32<T>(top));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = r0 + (threadIdx.x >> 4) + 16 * i;
        if (r >= a.n_rows) break;
        f8_store<T, S>(a.q + r * a.qs + c, a.n_cols - c, d[i], f);
    }
    if (threadIdx.x == 0) a.scale[(int64_t)blockIdx.x * a.nb + blockIdx.y] = f.s;
}

}  // namespace rb

using namespace rb;

extern "C" int rabbit_cuda_f8_quantise_dev(int dtype, const void *d_x, int64_t x_stride, int x_rows,
                                           const int *d_rows, void *d_q, int64_t q_stride,
                                           float *d_scale, int n_rows, int n_cols, int block_rows,
                                           void *stream) {
    const int size = dtype_size(dtype);
    if (!size || n_rows < 0 || n_cols < 1 || n_cols > 1 << 20 || (block_rows != 1 && block_rows != 128))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "f8_quantise: unknown dtype, n_rows below 0, n_cols not in 1..2^20 or block_rows "
                    "not 1 or 128");
    if (n_rows == 0) return ok();
    if (!d_x || !d_q || !d_scale) return fail(RABBIT_CUDA_ERR_ARGS, "f8_quantise: NULL pointer");
    if (d_rows && (block_rows != 1 || x_rows < 1))
        return fail(RABBIT_CUDA_ERR_ARGS, "f8_quantise: d_rows needs block_rows 1 and x_rows above 0");
    F8Args a;
    a.x = d_x;
    a.xs = x_stride ? x_stride : n_cols;
    a.rows = d_rows;
    a.x_rows = x_rows;
    a.q = static_cast<uint8_t *>(d_q);
    a.qs = q_stride ? q_stride : n_cols;
    a.scale = d_scale;
    a.n_rows = n_rows;
    a.n_cols = n_cols;
    a.nb = (n_cols + 127) / 128;
    if ((int64_t)n_rows * a.nb >= (int64_t)1 << 31)
        return fail(RABBIT_CUDA_ERR_ARGS, "f8_quantise: 2^31 blocks or more");
    const uintptr_t x = reinterpret_cast<uintptr_t>(d_x), q = reinterpret_cast<uintptr_t>(d_q);
    if (a.xs < n_cols || a.qs < n_cols || (x & (size - 1)) ||
        (reinterpret_cast<uintptr_t>(d_scale) & 3) || (reinterpret_cast<uintptr_t>(d_rows) & 3))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "f8_quantise: a stride below n_cols, or a pointer not aligned to its element");
    // i / nb as a product: with 2^(31 + l) / nb rounded up, 2^l >= nb, exact below 2^31
    int l = 0;
    while ((1 << l) < a.nb) ++l;
    a.magic = a.nb == 1 ? 0 : (uint32_t)((((uint64_t)1 << (31 + l)) + a.nb - 1) / a.nb);
    a.shift = l - 1;
    const bool vec = (x & 15) == 0 && a.xs * size % 16 == 0 && (q & 7) == 0 && a.qs % 8 == 0;
    const int sms = device_sms();
    if (!sms) return fail(RABBIT_CUDA_ERR_DEVICE, "f8_quantise: no device %d", current_device());
    DeviceScope scope(current_device());
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    // Rows: blocks are handed out warp by warp, in one wave of the SMs at most.
    const int64_t ctas = ((int64_t)n_rows * a.nb + kF8Threads / 8 - 1) / (kF8Threads / 8);
    const dim3 grid = block_rows == 1 ? dim3((unsigned)(ctas < kF8Resident * sms ? ctas : kF8Resident * sms))
                                      : dim3((n_rows - 1) / 128 + 1, a.nb);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        auto k = block_rows == 1 ? (vec ? k_f8_rows<T, true> : k_f8_rows<T, false>)
                                 : (vec ? k_f8_blocks<T, true> : k_f8_blocks<T, false>);
        scope.launch(launch_pdl(k, grid, dim3(kF8Threads), 0, static_cast<cudaStream_t>(stream), a),
                     "f8_quantise");
        return 0;
    });
    return scope.done();
}
