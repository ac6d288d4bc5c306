// rb_f8.cu -- C ABI: rows and blocks as e4m3 codes with a scale for each 128
// columns.
//
// Bound by memory: x is read and its codes are written once. The codes are those of the
// exact quotient x / s without a division for each value: with r within 2^-22 of 1 / s,
//   |x| r (1 - 2^-21) <= |x| / s <= |x| r (1 + 2^-21)
// holds for the computed products (they round by 2^-24 each), rounding to
// e4m3 is monotone, so where both ends give one code it is the quotient's. Where they give two
// neighbours, the sign of x - m s, m the middle between them, decides; one fma has it exactly.
// 16384 rows of 4096 bf16: see the launch below.
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

constexpr int kF8Threads = 256;
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
    float s, lo, hi;
    bool zero, bad, tiny;
};
constexpr float kF8Tiny = 0x1p-60f, kF8Grow = 0x1p64f;
__device__ __forceinline__ F8Scale f8_scale(uint32_t top) {
    F8Scale f;
    f.bad = top >= kInfBits;
    // top / 448 to nearest: a product and one correction (equal to the division for every
    // mantissa while nothing falls below fp32's normal numbers)
    const float t = __uint_as_float(top), q = t * (1.f / 448.f);
    f.s = fmaf(fmaf(-q, 448.f, t), 1.f / 448.f, q);
    if (t < 0x1p-100f) f.s = __fdiv_rn(t, 448.f);
    if (f.bad) f.s = __uint_as_float(0x7FC00000u);
    f.zero = f.s == 0.f;
    // below 2^-60 x and s are multiplied by 2^64, where 1 / s and the remainders are far from
    // fp32's smallest numbers
    f.tiny = f.s < kF8Tiny;
    const float r = __fdividef(1.f, f.tiny ? f.s * kF8Grow : f.s);
    f.lo = r * (1.f - 0x1p-21f);
    f.hi = r * (1.f + 0x1p-21f);
    return f;
}

// Codes of eight values, the first in the low byte.
__device__ __forceinline__ uint2 f8_codes(float (&x)[8], const F8Scale &f) {
    if (f.bad | f.zero) return f.bad ? make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu) : make_uint2(0u, 0u);
    float s = f.s;
    if (f.tiny) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= kF8Grow;
        s *= kF8Grow;
    }
    uint32_t a[2], b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float *v = x + 4 * i;
        a[i] = e4m3x2(v[0] * f.lo, v[1] * f.lo) | e4m3x2(v[2] * f.lo, v[3] * f.lo) << 16;
        b[i] = e4m3x2(v[0] * f.hi, v[1] * f.hi) | e4m3x2(v[2] * f.hi, v[3] * f.hi) << 16;
    }
    // one at a time: of 16-bit values, whose quotients are often ties, a lane has one or two
    uint64_t d = (uint64_t)(a[1] ^ b[1]) << 32 | (a[0] ^ b[0]);
    while (d) {
        const int i = (__ffsll((long long)d) - 1) >> 3, sh = 8 * (i & 3);
        d &= ~(0xFFull << (8 * i));
        float v = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) v = i == j ? x[j] : v;
        const uint32_t word = i < 4 ? a[0] : a[1], c = word >> sh & 255;  // below m; above it c + 1
        const float m = 0.5f * (fabsf(e4m3_value(c)) + fabsf(e4m3_value(c + 1)));
        const float r = fmaf(-m, s, fabsf(v));
        const uint32_t up = (r > 0.f || (r == 0.f && (c & 1))) ? 1u << sh : 0u;
        if (i < 4) a[0] += up;
        else a[1] += up;
    }
    return make_uint2(a[0], a[1]);
}

// Eight values of a row as they lie in memory, from column c on; past the row zeros.
template <typename T>
struct F8Raw {
    uint4 w[sizeof(T) / 2];
};
template <typename T, bool VEC>
__device__ __forceinline__ F8Raw<T> f8_load(const T *row, int c, int n_cols) {
    F8Raw<T> d;
    if (VEC && c + 8 <= n_cols) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) d.w[i] = reinterpret_cast<const uint4 *>(row + c)[i];
    } else {
        T *e = reinterpret_cast<T *>(&d);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = c + i < n_cols ? row[c + i] : from_f32<T>(0.f);
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
template <bool VEC>
__device__ __forceinline__ void f8_store(uint8_t *row, int c, int n_cols, uint2 w) {
    if (VEC && c + 8 <= n_cols) {
        *reinterpret_cast<uint2 *>(row + c) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < n_cols) row[c + i] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    }
}

// One scale for each row's block: eight lanes hold a block, a lane columns 8 l .. and
// 64 + 8 l .. of it; BATCH blocks of each eight lanes are in flight.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kF8Threads) k_f8_rows(const __grid_constant__ F8Args a) {
    constexpr int BATCH = 2;
    launch_dependents();
    wait_prerequisite();
    const int64_t items = (int64_t)a.n_rows * a.nb;
    const int lane = threadIdx.x & 7;
    const int64_t teams = (int64_t)gridDim.x * (kF8Threads / 8);
    for (int64_t i0 = ((int64_t)blockIdx.x * kF8Threads + threadIdx.x) / 32 * 4; i0 < items;
         i0 += teams * BATCH) {
        F8Raw<T> d[BATCH][2];
        int64_t at[BATCH];
        int block[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {  // a warp's four blocks side by side, then `teams` on
            const int64_t i = i0 + (threadIdx.x >> 3 & 3) + b * teams;
            at[b] = -1;
            if (i < items) {
                const int64_t r = items >> 31 ? i / a.nb : a.nb == 1 ? i : __umulhi((uint32_t)i, a.magic) >> a.shift;
                block[b] = (int)(i - r * a.nb);
                const int64_t src = a.rows ? __ldg(a.rows + r) : r;
                if (!a.rows || (src >= 0 && src < a.x_rows)) {
                    at[b] = r;
                    const T *row = static_cast<const T *>(a.x) + src * a.xs;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        d[b][h] = f8_load<T, VEC>(row, block[b] * 128 + h * 64 + lane * 8, a.n_cols);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            uint32_t top = at[b] >= 0 ? max(f8_top(d[b][0]), f8_top(d[b][1])) : 0u;
#pragma unroll
            for (int m = 4; m; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
            if (at[b] < 0) continue;
            const F8Scale f = f8_scale(f8_top_f32<T>(top));
            uint8_t *q = a.q + at[b] * a.qs;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
                f8_values(d[b][h], v);
                f8_store<VEC>(q, block[b] * 128 + h * 64 + lane * 8, a.n_cols, f8_codes(v, f));
            }
            if (lane == 0) a.scale[at[b] * a.nb + block[b]] = f.s;
        }
    }
}

// One scale for each 128 rows x 128 columns: a CTA holds the block in registers.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kF8Threads) k_f8_blocks(const __grid_constant__ F8Args a) {
    __shared__ uint32_t warp_top[kF8Threads / 32];
    launch_dependents();
    wait_prerequisite();
    const int r0 = blockIdx.x * 128, c = blockIdx.y * 128 + (threadIdx.x & 15) * 8;
    F8Raw<T> d[8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = r0 + (threadIdx.x >> 4) + 16 * i;
        if (r < a.n_rows) {
            d[i] = f8_load<T, VEC>(static_cast<const T *>(a.x) + r * a.xs, c, a.n_cols);
            top = max(top, f8_top(d[i]));
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kF8Threads / 32; ++i) top = max(top, warp_top[i]);
    const F8Scale f = f8_scale(f8_top_f32<T>(top));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = r0 + (threadIdx.x >> 4) + 16 * i;
        if (r >= a.n_rows) break;
        float v[8];
        f8_values(d[i], v);
        f8_store<VEC>(a.q + r * a.qs, c, a.n_cols, f8_codes(v, f));
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
    int sms = 0;
    DeviceScope scope(current_device());
    if (scope.status == RABBIT_CUDA_OK)
        scope.launch(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, current_device()), "f8_quantise: SM count");
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    // Rows: blocks are handed out warp by warp, in one wave of the SMs at most.
    const int64_t ctas = ((int64_t)n_rows * a.nb + kF8Threads / 8 - 1) / (kF8Threads / 8);
    const dim3 grid = block_rows == 1 ? dim3((unsigned)(ctas < 8 * sms ? ctas : 8 * sms))
                                      : dim3((n_rows + 127) / 128, a.nb);
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
