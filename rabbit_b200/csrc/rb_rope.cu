// rb_rope.cu -- C ABI: rotary positions (rope_rotate, src/forward_v2.c:92-104,
// generalised: both pair layouts, part of the head, scaled frequencies, three
// element types).
#include <math.h>

#include <new>

#include "rb_device.cuh"
#include "rb_launch.h"
#include "rb_rope.h"
#include "rb_runtime.h"
#include "rb_types.cuh"

struct rabbit_cuda_rope {
    rb::RopeTab tab;
    int head_dim;
    double freq[rb::kRopeMaxPairs];
};

namespace rb {

const RopeTab &rope_tab(const rabbit_cuda_rope *r, int *head_dim) {
    *head_dim = r->head_dim;
    return r->tab;
}

struct RopeArgs {
    RopeTab tab;
    const void *x;
    void *y;
    const int *pos;
    int64_t xs, ys;  // elements between rows
    int T, heads, hd;
    int tpc;         // tokens per CTA
    int nrot, per;   // items of a head that rotate, and all of them
};

constexpr int kRopeThreads = 256;

// Bound by memory: each element is read and written once. One CTA takes tpc
// tokens (and a part of a token's items, blockIdx.y): their angles are made in 64
// bits and shared by the heads; then a thread keeps its item of the row and goes
// through the tokens, BATCH of them in flight. An item is V channels (16 bytes;
// scalar form: one) that rotate with V others (HALF), or 16 bytes of whole pairs
// (INTERLEAVED; scalar form: one pair), or 16 bytes of the rest to copy.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(kRopeThreads, 4) k_rope(const __grid_constant__ RopeArgs a) {
    extern __shared__ __align__(16) float2 cs[];  // [tpc][rot / 2]
    // a vector holds one side of V pairs (HALF), or both sides of V / 2 (the scalar
    // form has two elements of one pair)
    constexpr int NV = HALF || V == 1 ? 2 : 1;    // vectors of an item
    constexpr int NP = NV == 2 ? V : V / 2;       // pairs of an item
    constexpr int BATCH = 4 / NV;
    struct alignas(V * sizeof(T)) Vec {
        T e[V];
    };
    launch_dependents();
    wait_prerequisite();
    const int np = a.tab.rot / 2, t0 = blockIdx.x * a.tpc, nt = min(a.tpc, a.T - t0);
    for (int i = threadIdx.x; i < nt * np; i += kRopeThreads) {
        const int t = i / np;
        const double2 k = rope_cs(a.pos[t0 + t], a.tab.turns[i - t * np]);
        cs[i] = make_float2((float)(k.x * a.tab.mag), (float)(k.y * a.tab.mag));
    }
    __syncthreads();
    const int row = a.heads * a.per, second = HALF ? np : V;
    // short rows: several tokens side by side
    const int side = row <= kRopeThreads / 2 ? kRopeThreads / row : 1;
    const int first = side > 1 ? threadIdx.x / row : 0;
    if (first >= side) return;
    for (int r = side > 1 ? threadIdx.x - first * row : blockIdx.y * kRopeThreads + threadIdx.x; r < row;
         r += gridDim.y * kRopeThreads) {
        const int h = r / a.per, u = r - h * a.per;
        const bool turn = u < a.nrot;
        const int c = h * a.hd + (turn ? (HALF ? u * V : u * V * NV) : a.tab.rot + (u - a.nrot) * V);
        const float2 *k0 = cs + (turn ? u * NP : 0);
        const T *x = static_cast<const T *>(a.x) + (int64_t)(t0 + first) * a.xs + c;
        T *y = static_cast<T *>(a.y) + (int64_t)(t0 + first) * a.ys + c;
        for (int t = first; t < nt; t += BATCH * side) {
            Vec v[BATCH][NV];
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
                if (t + b * side < nt) {
                    const T *at = x + b * side * a.xs;
                    v[b][0] = *reinterpret_cast<const Vec *>(at);
                    if (NV == 2 && turn) v[b][NV - 1] = *reinterpret_cast<const Vec *>(at + second);
                }
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                if (t + b * side >= nt) continue;
                T *to = y + b * side * a.ys;
                if (turn) {
                    const float2 *kt = k0 + (t + b * side) * np;
                    float2 ks[NP];
                    if constexpr (NP % 2 == 0) {  // an even pair of the table
#pragma unroll
                        for (int e = 0; e < NP; e += 2) {
                            const float4 k = *reinterpret_cast<const float4 *>(kt + e);
                            ks[e] = make_float2(k.x, k.y);
                            ks[e + 1] = make_float2(k.z, k.w);
                        }
                    } else {
                        ks[0] = kt[0];
                    }
#pragma unroll
                    for (int e = 0; e < NP; ++e) {
                        T &e1 = v[b][0].e[NV == 2 ? e : 2 * e], &e2 = NV == 2 ? v[b][NV - 1].e[e] : v[b][0].e[(2 * e + 1) % V];
                        const float x1 = to_f32(e1), x2 = to_f32(e2);
                        e1 = from_f32<T>(x1 * ks[e].x - x2 * ks[e].y);
                        e2 = from_f32<T>(x2 * ks[e].x + x1 * ks[e].y);
                    }
                    if (NV == 2) *reinterpret_cast<Vec *>(to + second) = v[b][NV - 1];
                }
                *reinterpret_cast<Vec *>(to) = v[b][0];
            }
            x += BATCH * side * a.xs;
            y += BATCH * side * a.ys;
        }
    }
}

}  // namespace rb

using namespace rb;

extern "C" {

int rabbit_cuda_rope_create(const rabbit_cuda_rope_desc *d, rabbit_cuda_rope **out) {
    if (!d || !out) return fail(RABBIT_CUDA_ERR_ARGS, "rope_create: NULL argument");
    *out = nullptr;
    const int rot = d->rot_dim ? d->rot_dim : d->head_dim;
    if (d->head_dim < 2 || d->head_dim > 1024 || rot < 2 || (rot & 1) || rot > d->head_dim ||
        rot > 2 * kRopeMaxPairs)
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "rope_create: need head_dim in 2..1024 and an even rot_dim in 2..%d of it",
                    2 * kRopeMaxPairs);
    if (d->layout != RABBIT_CUDA_ROPE_INTERLEAVED && d->layout != RABBIT_CUDA_ROPE_HALF)
        return fail(RABBIT_CUDA_ERR_ARGS, "rope_create: unknown layout %d", d->layout);
    double base = d->base == 0.0 ? 10000.0 : d->base;
    const double factor = d->factor == 0.0 ? 1.0 : d->factor;
    if (!(base > 1.0) || !isfinite(base) || !(factor > 0.0) || !isfinite(factor) ||
        !isfinite(d->magnitude))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "rope_create: need base above 1, a positive factor, a finite magnitude");
    const int sc = d->scaling;
    if (sc < RABBIT_CUDA_ROPE_SCALE_NONE || sc > RABBIT_CUDA_ROPE_SCALE_YARN)
        return fail(RABBIT_CUDA_ERR_ARGS, "rope_create: unknown scaling %d", sc);
    const bool bands = sc == RABBIT_CUDA_ROPE_SCALE_BANDS, yarn = sc == RABBIT_CUDA_ROPE_SCALE_YARN;
    const double low = d->low == 0.0 ? 1.0 : d->low;
    const double high = d->high == 0.0 ? (yarn ? 32.0 : 4.0) : d->high;
    if ((bands || yarn) && (d->original_ctx < 1 || !(low > 0.0) || !(high > low) || !isfinite(high)))
        return fail(RABBIT_CUDA_ERR_ARGS, "rope_create: need original_ctx > 0 and 0 < low < high");
    if (sc == RABBIT_CUDA_ROPE_SCALE_NTK) {
        if (rot < 4)
            return fail(RABBIT_CUDA_ERR_ARGS, "rope_create: base scaling needs rot_dim above 2");
        base *= pow(factor, rot / (rot - 2.0));
    }
    const double two_pi = 6.283185307179586476925286766559;
    const double ctx = d->original_ctx;
    double lo_pair = 0.0, hi_pair = 0.0;  // YaRN: the ramp over pair indices
    if (yarn) {
        lo_pair = floor(rot * log(ctx / (high * two_pi)) / (2.0 * log(base)));
        hi_pair = ceil(rot * log(ctx / (low * two_pi)) / (2.0 * log(base)));
        if (lo_pair < 0.0) lo_pair = 0.0;
        if (hi_pair > rot - 1.0) hi_pair = rot - 1.0;
    }
    auto *r = new (std::nothrow) rabbit_cuda_rope();
    if (!r) return fail(RABBIT_CUDA_ERR_MEM, "rope_create: out of host memory");
    r->head_dim = d->head_dim;
    r->tab.rot = rot;
    r->tab.layout = d->layout;
    r->tab.mag = d->magnitude != 0.0 ? d->magnitude
                 : yarn && factor > 1.0 ? 1.0 + 0.1 * log(factor)
                                        : 1.0;
    for (int i = 0; i < rot / 2; ++i) {
        double f = pow(base, -2.0 * i / rot), keep = 1.0;  // keep: share of the unscaled frequency
        if (sc == RABBIT_CUDA_ROPE_SCALE_LINEAR) keep = 0.0;
        if (bands) keep = (ctx * f / two_pi - low) / (high - low);
        if (yarn) {
            const double w = hi_pair - lo_pair;
            keep = 1.0 - (i - lo_pair) / (w > 0.001 ? w : 0.001);
        }
        keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        f = keep * f + (1.0 - keep) * (f / factor);
        r->freq[i] = f;
        r->tab.turns[i] = f / two_pi;
    }
    *out = r;
    return ok();
}

int rabbit_cuda_rope_free(rabbit_cuda_rope *r) {
    delete r;
    return ok();
}

int rabbit_cuda_rope_freqs(const rabbit_cuda_rope *r, double *freq, double *magnitude) {
    if (!r) return fail(RABBIT_CUDA_ERR_ARGS, "rope_freqs: NULL rope");
    for (int i = 0; freq && i < r->tab.rot / 2; ++i) freq[i] = r->freq[i];
    if (magnitude) *magnitude = r->tab.mag;
    return ok();
}

int rabbit_cuda_rope_dev(const rabbit_cuda_rope *r, int dtype, const void *d_x, int64_t x_stride,
                         void *d_y, int64_t y_stride, const int *d_positions, int n_tokens,
                         int n_heads, void *stream) {
    if (!r || !dtype_size(dtype) || n_tokens < 0 || n_heads < 1 || n_heads > 65536)
        return fail(RABBIT_CUDA_ERR_ARGS, "rope_dev: NULL rope, unknown dtype or a bad count");
    if (n_tokens == 0) return ok();
    if (!d_x || !d_y || !d_positions)
        return fail(RABBIT_CUDA_ERR_ARGS, "rope_dev: NULL pointer");
    RopeArgs a;
    a.tab = r->tab;
    a.hd = r->head_dim;
    const int64_t row = (int64_t)n_heads * a.hd;
    a.xs = x_stride ? x_stride : row;
    a.ys = y_stride ? y_stride : row;
    const int size = dtype_size(dtype);
    const uintptr_t off = reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_y);
    if (a.xs < row || a.ys < row || (off & (size - 1)) ||
        (reinterpret_cast<uintptr_t>(d_positions) & 3) || (d_x == d_y && a.xs != a.ys))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "rope_dev: strides below n_heads * head_dim (or different in place), or a "
                    "pointer not aligned to its element");
    a.x = d_x;
    a.y = d_y;
    a.pos = d_positions;
    a.T = n_tokens;
    a.heads = n_heads;
    const bool half = a.tab.layout == RABBIT_CUDA_ROPE_HALF;
    // 16-byte vectors where rows, heads and both sides of the pairs allow them
    const int side = half ? a.tab.rot / 2 : a.tab.rot;
    const bool vec = (off & 15) == 0 && a.xs * size % 16 == 0 && a.ys * size % 16 == 0 &&
                     a.hd * size % 16 == 0 && side * size % 16 == 0 && a.tab.rot * size % 16 == 0;
    const int V = vec ? 16 / size : 1;
    a.nrot = half || !vec ? a.tab.rot / 2 / V : a.tab.rot / V;
    a.per = a.nrot + (d_x != d_y ? (a.hd - a.tab.rot) / V : 0);
    // Tokens per CTA: all tokens in one wave of four CTAs an SM (a CTA makes its
    // tokens' angles before it can rotate, so few and long ones), up to 32; where
    // there are fewer tokens than SMs, a token's items are spread over blockIdx.y,
    // up to a CTA an SM in all. 16384 x 32 x 128 bf16: 28 tokens a CTA 55 us (4.9
    // TB/s), 2 tokens 74 us.
    const int64_t items = (int64_t)n_heads * a.per;
    int sms = 0;
    DeviceScope scope(current_device());
    if (scope.status == RABBIT_CUDA_OK)
        scope.launch(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, current_device()), "rope_dev: SM count");
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    const int64_t wave = ((int64_t)n_tokens + 4 * sms - 1) / (4 * sms);
    const int most = 48 * 1024 / (int)(sizeof(float2) * (a.tab.rot / 2));  // their angles' shared memory
    a.tpc = wave > 32 ? 32 : (int)wave;
    if (a.tpc > most) a.tpc = most;
    const int groups = (int)(((int64_t)n_tokens + a.tpc - 1) / a.tpc);
    int64_t split = (items + kRopeThreads - 1) / kRopeThreads;
    if (split > sms / groups) split = sms / groups;
    const dim3 grid(groups, split < 1 ? 1 : (unsigned)split);
    const size_t smem = sizeof(float2) * (size_t)a.tpc * (a.tab.rot / 2);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int VT = 16 / sizeof(T);
        auto k = half ? (vec ? k_rope<T, VT, true> : k_rope<T, 1, true>)
                      : (vec ? k_rope<T, VT, false> : k_rope<T, 1, false>);
        scope.launch(launch_pdl(k, grid, dim3(kRopeThreads), smem, static_cast<cudaStream_t>(stream), a),
                     "rope_dev");
        return 0;
    });
    return scope.done();
}

}  // extern "C"
