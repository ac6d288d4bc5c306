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
    int tpc;       // tokens per CTA
    bool copy;     // y is not x: the channels that do not rotate are copied
};

constexpr int kRopeThreads = 256;

// One CTA: tpc tokens. Their angles once into shared memory, then a thread per
// pair of a (token, head).
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) k_rope(const __grid_constant__ RopeArgs a) {
    extern __shared__ __align__(16) float2 cs[];  // [tpc][rot / 2]
    launch_dependents();
    wait_prerequisite();
    const int np = a.tab.rot / 2, t0 = blockIdx.x * a.tpc, nt = min(a.tpc, a.T - t0);
    for (int i = threadIdx.x; i < nt * np; i += kRopeThreads) {
        const double2 v = rope_cs(a.pos[t0 + i / np], a.tab.turns[i % np]);
        cs[i] = make_float2((float)(v.x * a.tab.mag), (float)(v.y * a.tab.mag));
    }
    __syncthreads();
    const int rest = a.copy ? a.hd - a.tab.rot : 0, per = np + rest;
    const bool half = a.tab.layout == RABBIT_CUDA_ROPE_HALF;
    for (int64_t i = threadIdx.x; i < (int64_t)nt * a.heads * per; i += kRopeThreads) {
        const int u = (int)(i % per), h = (int)(i / per % a.heads), t = (int)(i / per / a.heads);
        const T *x = static_cast<const T *>(a.x) + (t0 + t) * a.xs + (int64_t)h * a.hd;
        T *y = static_cast<T *>(a.y) + (t0 + t) * a.ys + (int64_t)h * a.hd;
        if (u >= np) {
            y[a.tab.rot + u - np] = x[a.tab.rot + u - np];
            continue;
        }
        const int c1 = half ? u : 2 * u, c2 = half ? u + np : 2 * u + 1;
        const float x1 = to_f32(x[c1]), x2 = to_f32(x[c2]);
        const float2 v = cs[t * np + u];
        y[c1] = from_f32<T>(x1 * v.x - x2 * v.y);
        y[c2] = from_f32<T>(x2 * v.x + x1 * v.y);
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
    const uintptr_t off = reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_y);
    if (a.xs < row || a.ys < row || (off & (dtype_size(dtype) - 1)) || (d_x == d_y && a.xs != a.ys))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "rope_dev: strides below n_heads * head_dim (or different in place), or a "
                    "pointer not aligned to its element");
    a.x = d_x;
    a.y = d_y;
    a.pos = d_positions;
    a.T = n_tokens;
    a.heads = n_heads;
    a.copy = d_x != d_y;
    a.tpc = 1;
    DeviceScope scope(current_device());
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    const size_t smem = sizeof(float2) * (size_t)a.tpc * (a.tab.rot / 2);
    with_dtype(dtype, [&](auto t) {
        scope.launch(launch_pdl(k_rope<decltype(t)>, dim3((n_tokens + a.tpc - 1) / a.tpc),
                                dim3(kRopeThreads), smem, static_cast<cudaStream_t>(stream), a),
                     "rope_dev");
        return 0;
    });
    return scope.done();
}

}  // extern "C"
