// rb_kv4.cu -- C ABI: the paged 4-bit key / value cache; appending to it with
// the rotation of the keys on the way, and reading rows back.
#include <new>

#include "rb_device.cuh"
#include "rb_kv4.cuh"
#include "rb_launch.h"
#include "rb_rope.h"
#include "rb_types.cuh"

namespace rb {

constexpr int kAppendThreads = 256;

struct Kv4AppendArgs {
    Kv4View c;
    const void *x[2];   // keys, values
    int64_t xs[2];
    const int64_t *slots;
    const int *pos;     // NULL: keys as they are
    int T, tpc;         // tokens, tokens per CTA
};

struct Kv4AppendRopeArgs {
    Kv4AppendArgs a;
    RopeTab tab;
};

// rint(x / s) of the real quotient, halves to even. The fp32 product with the
// reciprocal is within 2^-20 of the quotient (|x / s| < 8), so only a quotient
// within 2^-12 of a half needs the division in 64 bits. Scales near the
// smallest fp32 have no finite reciprocal and always take it.
__device__ __forceinline__ int kv4_code(double x, float s, float inv) {
    const float t = (float)x * inv;
    float q = rintf(t);
    if (fabsf(fabsf(t - q) - 0.5f) < 2.44140625e-4f || s < 1e-30f) q = (float)rint(x / (double)s);
    return (int)q;
}

// A thread: 8 consecutive channels of one (token, head) of the keys
// (blockIdx.z = 0) or the values; 4 threads a group.
template <typename T, bool VEC, bool ROPE>
__global__ void __launch_bounds__(kAppendThreads) k_kv4_append(const __grid_constant__ Kv4AppendRopeArgs aa) {
    extern __shared__ __align__(16) double2 cs[];  // [tpc][rot / 2], keys only
    const Kv4AppendArgs &a = aa.a;
    const RopeTab &tab = aa.tab;
    const Kv4View &c = a.c;
    launch_dependents();
    wait_prerequisite();
    const int kv = blockIdx.z, t0 = blockIdx.x * a.tpc, nt = min(a.tpc, a.T - t0);
    const bool rot = ROPE && kv == 0;
    const int np = ROPE ? tab.rot / 2 : 0;
    if constexpr (ROPE) {
        if (rot) {
            for (int i = threadIdx.x; i < nt * np; i += kAppendThreads) {
                double2 v = rope_cs(a.pos[t0 + i / np], tab.turns[i % np]);
                v.x *= tab.mag;
                v.y *= tab.mag;
                cs[i] = v;
            }
            __syncthreads();
        }
    }
    const int per = c.nkv * c.ng * 4, total = nt * per;
    const bool halves = ROPE && tab.layout == RABBIT_CUDA_ROPE_HALF;
    for (int i0 = blockIdx.y * kAppendThreads; i0 < total; i0 += gridDim.y * kAppendThreads) {
        const int i = i0 + threadIdx.x;
        const bool in = i < total;
        const int tl = in ? i / per : 0, u = in ? i - tl * per : 0;
        const int head = u / (c.ng * 4), w = u - head * c.ng * 4, grp = w >> 2, t = w & 3;
        const int c0 = 8 * w;  // first channel
        const int64_t slot = in ? a.slots[t0 + tl] : -1;
        const bool write = slot >= 0 && slot < c.slots();
        if (in && slot >= c.slots() && c.err) atomicOr(c.err, RB_KV4_ERR_SLOT);
        double x[8];
        uint32_t top = 0;  // bits of max |x|: an integer maximum keeps a NaN
#pragma unroll
        for (int n = 0; n < 8; ++n) x[n] = 0.0;
        if (write && c0 < c.hd) {
            const T *row = static_cast<const T *>(a.x[kv]) + (t0 + tl) * a.xs[kv] + (int64_t)head * c.hd;
            float v[8];
            load8<VEC>(v, row + c0);
#pragma unroll
            for (int n = 0; n < 8; ++n) x[n] = v[n];
            if (rot && c0 < tab.rot) {
                // partners: the other channel of each pair
                float p[8];
                if (!halves) {
#pragma unroll
                    for (int n = 0; n < 8; ++n) p[n] = v[n ^ 1];
                } else if (np % 8 == 0) {
                    load8<VEC>(p, row + (c0 < np ? c0 + np : c0 - np));
                } else {
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const int ch = c0 + n;
                        p[n] = ch < tab.rot ? to_f32(row[ch < np ? ch + np : ch - np]) : 0.f;
                    }
                }
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const int ch = c0 + n;
                    if (ch < tab.rot) {
                        const bool first = halves ? ch < np : !(ch & 1);
                        const double2 k = cs[tl * np + (halves ? (first ? ch : ch - np) : ch >> 1)];
                        x[n] = (double)v[n] * k.x + (double)p[n] * (first ? -k.y : k.y);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) top = max(top, __float_as_uint(fabsf((float)x[n])));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (!write) continue;
        // a group with an infinity or a NaN has a NaN for its scale
        const float top7 = __fmul_rn(__uint_as_float(top), 1.0f / 7.0f);
        const __nv_bfloat16 sb = __float2bfloat16_rn(top7 < INFINITY ? top7 : __uint_as_float(0x7fc00000u));
        const float s = __bfloat162float(sb), inv = 1.0f / s;
        uint32_t word = 0x88888888u;
        if (s > 0.f) {
            word = 0;
#pragma unroll
            for (int n = 0; n < 8; ++n) word |= (uint32_t)(kv4_code(x[n], s, inv) + 8) << (4 * n);
        }
        const int64_t pg = slot / c.page;
        const int j = (int)(slot - pg * c.page) & (kKv4Granule - 1);
        uint8_t *g = c.granule(slot, head) + (kv ? kv4_v(c.ng) : 0);
        uint8_t *codes = g + j * kv4_row(c.ng);
        if (kv == 0) {
            reinterpret_cast<uint32_t *>(codes)[t * c.ng + grp] = word;
        } else {
            uint16_t *h = reinterpret_cast<uint16_t *>(codes);
            h[kv4_vplace(j, 2 * t) * c.ng + grp] = (uint16_t)word;
            h[kv4_vplace(j, 2 * t + 1) * c.ng + grp] = (uint16_t)(word >> 16);
        }
        if (t == 0)
            reinterpret_cast<__nv_bfloat16 *>(g + kv4_ks(c.ng))[j * c.ng + grp] = sb;
    }
}

struct Kv4ReadArgs {
    Kv4View c;
    void *y[2];
    const int64_t *slots;
    int T;
};

// A thread: 8 channels of one (token, head); keys in y[0], values in y[1].
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_kv4_read(const __grid_constant__ Kv4ReadArgs a) {
    launch_dependents();
    wait_prerequisite();
    const Kv4View &c = a.c;
    const int kv = blockIdx.z, per = c.nkv * c.ng * 4;
    if (!a.y[kv]) return;
    const int64_t total = (int64_t)a.T * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int tl = (int)(i / per), u = (int)(i - (int64_t)tl * per);
        const int head = u / (c.ng * 4), w = u - head * c.ng * 4, grp = w >> 2, t = w & 3;
        const int64_t slot = a.slots[tl];
        if (slot < 0 || 8 * w >= c.hd) continue;
        if (slot >= c.slots()) {
            atomicOr(c.err, RB_KV4_ERR_SLOT);
            continue;
        }
        const int j = (int)(slot % c.page) & (kKv4Granule - 1);
        const uint8_t *g = c.granule(slot, head) + (kv ? kv4_v(c.ng) : 0);
        const uint8_t *codes = g + j * kv4_row(c.ng);
        uint32_t word;
        if (kv == 0) {
            word = reinterpret_cast<const uint32_t *>(codes)[t * c.ng + grp];
        } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(codes);
            word = h[kv4_vplace(j, 2 * t) * c.ng + grp] |
                   (uint32_t)h[kv4_vplace(j, 2 * t + 1) * c.ng + grp] << 16;
        }
        const float s = __bfloat162float(
            reinterpret_cast<const __nv_bfloat16 *>(g + kv4_ks(c.ng))[j * c.ng + grp]);
        float v[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) v[n] = (float)((int)(word >> (4 * n) & 15u) - 8) * s;
        store8<VEC>(static_cast<T *>(a.y[kv]) + (int64_t)tl * c.nkv * c.hd + head * c.hd + 8 * w, v);
    }
}

static bool aligned(const void *p, uintptr_t n) {
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

}  // namespace rb

using namespace rb;

extern "C" {

int rabbit_cuda_kv4_create(const rabbit_cuda_kv4_desc *d, int device, rabbit_cuda_kv4 **out) {
    if (!d || !out) return fail(RABBIT_CUDA_ERR_ARGS, "kv4_create: NULL argument");
    *out = nullptr;
    if (d->n_layers < 1 || d->n_layers > 65536 || d->n_kv_heads < 1 || d->n_kv_heads > 1024 ||
        d->head_dim < 8 || d->head_dim > 32 * kKv4MaxGroups || (d->head_dim & 7) ||
        d->page_size < 16 || d->page_size > 1024 || (d->page_size & 15) || d->n_pages < 1)
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "kv4_create: need n_layers >= 1, n_kv_heads in 1..1024, head_dim a multiple of "
                    "8 up to %d, page_size a multiple of 16 up to 1024, n_pages >= 1",
                    32 * kKv4MaxGroups);
    int prev = 0;
    cudaGetDevice(&prev);
    int st;
    DevCtx *ctx = dev_ctx(device, &st);
    if (!ctx) {
        cudaSetDevice(prev);
        return st;
    }
    auto *c = new (std::nothrow) rabbit_cuda_kv4();
    if (!c) {
        cudaSetDevice(prev);
        return fail(RABBIT_CUDA_ERR_MEM, "kv4_create: out of host memory");
    }
    c->device = device;
    c->ctx = ctx;
    c->n_layers = d->n_layers;
    c->view.nkv = d->n_kv_heads;
    c->view.hd = d->head_dim;
    c->view.ng = (d->head_dim + kKv4Group - 1) / kKv4Group;
    c->view.page = d->page_size;
    c->view.n_pages = d->n_pages;
    c->layer_bytes = (size_t)d->n_pages * c->view.page_bytes();
    const size_t bytes = (size_t)d->n_layers * c->layer_bytes;
    void *base = nullptr;
    cudaError_t e = cudaMalloc(&base, bytes);
    if (e == cudaSuccess) {
        c->view.base = static_cast<uint8_t *>(base);
        if ((e = cudaMalloc(&c->d_err, sizeof(int))) == cudaSuccess &&
            (e = cudaMemset(c->d_err, 0, sizeof(int))) == cudaSuccess &&
            (e = cudaMemset(base, 0, bytes)) == cudaSuccess)
            e = cudaStreamSynchronize(nullptr);  // zeroed before any stream uses it
    }
    c->view.err = c->d_err;
    if (e != cudaSuccess) {
        rabbit_cuda_kv4_free(c);
        cudaSetDevice(prev);
        cudaGetLastError();
        return e == cudaErrorMemoryAllocation
                   ? fail(RABBIT_CUDA_ERR_MEM, "kv4_create: %zu bytes of device memory", bytes)
                   : cuda_fail(e, "kv4_create: device memory");
    }
    cudaSetDevice(prev);
    *out = c;
    return ok();
}

int rabbit_cuda_kv4_free(rabbit_cuda_kv4 *kv) {
    if (!kv) return ok();
    {
        DeviceScope scope(kv->device);
        if (kv->view.base) cudaFree(kv->view.base);
        if (kv->d_err) cudaFree(kv->d_err);
    }
    delete kv;
    return ok();
}

uint64_t rabbit_cuda_kv4_bytes(const rabbit_cuda_kv4 *kv) {
    return kv ? (uint64_t)kv->n_layers * kv->layer_bytes : 0;
}

int rabbit_cuda_kv4_append_dev(rabbit_cuda_kv4 *kv, int layer, int dtype, const void *d_k,
                               int64_t k_stride, const void *d_v, int64_t v_stride,
                               const int64_t *d_slots, int n_tokens, const rabbit_cuda_rope *rope,
                               const int *d_positions, void *stream) {
    if (!kv || layer < 0 || layer >= kv->n_layers || !dtype_size(dtype) || n_tokens < 0)
        return fail(RABBIT_CUDA_ERR_ARGS, "kv4_append: NULL cache, a bad layer, dtype or count");
    if (n_tokens == 0) return ok();
    if (!d_k || !d_v || !d_slots || (rope && !d_positions))
        return fail(RABBIT_CUDA_ERR_ARGS, "kv4_append: NULL pointer");
    Kv4AppendRopeArgs aa;
    Kv4AppendArgs &a = aa.a;
    a.c = kv->layer(layer);
    const int64_t row = (int64_t)a.c.nkv * a.c.hd;
    const int size = dtype_size(dtype);
    a.x[0] = d_k;
    a.x[1] = d_v;
    a.xs[0] = k_stride ? k_stride : row;
    a.xs[1] = v_stride ? v_stride : row;
    if (a.xs[0] < row || a.xs[1] < row || !aligned(d_k, size) || !aligned(d_v, size) ||
        !aligned(d_slots, 8) || !aligned(d_positions, 4))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "kv4_append: a stride below n_kv_heads * head_dim, or a pointer not aligned to "
                    "its element");
    int np = 0;
    if (rope) {
        int hd;
        aa.tab = rope_tab(rope, &hd);
        if (hd != a.c.hd)
            return fail(RABBIT_CUDA_ERR_ARGS, "kv4_append: the rope's head_dim is %d, the cache's %d",
                        hd, a.c.hd);
        np = aa.tab.rot / 2;
    }
    a.slots = d_slots;
    a.pos = rope ? d_positions : nullptr;
    a.T = n_tokens;
    a.tpc = 1;
    const bool vec = aligned(d_k, 16) && aligned(d_v, 16) && a.xs[0] * size % 16 == 0 &&
                     a.xs[1] * size % 16 == 0 && (int64_t)a.c.hd * size % 16 == 0;
    DeviceScope scope(kv->device);
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    const int items = a.tpc * a.c.nkv * a.c.ng * 4;
    const dim3 grid((n_tokens + a.tpc - 1) / a.tpc, (items + kAppendThreads - 1) / kAppendThreads, 2);
    const size_t smem = sizeof(double2) * (size_t)a.tpc * np;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        auto k = rope ? (vec ? k_kv4_append<T, true, true> : k_kv4_append<T, false, true>)
                      : (vec ? k_kv4_append<T, true, false> : k_kv4_append<T, false, false>);
        scope.launch(launch_pdl(k, grid, dim3(kAppendThreads), smem,
                                static_cast<cudaStream_t>(stream), aa),
                     "kv4_append");
        return 0;
    });
    return scope.done();
}

int rabbit_cuda_kv4_read_dev(rabbit_cuda_kv4 *kv, int layer, int dtype, const int64_t *d_slots,
                             int n_tokens, void *d_k, void *d_v, void *stream) {
    if (!kv || layer < 0 || layer >= kv->n_layers || !dtype_size(dtype) || n_tokens < 0)
        return fail(RABBIT_CUDA_ERR_ARGS, "kv4_read: NULL cache, a bad layer, dtype or count");
    if (n_tokens == 0 || (!d_k && !d_v)) return ok();
    const int size = dtype_size(dtype);
    if (!d_slots || !aligned(d_slots, 8) || !aligned(d_k, size) || !aligned(d_v, size))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "kv4_read: NULL slots, or a pointer not aligned to its element");
    Kv4ReadArgs a;
    a.c = kv->layer(layer);
    a.y[0] = d_k;
    a.y[1] = d_v;
    a.slots = d_slots;
    a.T = n_tokens;
    const bool vec = aligned(d_k, 16) && aligned(d_v, 16) && (int64_t)a.c.hd * size % 16 == 0;
    const int64_t items = (int64_t)n_tokens * a.c.nkv * a.c.ng * 4;
    const int64_t blocks = (items + 255) / 256, most = 16ll * kv->ctx->sm_count;
    DeviceScope scope(kv->device);
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        scope.launch(launch_pdl(vec ? k_kv4_read<T, true> : k_kv4_read<T, false>,
                                dim3((unsigned)(blocks < most ? blocks : most), 1, 2), dim3(256), 0,
                                static_cast<cudaStream_t>(stream), a),
                     "kv4_read");
        return 0;
    });
    return scope.done();
}

int rabbit_cuda_kv4_check(rabbit_cuda_kv4 *kv, void *stream) {
    if (!kv) return fail(RABBIT_CUDA_ERR_ARGS, "kv4_check: NULL cache");
    DeviceScope scope(kv->device);
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int h = 0;
    RB_CUDA(cudaMemcpyAsync(&h, kv->d_err, sizeof(int), cudaMemcpyDeviceToHost, s));
    RB_CUDA(cudaStreamSynchronize(s));
    if (h == 0) return ok();
    RB_CUDA(cudaMemsetAsync(kv->d_err, 0, sizeof(int), s));
    RB_CUDA(cudaStreamSynchronize(s));
    if (h & (RB_KV4_ERR_SLOT | RB_KV4_ERR_PAGE | RB_KV4_ERR_LEN | RB_KV4_ERR_ROWS))
        return fail(RABBIT_CUDA_ERR_ARGS, "kv4: out of range on the device:%s%s%s%s",
                    h & RB_KV4_ERR_SLOT ? " slot" : "", h & RB_KV4_ERR_PAGE ? " page" : "",
                    h & RB_KV4_ERR_LEN ? " kv_len" : "", h & RB_KV4_ERR_ROWS ? " q_start" : "");
    return h & 15 ? fail(RABBIT_CUDA_ERR_TIMEOUT, "kv4: a bounded device wait ran out")
                  : fail(RABBIT_CUDA_ERR_DEVICE, "kv4: device error code %d", h);
}

}  // extern "C"
