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

// Channel `ch` of a head's row in 64 bits; its first `rot` channels rotated by
// the token's table.
template <typename T>
__device__ __forceinline__ double exact_channel(const T *row, int ch, const double2 *table, int rot, bool halves) {
    if (ch >= rot) return to_f32(row[ch]);
    const int np = rot / 2;
    const bool first = halves ? ch < np : !(ch & 1);
    const int other = halves ? (first ? ch + np : ch - np) : ch ^ 1;
    const double2 k = table[halves ? (first ? ch : other) : ch >> 1];
    return (double)to_f32(row[ch]) * k.x + (double)to_f32(row[other]) * (first ? -k.y : k.y);
}
// Channels ch .. ch + 7 again where 32 bits leave a rounding open: the bits of the
// largest magnitude in fp32, and the codes (4 bits each).
template <typename T>
__device__ __noinline__ uint32_t exact_top(const T *row, int ch, const double2 *table, int rot, bool halves) {
    uint32_t top = 0;
#pragma unroll 1
    for (int n = 0; n < 8; ++n)
        top = max(top, __float_as_uint(fabsf((float)exact_channel(row, ch + n, table, rot, halves))));
    return top;
}
template <typename T>
__device__ __noinline__ uint32_t exact_codes(const T *row, int ch, const double2 *table, int rot, bool halves, float s) {
    uint32_t word = 0;
#pragma unroll 1
    for (int n = 0; n < 8; ++n) {
        // (a scale among bf16's smallest numbers may have been rounded down by up to a half)
        const double q = rint(exact_channel(row, ch + n, table, rot, halves) / (double)s);
        word |= ((uint32_t)(int)fmin(fmax(q, -7.0), 7.0) & 15u) << (4 * n);
    }
    return word;
}

// One CTA: tpc tokens, a thread 8 consecutive channels of one (token, head) of
// the keys (blockIdx.z = 0) or the values, 4 threads a group.
//
// The codes are those of the exact value, at the cost of 32-bit arithmetic: the
// rotation, the scale and the quotients are made in fp32 with a bound on their
// error, and only where the bound leaves the rounding open (the scale's to bf16, a
// quotient's to a whole number: about one value in 10^4) once more in 64 bits, from
// the 64-bit cosine and sine that the token's table holds too. All in 64 bits the
// conversions alone took 40 us for 8191 x 8 x 80 fp16 with a rotation; so the kernel
// takes 31 us, 24 us without a rotation.
template <typename T, bool VEC, bool ROPE>
__global__ void __launch_bounds__(kAppendThreads, 4) k_kv4_append(const __grid_constant__ Kv4AppendRopeArgs aa) {
    extern __shared__ __align__(16) double2 cs[];  // [tpc][rot / 2], keys only; then the same in fp32
    const Kv4AppendArgs &a = aa.a;
    const RopeTab &tab = aa.tab;
    const Kv4View &c = a.c;
    launch_dependents();
    wait_prerequisite();
    const int kv = blockIdx.z, t0 = blockIdx.x * a.tpc, nt = min(a.tpc, a.T - t0);
    const bool rot = ROPE && kv == 0;
    const int np = ROPE ? tab.rot / 2 : 0;
    float2 *cs32 = reinterpret_cast<float2 *>(cs + a.tpc * np);
    float mag = 0.f;
    if constexpr (ROPE) {
        mag = fabsf((float)tab.mag);
        if (rot) {
            for (int i = threadIdx.x; i < nt * np; i += kAppendThreads) {
                double2 v = rope_cs(a.pos[t0 + i / np], tab.turns[i % np]);
                v.x *= tab.mag;
                v.y *= tab.mag;
                cs[i] = v;
                cs32[i] = make_float2((float)v.x, (float)v.y);
            }
            __syncthreads();
        }
    }
    const bool halves = ROPE && tab.layout == RABBIT_CUDA_ROPE_HALF;
    // a thread keeps its item of the row and goes through the tokens; short rows:
    // several tokens side by side
    const int per = c.nkv * c.ng * 4;
    const int side = per <= kAppendThreads / 2 ? kAppendThreads / per : 1;
    const int first = side > 1 ? threadIdx.x / per : 0;
    for (int u0 = side > 1 ? 0 : blockIdx.y * kAppendThreads; u0 < per; u0 += gridDim.y * kAppendThreads) {
        const int u = u0 + threadIdx.x - first * per;
        const bool mine = u < per && first < side;
        const int head = u / (c.ng * 4), w = u - head * c.ng * 4, grp = w >> 2, t = w & 3;
        const int c0 = 8 * w;  // first channel
        const T *row = static_cast<const T *>(a.x[kv]) + (t0 + first - side) * a.xs[kv] + (int64_t)head * c.hd;
        const int64_t step = side * a.xs[kv];
        const size_t part = (size_t)head * c.head_bytes() + (kv ? kv4_v(c.ng) : 0);
        for (int ta = 0; ta < nt; ta += side) {
            const int tl = ta + first;
            row += step;
            const bool in = mine && tl < nt;
            const int64_t slot = in ? a.slots[t0 + tl] : -1;
            const bool write = slot >= 0 && slot < c.slots();
            if (in && slot >= c.slots()) atomicOr(c.err, RB_KV4_ERR_SLOT);
            const bool turn = ROPE && rot && c0 < tab.rot;
            // v, p: each channel and the other of its pair before the rotation; x: after it
            float x[8], v[8], p[8], big = 0.f;  // big: the largest |v| + |p|
#pragma unroll
            for (int n = 0; n < 8; ++n) x[n] = v[n] = p[n] = 0.f;
            if (write && c0 < c.hd) {
                load8<VEC>(v, row + c0);
#pragma unroll
                for (int n = 0; n < 8; ++n) x[n] = v[n];
                if constexpr (ROPE) {
                    if (turn) {
                        float2 k[8];  // x = v k.x + p k.y
                        const float2 *ct = cs32 + tl * np;
                        if (!halves) {
#pragma unroll
                            for (int n = 0; n < 8; ++n) {
                                p[n] = v[n ^ 1];
                                if (!(n & 1)) k[n] = k[n + 1] = c0 + n < tab.rot ? ct[(c0 + n) / 2] : make_float2(1.f, 0.f);
                                if (!(n & 1)) k[n].y = -k[n].y;
                            }
                        } else if (np % 8 == 0) {  // all 8 are first or second
                            const bool first = c0 < np;
                            load8<VEC>(p, row + (first ? c0 + np : c0 - np));
                            const float4 *c4 = reinterpret_cast<const float4 *>(ct + (first ? c0 : c0 - np));
#pragma unroll
                            for (int n = 0; n < 8; n += 2) {
                                const float4 y = c4[n / 2];
                                k[n] = make_float2(y.x, first ? -y.y : y.y);
                                k[n + 1] = make_float2(y.z, first ? -y.w : y.w);
                            }
                        } else {
#pragma unroll
                            for (int n = 0; n < 8; ++n) {
                                const int ch = c0 + n;
                                k[n] = make_float2(1.f, 0.f);
                                if (ch < tab.rot) {
                                    p[n] = to_f32(row[ch < np ? ch + np : ch - np]);
                                    k[n] = ct[ch < np ? ch : ch - np];
                                    if (ch < np) k[n].y = -k[n].y;
                                }
                            }
                        }
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            x[n] = fmaf(v[n], k[n].x, p[n] * k[n].y);
                            big = fmaxf(big, fabsf(v[n]) + fabsf(p[n]));
                        }
                    }
                }
            }
            auto scale_of = [](float top) {
                const float top7 = __fmul_rn(top, 1.0f / 7.0f);
                // a group with an infinity or a NaN has a NaN for its scale
                return __float2bfloat16_rn(top7 < INFINITY ? top7 : __uint_as_float(0x7fc00000u));
            };
            // the group's largest: an integer maximum of the bits keeps a NaN
            uint32_t top = 0;
#pragma unroll
            for (int n = 0; n < 8; ++n) top = max(top, __float_as_uint(fabsf(x[n])));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            __nv_bfloat16 sb = scale_of(__uint_as_float(top));
            float off = 0.f;  // how far the rotated values may be off
            if constexpr (ROPE) {
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                // cosine and sine half a step off, a product and a sum rounded: at most
                // 4 2^-24 (|v| + |p|) of the magnitude, and a few of fp32's smallest steps
                off = big > 0.f ? fmaf(big * mag, 2.4e-7f, 6e-45f) : 0.f;
                const float a0 = __uint_as_float(top) - off, a1 = __uint_as_float(top) + off;
                const bool open = off > 0.f && !(__bfloat162float(scale_of(fmaxf(a0, 0.f))) == __bfloat162float(scale_of(a1)));
                if (__any_sync(0xffffffffu, open)) {
                    uint32_t e = 0;
                    if (write && c0 < c.hd) e = exact_top(row, c0, cs + tl * np, turn ? tab.rot : 0, halves);
                    e = max(e, __shfl_xor_sync(0xffffffffu, e, 1));
                    e = max(e, __shfl_xor_sync(0xffffffffu, e, 2));
                    if (open) sb = scale_of(__uint_as_float(e));
                }
            }
            if (!write) continue;
            const float s = __bfloat162float(sb), inv = __fdividef(1.0f, s);
            uint32_t word = 0x88888888u;
            if (s > 0.f) {
                // quotients off by off / s and 2^-21 |q|, |q| < 8; a scale near the smallest
                // fp32 has no finite reciprocal
                const float room = fmaf(off, inv, 4e-6f);
                float least = s < 1e-30f ? -1.f : 1.f;  // the least distance from a half
                word = 0;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    // the whole number lies in the low bits of a sum with 3 2^22
                    const float q = x[n] * inv, m = q + 12582912.0f;
                    word |= (__float_as_uint(m) & 15u) << (4 * n);
                    least = fminf(least, fabsf(fabsf(q - (m - 12582912.0f)) - 0.5f));
                }
                if (!(least > room) && off == 0.f && s >= 1e-30f) {
                    // Values as they came (of few bits, often halves exactly): (k + 1/2) s has 12
                    // bits, so the sign of x - (k + 1/2) s in fp32 is exact.
                    word = 0;
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const float k = floorf(x[n] * inv), r = fmaf(-(k + 0.5f), s, x[n]);
                        const int code = (int)k;
                        word |= (uint32_t)((r > 0.f || (r == 0.f && (code & 1)) ? code + 1 : code) & 15) << (4 * n);
                    }
                } else if (!(least > room))
                    word = c0 < c.hd ? exact_codes(row, c0, ROPE ? cs + tl * np : nullptr, turn ? tab.rot : 0, halves, s) : 0u;
                word ^= 0x88888888u;  // plus 8
            }
            const int j = (int)slot & (kKv4Granule - 1);  // pages are whole granules
            uint8_t *g = c.row(slot) + part;
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
}

struct Kv4ReadArgs {
    Kv4View c;
    void *y[2];
    const int64_t *slots;
    int T, tpc;
};

// A thread: 8 channels of one (token, head); keys in y[0], values in y[1].
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) k_kv4_read(const __grid_constant__ Kv4ReadArgs a) {
    launch_dependents();
    wait_prerequisite();
    const Kv4View &c = a.c;
    const int kv = blockIdx.z, per = c.nkv * c.ng * 4, t0 = blockIdx.x * a.tpc, nt = min(a.tpc, a.T - t0);
    if (!a.y[kv]) return;
    const int side = per <= kAppendThreads / 2 ? kAppendThreads / per : 1;
    const int first = side > 1 ? threadIdx.x / per : 0;
    if (first >= side) return;
    for (int u = side > 1 ? threadIdx.x - first * per : blockIdx.y * kAppendThreads + threadIdx.x; u < per;
         u += gridDim.y * kAppendThreads) {
        const int head = u / (c.ng * 4), w = u - head * c.ng * 4, grp = w >> 2, t = w & 3;
        for (int tl = first; tl < nt; tl += side) {
            const int64_t slot = a.slots[t0 + tl];
            if (slot < 0 || 8 * w >= c.hd) continue;
            if (slot >= c.slots()) {
                atomicOr(c.err, RB_KV4_ERR_SLOT);
                continue;
            }
            const int j = (int)slot & (kKv4Granule - 1);  // pages are whole granules
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
            store8<VEC>(static_cast<T *>(a.y[kv]) + (int64_t)(t0 + tl) * c.nkv * c.hd + head * c.hd + 8 * w, v);
        }
    }
}

// err[0], taken and cleared in one step, into err[1].
__global__ void k_kv4_take(int *err) { err[1] = atomicExch(err, 0); }

// Tokens per CTA of the append and the read: one wave of four CTAs an SM for each
// of keys and values, up to 8; a token's items in one CTA each 256 (blockIdx.y).
static int tokens_per_cta(int n_tokens, int sms) {
    const int64_t n = ((int64_t)n_tokens + 4 * sms - 1) / (4 * sms);
    return n > 8 ? 8 : (int)n;
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
    c->view.head_nbytes = (size_t)(d->page_size / kKv4Granule) * kv4_bytes(c->view.ng);
    c->view.page_nbytes = d->n_kv_heads * c->view.head_nbytes;
    c->view.n_slots = (int64_t)d->n_pages * d->page_size;
    c->view.shift = -1;
    for (int i = 4; i <= 10; ++i)
        if (d->page_size == 1 << i) c->view.shift = i;
    c->layer_bytes = (size_t)d->n_pages * c->view.page_bytes();  // below 2^60
    size_t bytes = 0;
    void *base = nullptr;
    cudaError_t e = __builtin_mul_overflow((size_t)d->n_layers, c->layer_bytes, &bytes) ? cudaErrorMemoryAllocation
                                                                                      : cudaMalloc(&base, bytes);
    if (e == cudaSuccess) {
        c->view.base = static_cast<uint8_t *>(base);
        if ((e = cudaMalloc(&c->d_err, 2 * sizeof(int))) == cudaSuccess &&
            (e = cudaMemset(c->d_err, 0, 2 * sizeof(int))) == cudaSuccess &&
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
    a.tpc = tokens_per_cta(n_tokens, kv->ctx->sm_count);
    const bool vec = aligned(d_k, 16) && aligned(d_v, 16) && a.xs[0] * size % 16 == 0 &&
                     a.xs[1] * size % 16 == 0 && (int64_t)a.c.hd * size % 16 == 0;
    DeviceScope scope(kv->device);
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    const int items = a.c.nkv * a.c.ng * 4;
    const dim3 grid((unsigned)(((int64_t)n_tokens + a.tpc - 1) / a.tpc), (items + kAppendThreads - 1) / kAppendThreads, 2);
    const size_t smem = (sizeof(double2) + sizeof(float2)) * (size_t)a.tpc * np;
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
    a.tpc = tokens_per_cta(n_tokens, kv->ctx->sm_count);
    const int items = a.c.nkv * a.c.ng * 4;
    const dim3 grid((unsigned)(((int64_t)n_tokens + a.tpc - 1) / a.tpc), (items + kAppendThreads - 1) / kAppendThreads, 2);
    DeviceScope scope(kv->device);
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        scope.launch(launch_pdl(vec ? k_kv4_read<T, true> : k_kv4_read<T, false>,
                                grid, dim3(kAppendThreads), 0,
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
    RB_CUDA(cudaStreamSynchronize(s));
    {
        // what another stream's call sets meanwhile is taken now or stays for the next check
        std::lock_guard<std::mutex> hold(kv->taking);
        k_kv4_take<<<1, 1, 0, s>>>(kv->d_err);
        RB_CUDA(cudaGetLastError());
        RB_CUDA(cudaMemcpyAsync(&h, kv->d_err + 1, sizeof(int), cudaMemcpyDeviceToHost, s));
        RB_CUDA(cudaStreamSynchronize(s));
    }
    if (h == 0) return ok();
    // the timeout first: after it the caller has to replace a scratch
    const int range = h & (RB_KV4_ERR_SLOT | RB_KV4_ERR_PAGE | RB_KV4_ERR_LEN | RB_KV4_ERR_ROWS);
    return fail(h & RB_KV4_ERR_WAIT ? RABBIT_CUDA_ERR_TIMEOUT : RABBIT_CUDA_ERR_ARGS, "kv4: %s%s%s%s%s%s",
                h & RB_KV4_ERR_WAIT ? "a bounded device wait ran out; " : "",
                range ? "out of range on the device:" : "", h & RB_KV4_ERR_SLOT ? " slot" : "",
                h & RB_KV4_ERR_PAGE ? " page" : "", h & RB_KV4_ERR_LEN ? " kv_len" : "",
                h & RB_KV4_ERR_ROWS ? " q_start" : "");
}

}  // extern "C"
