// rb_kv4_attn.cu -- attention over the paged 4-bit key / value cache.
#include <math.h>

#include <new>

#include "rb_device.cuh"
#include "rb_kv4.cuh"
#include "rb_launch.h"
#include "rb_types.cuh"

struct rabbit_cuda_kv4_scratch {
    int device = -1;
};

namespace rb {

struct Kv4AttnArgs {
    Kv4View c;
    const void *q;
    void *out;
    int64_t qs, os;
    const int *q_start, *kv_len, *table;
    int n_seqs, max_pages, max_q, T, nh, window;
    float scale;
};

constexpr int kAttnPlainThreads = 128;

__device__ __forceinline__ float kv4_value(const uint8_t *codes, const uint8_t *scales, int j, int ng,
                                           int ch, bool v) {
    const int grp = ch >> 5, in = ch & 31;
    uint32_t w;
    if (!v)
        w = reinterpret_cast<const uint32_t *>(codes + j * kv4_row(ng))[(in >> 3) * ng + grp] >> (4 * (in & 7));
    else
        w = reinterpret_cast<const uint16_t *>(codes + j * kv4_row(ng))[kv4_vplace(j, in >> 2) * ng + grp] >>
            (4 * (in & 3));
    return (float)((int)(w & 15u) - 8) *
           __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(scales)[j * ng + grp]);
}

// A CTA per (query row, head), a warp per position, lanes over the channels.
template <typename T>
__global__ void __launch_bounds__(kAttnPlainThreads) k_kv4_attn(const __grid_constant__ Kv4AttnArgs a) {
    constexpr int NW = kAttnPlainThreads / 32;
    __shared__ float wm[NW], wl[NW], wo[NW][32 * kKv4MaxGroups];
    launch_dependents();
    wait_prerequisite();
    const Kv4View &c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x, head = blockIdx.y, kvh = head / (a.nh / c.nkv);
    int seq = row < a.n_seqs ? row : -1, first = row, last = row + 1;
    if (a.q_start) {
        seq = -1;
        for (int i = 0; i < a.n_seqs; ++i) {
            const int s0 = a.q_start[i], s1 = a.q_start[i + 1];
            if (s0 < 0 || s1 < s0 || s1 > a.T || s1 - s0 > a.max_q) {
                if (threadIdx.x == 0) atomicOr(c.err, RB_KV4_ERR_ROWS);
            } else if (s0 <= row && row < s1) {
                seq = i;
                first = s0;
                last = s1;
            }
        }
    }
    if (seq < 0) return;
    int len = a.kv_len[seq];
    if (len < 0 || (int64_t)len > (int64_t)a.max_pages * c.page) {
        if (threadIdx.x == 0) atomicOr(c.err, RB_KV4_ERR_LEN);
        len = 0;
    }
    const int at = len - (last - first) + (row - first);
    const int lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
    float q[kKv4MaxGroups], o[kKv4MaxGroups], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int g = 0; g < kKv4MaxGroups; ++g) {
        const int ch = 32 * g + lane;
        q[g] = ch < c.hd ? to_f32((static_cast<const T *>(a.q) + row * a.qs + (int64_t)head * c.hd)[ch]) : 0.f;
        o[g] = 0.f;
    }
    for (int p = lo + warp; p <= at; p += NW) {
        const int pg = a.table[(int64_t)seq * a.max_pages + p / c.page];
        if (pg < 0 || pg >= c.n_pages) {
            if (lane == 0) atomicOr(c.err, RB_KV4_ERR_PAGE);
            continue;
        }
        const uint8_t *gr = c.granule((int64_t)pg * c.page + p % c.page, kvh);
        const int j = p & 15;
        float d = 0.f;
#pragma unroll
        for (int g = 0; g < kKv4MaxGroups; ++g)
            if (g < c.ng) d = fmaf(q[g], kv4_value(gr, gr + kv4_ks(c.ng), j, c.ng, 32 * g + lane, false), d);
        for (int s = 16; s; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
        d *= a.scale;
        const float mn = fmaxf(m, d), corr = expf(m - mn), e = expf(d - mn);
        l = l * corr + e;
        m = mn;
#pragma unroll
        for (int g = 0; g < kKv4MaxGroups; ++g)
            if (g < c.ng)
                o[g] = o[g] * corr + e * kv4_value(gr + kv4_v(c.ng), gr + kv4_vs(c.ng), j, c.ng,
                                                   32 * g + lane, true);
    }
    if (lane == 0) {
        wm[warp] = m;
        wl[warp] = l;
    }
#pragma unroll
    for (int g = 0; g < kKv4MaxGroups; ++g) wo[warp][32 * g + lane] = o[g];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < NW; ++w) M = fmaxf(M, wm[w]);
    for (int w = 0; w < NW; ++w) L += wl[w] > 0.f ? wl[w] * expf(wm[w] - M) : wl[w];
    for (int ch = threadIdx.x; ch < c.hd; ch += kAttnPlainThreads) {
        float s = 0.f;
        for (int w = 0; w < NW; ++w) s += wl[w] != 0.f ? wo[w][ch] * expf(wm[w] - M) : 0.f;
        (static_cast<T *>(a.out) + row * a.os + (int64_t)head * c.hd)[ch] = from_f32<T>(L != 0.f ? s / L : 0.f);
    }
}

}  // namespace rb

using namespace rb;

extern "C" {

int rabbit_cuda_kv4_scratch_create(const rabbit_cuda_kv4 *kv, rabbit_cuda_kv4_scratch **out) {
    if (!kv || !out) return fail(RABBIT_CUDA_ERR_ARGS, "kv4_scratch_create: NULL argument");
    *out = new (std::nothrow) rabbit_cuda_kv4_scratch();
    if (!*out) return fail(RABBIT_CUDA_ERR_MEM, "kv4_scratch_create: out of host memory");
    (*out)->device = kv->device;
    return ok();
}

int rabbit_cuda_kv4_scratch_free(rabbit_cuda_kv4_scratch *ws) {
    delete ws;
    return ok();
}

int rabbit_cuda_kv4_attention_dev(rabbit_cuda_kv4 *kv, int layer, rabbit_cuda_kv4_scratch *ws,
                                  int dtype, const void *d_q, int64_t q_stride, void *d_out,
                                  int64_t out_stride, int n_tokens, int n_heads,
                                  const rabbit_cuda_kv4_batch *b, float scale, int window,
                                  void *stream) {
    if (!kv || !ws || !b || layer < 0 || layer >= kv->n_layers || !dtype_size(dtype) ||
        n_tokens < 0 || n_heads < 1 || n_heads > 65535 || n_heads % kv->view.nkv || window < 0 ||
        !isfinite(scale))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "kv4_attention: NULL cache, scratch or batch, a bad layer, dtype, count, scale or "
                    "window, or n_heads not a multiple of n_kv_heads");
    if (b->n_seqs < 0 || b->n_seqs > 65535 || b->max_pages < 0 || b->max_q_len < 0)
        return fail(RABBIT_CUDA_ERR_ARGS, "kv4_attention: a bad count in the batch");
    if (ws->device != kv->device)
        return fail(RABBIT_CUDA_ERR_ARGS, "kv4_attention: the scratch is of another device");
    if (n_tokens == 0 || b->n_seqs == 0) return ok();
    const int size = dtype_size(dtype);
    Kv4AttnArgs a;
    a.c = kv->layer(layer);
    const int64_t row = (int64_t)n_heads * a.c.hd;
    a.qs = q_stride ? q_stride : row;
    a.os = out_stride ? out_stride : row;
    if (!d_q || !d_out || !b->d_kv_len || (!b->d_page_table && b->max_pages) || a.qs < row ||
        a.os < row || (reinterpret_cast<uintptr_t>(d_q) & (size - 1)) ||
        (reinterpret_cast<uintptr_t>(d_out) & (size - 1)) || (d_q == d_out && a.qs != a.os))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "kv4_attention: NULL pointer, a stride below n_heads * head_dim (or different in "
                    "place), or a pointer not aligned to its element");
    a.q = d_q;
    a.out = d_out;
    a.q_start = b->d_q_start;
    a.kv_len = b->d_kv_len;
    a.table = b->d_page_table;
    a.n_seqs = b->n_seqs;
    a.max_pages = b->max_pages;
    a.max_q = b->max_q_len ? b->max_q_len : 1;
    a.T = n_tokens;
    a.nh = n_heads;
    a.window = window;
    a.scale = scale != 0.f ? scale : 1.0f / sqrtf((float)a.c.hd);
    DeviceScope scope(kv->device);
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    with_dtype(dtype, [&](auto t) {
        scope.launch(launch_pdl(k_kv4_attn<decltype(t)>, dim3(n_tokens, n_heads),
                                dim3(kAttnPlainThreads), 0, static_cast<cudaStream_t>(stream), a),
                     "kv4_attention");
        return 0;
    });
    return scope.done();
}

}  // extern "C"
