// rb_experts.cu -- C ABI: which experts a token goes to and the order by expert
// (select_top_k, src/forward_v2.c:248-278, for many tokens), and the weighted sum of the
// experts' rows (:356-357, 398-399).
#include <math.h>

#include <atomic>
#include <type_traits>

#include "rb_device.cuh"
#include "rb_launch.h"
#include "rb_runtime.h"
#include "rb_types.cuh"

namespace rb {

constexpr int kRouteThreads = 1024, kRouteWarps = kRouteThreads / 32;
constexpr int kRouteCluster = 8;
constexpr int kRouteExperts = 1024, kRouteK = 32;

struct RouteArgs {
    const float *scores;
    int64_t stride;
    int T, E, k, over_all;
    int *ids;
    float *weights;
    int *offsets, *rows, *place;
};

// Order of scores as unsigned numbers; 0 for what is never taken (-inf, NaN).
__device__ __forceinline__ uint32_t score_key(float s) {
    if (!(s > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(s + 0.f);  // -0 counts as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One token by one warp: lane l holds experts l, l + 32, ... A pick is the warp's largest
// key and among equals its lowest id. Bound by the k dependent picks (two warp
// reductions and a shuffle each), not by the scores' bytes.
template <int V>
__device__ void route_token(const RouteArgs &a, int t, int lane) {
    const float *row = a.scores + (int64_t)t * a.stride;
    float s[V];
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 32 * i;
        s[i] = e < a.E ? row[e] : -INFINITY;
        key[i] = score_key(s[i]);
    }
    int my_id = -1;            // lane j keeps pick j
    float my_s = -INFINITY, top = -INFINITY;
    for (int j = 0; j < a.k; ++j) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) best = max(best, key[i]);
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0) break;
        int id = kRouteExperts;
        float found = 0.f;
#pragma unroll
        for (int i = V - 1; i >= 0; --i)
            if (key[i] == most) {
                id = lane + 32 * i;
                found = s[i];
            }
        const int first = __reduce_min_sync(0xffffffffu, id);
        found = __shfl_sync(0xffffffffu, found, first & 31);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (lane + 32 * i == first) key[i] = 0;
        if (j == 0) top = found;
        if (lane == j) {
            my_id = first;
            my_s = found;
        }
    }
    // exp(s - top), 1 at the top (an infinite one as well)
    auto part = [&](float v) { return v == top ? 1.f : v > -INFINITY ? expf(v - top) : 0.f; };
    const float mine = my_id >= 0 ? part(my_s) : 0.f;
    float sum = 0.f;
    if (a.over_all) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum += top > -INFINITY ? part(s[i]) : 0.f;
    } else {
        sum = mine;
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (lane < a.k) {
        a.ids[(int64_t)t * a.k + lane] = my_id;
        a.weights[(int64_t)t * a.k + lane] = my_id >= 0 ? mine / sum : 0.f;
    }
}

template <int V>
__global__ void __launch_bounds__(256) k_route(const __grid_constant__ RouteArgs a) {
    launch_dependents();
    wait_prerequisite();
    for (int t = blockIdx.x * 8 + (threadIdx.x >> 5); t < a.T; t += gridDim.x * 8)
        route_token<V>(a, t, threadIdx.x & 31);
}

// Lanes with the same low `bits` bits of e (a vote for each: of 32 values that mostly differ,
// match.any takes several times as long).
__device__ __forceinline__ uint32_t lanes_alike(int e, int bits) {
    uint32_t same = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
        const bool set = e >> b & 1;
        const uint32_t v = __ballot_sync(0xffffffffu, set);
        same &= set ? v : ~v;
    }
    return same;
}

// A counting sort of the pairs by expert that keeps their order, one cluster of CTAs: CTA r
// and in it warp w have the r-th and w-th part of the pairs. Each warp counts its pairs of
// each expert in its own column of shared memory; the counts become places (experts, CTAs, warps in
// turn); then each warp takes its pairs again, 32 at a time, a pair's place its
// column's plus the equal experts on lower lanes: the same places each time.
// 8191 tokens of 6 given ids among 64 experts: 10 us, 4096 of 8 among 1024: 12 us; one token 5.5 us.
// PICK above 0: the tokens' experts are chosen here, too, PICK scores a lane.
template <int PICK>
__global__ void __launch_bounds__(kRouteThreads, 1) k_route_order(const __grid_constant__ RouteArgs a) {
    extern __shared__ int route_smem[];
    int *count = route_smem;                       // [warps][E]
    int *total = route_smem + kRouteWarps * a.E;   // [E] of this CTA
    int *base = total + a.E;                       // [E] first place of an expert here
    __shared__ int warp_sum[kRouteWarps];
    __shared__ int everything;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = gridDim.x, cta = blockIdx.x;
    launch_dependents();
    wait_prerequisite();
    const int warps = ctas * kRouteWarps, w = cta * kRouteWarps + warp;
    const int t0 = (int)((int64_t)a.T * w / warps), t1 = (int)((int64_t)a.T * (w + 1) / warps);
    if constexpr (PICK > 0)
        for (int t = t0; t < t1; ++t) route_token<PICK>(a, t, lane);
    __syncwarp();
    int *mine = count + warp * a.E;
    for (int e = lane; e < a.E; e += 32) mine[e] = 0;
    __syncwarp();
    const int p0 = t0 * a.k, p1 = t1 * a.k;
    auto expert = [&](int p) {
        const int e = p < p1 ? a.ids[p] : -1;
        return e >= 0 && e < a.E ? e : -1;
    };
    const int bits = 32 - __clz(a.E);  // of an expert and of -1's low bits
    constexpr int B = 8;  // pairs of a lane read at a time: one after the other they took 8 us
    for (int p = p0; p < p1; p += 32 * B) {
        int es[B];
#pragma unroll
        for (int b = 0; b < B; ++b) es[b] = expert(p + 32 * b + lane);
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (es[b] >= 0) atomicAdd(&mine[es[b]], 1);  // (a sum of whole numbers: in any order)
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += kRouteThreads) {  // columns: first place in the CTA
        int n = 0;
#pragma unroll
        for (int i0 = 0; i0 < kRouteWarps; i0 += 16) {
            int c[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) c[i] = count[(i0 + i) * a.E + e];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                count[(i0 + i) * a.E + e] = n;
                n += c[i];
            }
        }
        total[e] = n;
    }
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    } else {
        __syncthreads();
    }
    int before = 0, all = 0;  // of this thread's expert: in the CTAs before, in all
    if (threadIdx.x < a.E) {
        for (int r = 0; r < ctas; ++r) {
            int n;
            if (ctas > 1) {
                uint32_t at;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(total + threadIdx.x)), "r"(r));
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(n) : "r"(at) : "memory");
            } else {
                n = total[threadIdx.x];
            }
            if (r < cta) before += n;
            all += n;
        }
    }
    int up = all;  // over the experts up to this thread's
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, up, d);
        if (lane >= d) up += n;
    }
    if (lane == 31) warp_sum[warp] = up;
    __syncthreads();
    if (warp == 0) {
        int n = warp_sum[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int m = __shfl_up_sync(0xffffffffu, n, d);
            if (lane >= d) n += m;
        }
        warp_sum[lane] = n;
        if (lane == 31) everything = n;
    }
    __syncthreads();
    if (warp > 0) up += warp_sum[warp - 1];
    if (threadIdx.x < a.E) {
        base[threadIdx.x] = up - all + before;
        if (cta == 0) {
            a.offsets[threadIdx.x + 1] = up;
            if (threadIdx.x == 0) a.offsets[0] = 0;
        }
    }
    __syncthreads();
    for (int p = p0; p < p1; p += 32 * B) {
        int es[B];
#pragma unroll
        for (int b = 0; b < B; ++b) es[b] = expert(p + 32 * b + lane);
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int q = p + 32 * b + lane, e = es[b];
            if (p + 32 * b >= p1) break;
            const uint32_t same = lanes_alike(e, bits);
            int at = -1;
            if (e >= 0) {
                at = base[e] + mine[e] + __popc(same & ((1u << lane) - 1));
                a.rows[at] = q / a.k;
            }
            if (q < p1) a.place[q] = at;
            __syncwarp();
            if (e >= 0 && (same >> lane) == 1) mine[e] += __popc(same);
            __syncwarp();
        }
    }
    // behind the last place
    const int n = a.T * a.k;
    for (int p = everything + cta * kRouteThreads + threadIdx.x; p < n; p += ctas * kRouteThreads)
        a.rows[p] = -1;
    if (ctas > 1)  // nobody leaves while its counts are read
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

constexpr size_t route_smem_bytes(int E) { return sizeof(int) * (size_t)E * (kRouteWarps + 2); }

// What a kernel may take of shared memory belongs to it, for every thread's calls: the most that
// any call takes, once for each device. (With experts chosen in it k_route_order has at most 256.)
static cudaError_t route_prepare() {
    static_assert(route_smem_bytes(256) < 48 * 1024 - 256, "a launch has that unasked");
    static std::atomic<bool> done[kMaxDevices];
    std::atomic<bool> &mine = done[current_device()];
    if (mine.load()) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void *>(k_route_order<0>),
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)route_smem_bytes(kRouteExperts));
    if (e == cudaSuccess) mine.store(true);
    return e;
}

struct CombineArgs {
    const void *y;
    int64_t ys;
    int y_rows;
    const int *place;
    const float *weights;
    int T, k, cols, shift;
    const void *base;
    int64_t bs;
    void *out;
    int64_t os;
};

constexpr int kCombineThreads = 256;

// Eight elements side by side as they lie in memory (VEC), or four `step` apart, `left` elements
// from the first on.
template <typename T, bool VEC>
struct Piece {
    static constexpr int V = VEC ? 8 : 4;
    using W = typename std::conditional<VEC, uint4, T>::type;
    W w[VEC ? sizeof(T) / 2 : V];
    __device__ __forceinline__ void load(const T *p, int step, int left) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4 *>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = i * step < left ? p[i * step] : from_f32<T>(0.f);
        }
    }
    __device__ __forceinline__ void values(float (&v)[V]) const {
        const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f32(e[i]);
    }
};

// Bound by memory: each row of y is read once. 2^shift threads have a token, a thread eight
// columns at a time (rows that do not lie on 16 bytes: four, 2^shift apart).
template <typename Y, typename O, bool VEC>
__global__ void __launch_bounds__(kCombineThreads, 4) k_combine(const __grid_constant__ CombineArgs a) {
    constexpr int V = VEC ? 8 : 4, B = 2;  // B rows of y in flight
    launch_dependents();
    wait_prerequisite();
    const int t = (blockIdx.x * kCombineThreads + threadIdx.x) >> a.shift;
    if (t >= a.T) return;
    const int *place = a.place + (int64_t)t * a.k;
    const float *weights = a.weights + (int64_t)t * a.k;
    const int step = 1 << a.shift;
    for (int c = (threadIdx.x & (step - 1)) * (VEC ? V : 1); c < a.cols; c += V * step) {
        const int left = a.cols - c;
        Piece<O, VEC> base;
        if (a.base) base.load(static_cast<const O *>(a.base) + t * a.bs + c, step, left);
        float acc[V], v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.f;
        for (int j0 = 0; j0 < a.k; j0 += B) {
            Piece<Y, VEC> d[B];
            float w[B];
            bool some[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int p = j0 + b < a.k ? __ldg(place + j0 + b) : -1;
                some[b] = p >= 0 && p < a.y_rows;
                if (some[b]) {
                    w[b] = __ldg(weights + j0 + b);
                    d[b].load(static_cast<const Y *>(a.y) + p * a.ys + c, step, left);
                }
            }
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (some[b]) {
                    d[b].values(v);
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[e] = fmaf(w[b], v[e], acc[e]);
                }
        }
        if (a.base) {
            base.values(v);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = v[e] + acc[e];
        }
        O *o = static_cast<O *>(a.out) + t * a.os + c;
        if constexpr (VEC) {
            store8<true>(o, acc);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e * step < left) o[e * step] = from_f32<O>(acc[e]);
        }
    }
}

}  // namespace rb

using namespace rb;

extern "C" {

int rabbit_cuda_experts_route_dev(const float *d_scores, int64_t score_stride, int n_tokens,
                                  int n_experts, int k, int over_all, int *d_ids, float *d_weights,
                                  int *d_offsets, int *d_rows, int *d_place, void *stream) {
    if (n_tokens < 0 || n_experts < 1 || n_experts > kRouteExperts || k < 1 || k > kRouteK ||
        k > n_experts || (int64_t)n_tokens * k >= 1 << 30 || (over_all & ~1))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "experts_route: need n_tokens >= 0, n_experts in 1..%d, k in 1..min(n_experts, %d), "
                    "n_tokens * k below 2^30, over_all 0 or 1", kRouteExperts, kRouteK);
    if (!d_offsets || (n_tokens && (!d_ids || !d_rows || !d_place || (d_scores && !d_weights))))
        return fail(RABBIT_CUDA_ERR_ARGS, "experts_route: NULL pointer");
    const uintptr_t off = reinterpret_cast<uintptr_t>(d_scores) | reinterpret_cast<uintptr_t>(d_ids) |
                          reinterpret_cast<uintptr_t>(d_weights) | reinterpret_cast<uintptr_t>(d_offsets) |
                          reinterpret_cast<uintptr_t>(d_rows) | reinterpret_cast<uintptr_t>(d_place);
    RouteArgs a;
    a.scores = d_scores;
    a.stride = score_stride ? score_stride : n_experts;
    if ((off & 3) || (d_scores && a.stride < n_experts))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "experts_route: score_stride below n_experts, or a pointer not aligned to its element");
    a.T = n_tokens;
    a.E = n_experts;
    a.k = k;
    a.over_all = over_all;
    a.ids = d_ids;
    a.weights = d_weights;
    a.offsets = d_offsets;
    a.rows = d_rows;
    a.place = d_place;
    if (!device_sms()) return fail(RABBIT_CUDA_ERR_DEVICE, "experts_route: no device %d", current_device());
    DeviceScope scope(current_device());
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const size_t smem = route_smem_bytes(a.E);
    // Up to a token a warp of the cluster the picks are made by the kernel that orders: one launch.
    // (With more than 256 experts a lane has too many for that kernel's registers.)
    const int v = n_experts <= 32 ? 1 : n_experts <= 64 ? 2 : n_experts <= 128 ? 4 : n_experts <= 256 ? 8 : 32;
    const bool pick = d_scores && n_tokens <= kRouteCluster * kRouteWarps && v <= 8;
    const unsigned ctas = n_tokens <= kRouteWarps ? 1 : kRouteCluster;
    scope.launch(route_prepare(), "experts_route: shared memory");
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    if (d_scores && !pick) {
        const int sms = device_sms();
        const int64_t want = ((int64_t)n_tokens + 7) / 8;
        auto k = v == 1 ? k_route<1> : v == 2 ? k_route<2> : v == 4 ? k_route<4> : v == 8 ? k_route<8> : k_route<32>;
        scope.launch(launch_pdl(k, dim3((unsigned)(want < 8 * sms ? want : 8 * sms)), dim3(256), 0, s, a),
                     "experts_route");
    }
    auto kern = !pick ? k_route_order<0> : v == 1 ? k_route_order<1> : v == 2 ? k_route_order<2>
                : v == 4 ? k_route_order<4> : k_route_order<8>;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kRouteThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
    if (scope.status == RABBIT_CUDA_OK) scope.launch(cudaLaunchKernelEx(&cfg, kern, a), "experts_route");
    return scope.done();
}

int rabbit_cuda_experts_combine_dev(int dtype, const void *d_y, int64_t y_stride, int y_rows,
                                    const int *d_place, const float *d_weights, int n_tokens, int k,
                                    int n_cols, int out_dtype, const void *d_base,
                                    int64_t base_stride, void *d_out, int64_t out_stride,
                                    void *stream) {
    const int ys = dtype_size(dtype), os = dtype_size(out_dtype);
    if (!ys || !os || y_rows < 0 || n_tokens < 0 || n_tokens >= 1 << 23 || k < 1 || k > kRouteK || n_cols < 1 || n_cols > 1 << 20)
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "experts_combine: unknown dtype, a negative count, 2^23 tokens or more, k not in 1..%d or "
                    "n_cols not in 1..2^20", kRouteK);
    if (n_tokens == 0) return ok();
    if (!d_y || !d_place || !d_weights || !d_out)
        return fail(RABBIT_CUDA_ERR_ARGS, "experts_combine: NULL pointer");
    CombineArgs a;
    a.y = d_y;
    a.ys = y_stride ? y_stride : n_cols;
    a.y_rows = y_rows;
    a.place = d_place;
    a.weights = d_weights;
    a.T = n_tokens;
    a.k = k;
    a.cols = n_cols;
    a.base = d_base;
    a.bs = base_stride ? base_stride : n_cols;
    a.out = d_out;
    a.os = out_stride ? out_stride : n_cols;
    const uintptr_t y = reinterpret_cast<uintptr_t>(d_y),
                    o = reinterpret_cast<uintptr_t>(d_base) | reinterpret_cast<uintptr_t>(d_out);
    if (a.ys < n_cols || a.os < n_cols || (d_base && a.bs < n_cols) || (y & (ys - 1)) || (o & (os - 1)) ||
        ((reinterpret_cast<uintptr_t>(d_place) | reinterpret_cast<uintptr_t>(d_weights)) & 3) ||
        (d_base == d_out && a.bs != a.os))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "experts_combine: a stride below n_cols (or different in place), or a pointer not "
                    "aligned to its element");
    const bool vec = (y & 15) == 0 && (o & 15) == 0 && a.ys * ys % 16 == 0 && a.os * os % 16 == 0 &&
                     (!d_base || a.bs * os % 16 == 0) && n_cols % 8 == 0;
    a.shift = 0;  // up to a CTA's threads to a token
    while (a.shift < 8 && (1 << a.shift) * (vec ? 8 : 4) < n_cols) ++a.shift;
    const int64_t threads = (int64_t)n_tokens << a.shift;  // below 2^31
    DeviceScope scope(current_device());
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    const dim3 grid((unsigned)((threads + kCombineThreads - 1) / kCombineThreads));
    with_dtype(dtype, [&](auto yt) {
        return with_dtype(out_dtype, [&](auto ot) {
            using Y = decltype(yt);
            using O = decltype(ot);
            scope.launch(launch_pdl(vec ? k_combine<Y, O, true> : k_combine<Y, O, false>, grid,
                                    dim3(kCombineThreads), 0, static_cast<cudaStream_t>(stream), a),
                         "experts_combine");
            return 0;
        });
    });
    return scope.done();
}

}  // extern "C"
