// rb_linear.cu -- C ABI: products with e4m3 (a scale for each block of 128) or
// 16-bit weights, one matrix or one for each expert (rb_linear.cuh).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <new>

#include "rb_launch.h"
#include "rb_linear_rows.cuh"

struct rabbit_cuda_linear {
    int device = -1;
    rb::DevCtx *ctx = nullptr;
    rabbit_cuda_linear_desc d = {};
    CUtensorMap map = {};
    PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    int *d_err = nullptr;  // the error word, and what a check took of it
    std::mutex taking;     // one check at a time
    std::atomic<int> withhold{0};  // test hook for the next call: a bit for each CTA of a pair
};

namespace rb {

__global__ void k_linear_take(int *err) { err[1] = atomicExch(err, 0); }

static bool aligned(const void *p, uintptr_t n) {
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

static int operand_size(int dtype) {
    return dtype == RABBIT_CUDA_E4M3 ? 1
           : dtype == RABBIT_CUDA_F16 || dtype == RABBIT_CUDA_BF16 ? 2 : 0;
}

using LinKernel = void (*)(LinArgs, CUtensorMap, CUtensorMap);

template <int MODE, bool PAIR>
static LinKernel lin_kernel_of(bool gated, int out_dtype) {
    LinKernel k = nullptr;
    with_dtype(out_dtype, [&](auto t) {
        k = gated ? k_linear<MODE, PAIR, true, decltype(t)> : k_linear<MODE, PAIR, false, decltype(t)>;
        return 0;
    });
    return k;
}
static LinKernel lin_kernel(int mode, bool pair, bool gated, int out_dtype) {
    if (mode == kLinF8 && pair) {
        LinKernel k = nullptr;
        with_dtype(out_dtype, [&](auto t) {
            k = gated ? k_linear_rows<true, decltype(t)> : k_linear_rows<false, decltype(t)>;
            return 0;
        });
        return k;
    }
    if (mode == kLinF8) return lin_kernel_of<kLinF8, false>(gated, out_dtype);
    if (mode == kLinParts)
        return pair ? lin_kernel_of<kLinParts, true>(gated, out_dtype) : lin_kernel_of<kLinParts, false>(gated, out_dtype);
    return pair ? lin_kernel_of<kLinWhole, true>(gated, out_dtype) : lin_kernel_of<kLinWhole, false>(gated, out_dtype);
}

// The current device's kernels for an object, once: their shared memory; `fits`: those that
// share out registers were built to be launched with the 128 a thread that the shares add up to.
static cudaError_t lin_prepare_kernels(int device, bool f8, bool gated, bool *fits) {
    static std::atomic<bool> done[kMaxDevices][4];
    std::atomic<bool> &mine = done[device][2 * f8 + gated];
    if (mine.load()) return cudaSuccess;
    for (int mode = f8 ? kLinF8 : kLinWhole; mode <= (f8 ? kLinF8 : kLinParts); ++mode)
        for (int i = 0; i < 6; ++i) {
            const void *k = reinterpret_cast<const void *>(lin_kernel(mode, i & 1, gated, i >> 1));
            cudaFuncAttributes at;
            cudaError_t e = cudaFuncGetAttributes(&at, k);
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynSmem);
            if (e != cudaSuccess) return e;
            if (mode != kLinWhole && at.numRegs != 128) *fits = false;
        }
    if (*fits) mine.store(true);
    return cudaSuccess;
}

// A map of rows of `cols` elements, `stride` elements apart: boxes of 128 bytes of
// `box` rows, swizzled by 128 bytes; past the rows and columns reads zero.
static bool rows_map(const rabbit_cuda_linear *lin, CUtensorMap *map, const void *base, int rank,
                     const cuuint64_t *dims, const cuuint64_t *strides, int box) {
    const bool f8 = lin->d.dtype == RABBIT_CUDA_E4M3;
    const cuuint32_t boxes[4] = {f8 ? 128u : 64u, (cuuint32_t)box, 1, 1}, one[4] = {1, 1, 1, 1};
    return lin->encode(map, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                       rank, const_cast<void *>(base), dims, strides, boxes, one,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int up_to(int64_t n, int unit) { return (int)((n + unit - 1) / unit * unit); }

// Microseconds that a step of 128 bytes of K takes with tiles of `cols` tokens, and that a
// cluster takes to sum the parts of a tile, from 2048 and 8192 x 1024 .. 14336 at 40 to 512 rows
// (us, one CTA a tile / pairs; n_out 14336 shows the steps, 1024 the sums):
//   bf16 8192 x 14336   64 rows 40 / 39    128 rows 43 / 42    256 rows 58 / 54    512 rows 107 / 95
//   bf16 8192 x 1024    64 rows 14 / 27    128 rows 17 / 30    256 rows 27 / 44    512 rows 50 / 44
//   e4m3 8192 x 14336   64 rows 31 / 40    128 rows 74 / 41    256 rows 110 / 42   512 rows 215 / 75
//   e4m3 8192 x 1024    64 rows 15 / 36    128 rows 24 / 37    256 rows 36 / 37    512 rows 68 / 37
// Groups of fewer rows go by the same numbers. Measured for 8 experts of 64, gated, 2048 x 1024, listed, in a graph:
//   bf16   1 row 15.8 / 16.8    4 rows 15.7 / 16.7    16 rows 15.4 / 16.6    32 rows 25.4 / 16.8
//   e4m3   1 row 14.5 / 18.7                          16 rows 12.2 / 17.3
// so in 16 bits the estimate takes pairs up to 32 rows on where one CTA a tile would save up to 1 us to 16 rows.
static double lin_step_us(bool f8, bool pair, int64_t cols) {
    if (pair) return f8 ? 0.44 : 0.16 + 0.0005 * cols;
    if (f8) return cols <= 64 ? 0.3 : 0.4 + 0.0047 * cols;
    return 0.2 + 0.0006 * cols;
}
static double lin_sum_us(int64_t cols) { return 0.058 * cols; }

// The launch's shape from the sizes alone (the groups' rows are on the device).
static bool lin_plan(LinArgs &a, int mode, int sms, int64_t *tiles, size_t *smem) {
    const bool f8 = mode == kLinF8;
    const int64_t mean = ((int64_t)a.R + a.E - 1) / a.E, groups = a.E < a.R ? a.E : a.R;
    const int outputs = a.gated ? 64 : 128;
    auto div_up = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
    // a pair of CTAs a tile, or one CTA and a split of K: by the estimate above, every
    // expert with the mean's rows
    const int64_t cols = mean < 256 ? mean : 256, token_tiles_est = (a.E == 1 ? 1 : groups) * div_up(mean, 256);
    const double by_pairs = lin_step_us(f8, true, cols) * a.steps *
                            div_up(token_tiles_est * div_up(a.N, 2 * outputs), sms / 2);
    const int64_t one_tiles = token_tiles_est * div_up(a.N, outputs);
    double by_one = 0;
    for (int split = 1; split <= 8 && (split == 1 || (one_tiles * split <= sms && a.steps / split >= 2)); split *= 2) {
        const double us = lin_step_us(f8, false, cols) * div_up(a.steps, split) * div_up(one_tiles * split, sms) +
                          (split > 1 ? lin_sum_us(cols) : 0.0);
        if (split == 1 || us < by_one) {
            by_one = us;
            a.split = split;
        }
    }
    const bool pair = by_pairs < by_one, as_rows = pair && f8;
    if (pair) a.split = 1;
    a.mt = (int)div_up(a.N, pair ? 2 * outputs : outputs);
    a.unit = as_rows ? 256 : pair ? 64 : 16;
    // tokens of a tile: a multiple of 16 or, with more than one box, of the box's rows; room
    // for four times the mean where the experts' rows differ
    const int64_t want = a.E == 1 ? mean : 4 * mean, rows = want < a.R ? want : a.R;
    a.bn = as_rows || rows >= 256 ? 256 : pair ? up_to(rows, 64) : rows <= 16 ? 16 : up_to(rows, 32);
    a.buf_shift = 1;
    while (a.buf_shift < 3 && (2 << a.buf_shift) * a.bn <= 512) ++a.buf_shift;
    a.bufs = 1 << a.buf_shift;
    static_assert(kLinBufs == 1 << 3, "buffers of tensor memory");
    *tiles = (a.E == 1 ? div_up(a.R, a.bn) : groups + a.R / a.bn) * a.mt;
    a.box = as_rows ? 128 : a.bn < 32 ? a.bn : 32;
    a.band = 8;
    const size_t stage = as_rows ? kRowsStage : lin_stage_bytes(pair, a.bn);
    const size_t fixed = as_rows ? lin_rows_fixed(a.E) : lin_fixed(f8, a.gated, a.bn, a.bufs, a.E);
    a.stages = (int)((kMaxDynSmem - fixed) / stage);
    if (a.stages > kLinStages) a.stages = kLinStages;
    *smem = fixed + a.stages * stage;
    return pair;
}

static int lin_run(rabbit_cuda_linear *lin, const char *what, const void *d_x, int64_t x_stride,
                   int x_rows, const float *d_x_scale, int64_t x_scale_stride, const int *d_rows,
                   const int *d_offsets, int out_dtype, void *d_y, int64_t y_stride, int n_rows,
                   void *stream) {
    const rabbit_cuda_linear_desc &d = lin->d;
    const int size = operand_size(d.dtype), out = dtype_size(out_dtype);
    const bool f8 = d.dtype == RABBIT_CUDA_E4M3;
    if (!out || n_rows < 0 || n_rows > 1 << 30)
        return fail(RABBIT_CUDA_ERR_ARGS, "%s: unknown out_dtype, or n_rows not in 0..2^30", what);
    if (n_rows == 0) return ok();
    LinArgs a = {};
    a.N = d.n_out;
    a.E = d.n_experts;
    a.R = n_rows;
    a.x_rows = x_rows;
    a.steps = (int)(((int64_t)d.n_in * size + 127) / 128);
    a.gated = d.gated;
    const int64_t xs = x_stride ? x_stride : d.n_in;
    const int64_t scale_stride = x_scale_stride ? x_scale_stride : a.steps;
    a.xs_stride = (uint32_t)scale_stride;
    a.y_stride = y_stride ? y_stride : d.n_out;
    if (!d_x || !d_y || (f8 && !d_x_scale))
        return fail(RABBIT_CUDA_ERR_ARGS, "%s: NULL pointer", what);
    if (!aligned(d_x, 16) || xs < d.n_in || xs > (1 << 30) || xs * size % 16 || !aligned(d_y, out) ||
        a.y_stride < d.n_out || !aligned(d_rows, 4) || !aligned(d_offsets, 4))
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "%s: x not aligned to 16 bytes, a stride below its row or (x) not a multiple of "
                    "16 bytes, or a pointer not aligned to its element", what);
    if (f8 && (scale_stride < a.steps || scale_stride > 1 << 30 || !aligned(d_x_scale, 4)))
        return fail(RABBIT_CUDA_ERR_ARGS, "%s: x_scale_stride below its row or above 2^30, or scales not aligned", what);
    if (x_rows < 1 || (!d_rows && x_rows < n_rows))
        return fail(RABBIT_CUDA_ERR_ARGS, "%s: x_rows of %d for %d rows", what, x_rows, n_rows);
    // The tensor cores' sums of 16-bit products lose up to 2^-22 of the sum so far at each of K / 16
    // steps: of terms of one sign 2.5e-5 at K 4096 and 1.0e-4 at 16384. Kept to a tenth of half a step of the
    // output (f16: 2^-12 and more, bf16: 2^-9), parts beyond and for fp32 outputs. (8192 x 4096 x 14336 to f16: 780 us in
    // parts, 720 whole; 8192 x 4096 x 4096: 240 and 190.)
    const int whole = out_dtype == RABBIT_CUDA_F16 ? 4096 : out_dtype == RABBIT_CUDA_BF16 ? 16384 : 0;
    const int mode = f8 ? kLinF8 : d.n_in > whole ? kLinParts : kLinWhole;
    int64_t tiles;
    size_t smem;
    const int sms = lin->ctx->sm_count;
    const bool pair = lin_plan(a, mode, sms, &tiles, &smem);
    if (tiles * a.split >= (int64_t)1 << 30)
        return fail(RABBIT_CUDA_ERR_ARGS, "%s: 2^30 tiles or more", what);
    a.offsets = d_offsets;
    a.rows = d_rows;
    a.gather = d_rows && a.bn > 32;
    a.x = static_cast<const uint8_t *>(d_x);
    a.x_bytes = (uint32_t)(xs * size);
    a.k_bytes = d.n_in * size;
    a.vec = aligned(d_y, 16) && a.y_stride * out % 16 == 0;
    a.pairs = aligned(d_y, 2 * out) && a.y_stride % 2 == 0;
    a.xs = d_x_scale;
    a.ws = d.d_scale;
    a.y = d_y;
    a.format = d.dtype == RABBIT_CUDA_BF16;
    a.err = lin->d_err;
    a.wait_ns = wait_limit_ns();
    a.withhold = lin->withhold.exchange(0);
    if (!pair && a.withhold) a.withhold = 1;
    CUtensorMap mx;
    const cuuint64_t dims[2] = {(cuuint64_t)d.n_in, (cuuint64_t)x_rows};
    const cuuint64_t strides[1] = {(cuuint64_t)xs * size};
    if (!rows_map(lin, &mx, d_x, 2, dims, strides, d_rows && !a.gather ? 1 : a.box))
        return fail(RABBIT_CUDA_ERR_DEVICE, "%s: the driver could not encode the rows' tensor map", what);
    DeviceScope scope(lin->device);
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    const int team = pair ? 2 : a.split;
    const int64_t teams = a.split == 1 && tiles > sms / team ? sms / team : tiles;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = team;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(teams * team));
    cfg.blockDim = dim3(kLinThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = team > 1 ? 2 : 1;
    scope.launch(cudaLaunchKernelEx(&cfg, lin_kernel(mode, pair, d.gated, out_dtype), a, lin->map, mx), what);
    return scope.done();
}

}  // namespace rb

using namespace rb;

extern "C" {

int rabbit_cuda_linear_create(const rabbit_cuda_linear_desc *d, int device,
                              rabbit_cuda_linear **out) {
    if (!d || !out) return fail(RABBIT_CUDA_ERR_ARGS, "linear_create: NULL argument");
    *out = nullptr;
    const int size = operand_size(d->dtype);
    if (!size || d->n_experts < 1 || d->n_experts > kLinMaxExperts || (d->gated & ~1) ||
        d->n_out < 1 || d->n_out > 1 << 20 || d->n_in < 1 || d->n_in > 1 << 20)
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "linear_create: need dtype E4M3, F16 or BF16, n_experts in 1..%d, gated 0 or 1, "
                    "n_out and n_in in 1..2^20", kLinMaxExperts);
    const int64_t ws = d->w_stride ? d->w_stride : d->n_in;
    if (!d->d_w || !aligned(d->d_w, 16) || ws < d->n_in || ws > 1 << 30 || ws * size % 16)
        return fail(RABBIT_CUDA_ERR_ARGS,
                    "linear_create: weights NULL or not aligned to 16 bytes, or a stride below n_in "
                    "or not a multiple of 16 bytes");
    if ((size == 1) != (d->d_scale != nullptr) || !aligned(d->d_scale, 4))
        return fail(RABBIT_CUDA_ERR_ARGS, "linear_create: E4M3 weights, and no others, have scales");
    const uint64_t row = (uint64_t)ws * size, matrix = row * d->n_out;
    if (matrix * (1 + d->gated) >= (uint64_t)1 << 40)
        return fail(RABBIT_CUDA_ERR_ARGS, "linear_create: an expert of 2^40 bytes or more");
    int prev = 0;
    cudaGetDevice(&prev);
    int st;
    DevCtx *ctx = dev_ctx(device, &st);
    if (!ctx) {
        cudaSetDevice(prev);
        return st;
    }
    auto *lin = new (std::nothrow) rabbit_cuda_linear();
    if (!lin) {
        cudaSetDevice(prev);
        return fail(RABBIT_CUDA_ERR_MEM, "linear_create: out of host memory");
    }
    lin->device = device;
    lin->ctx = ctx;
    lin->d = *d;
    cudaDriverEntryPointQueryResult found;
    bool fits = true;
    void *fn = nullptr;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found);
    lin->encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    if (e == cudaSuccess && (e = cudaMalloc(&lin->d_err, 2 * sizeof(int))) == cudaSuccess &&
        (e = cudaMemset(lin->d_err, 0, 2 * sizeof(int))) == cudaSuccess &&
        (e = cudaStreamSynchronize(nullptr)) == cudaSuccess)  // zeroed before any stream uses it
        e = lin_prepare_kernels(device, d->dtype == RABBIT_CUDA_E4M3, d->gated, &fits);
    const cuuint64_t dims[4] = {(cuuint64_t)d->n_in, (cuuint64_t)d->n_out, (cuuint64_t)1 + d->gated,
                                (cuuint64_t)d->n_experts};
    const cuuint64_t strides[3] = {row, matrix, matrix * (1 + d->gated)};
    const bool mapped = e == cudaSuccess && fits && found == cudaDriverEntryPointSuccess &&
                        rows_map(lin, &lin->map, d->d_w, 4, dims, strides, d->gated ? 64 : 128);
    if (!mapped) {
        rabbit_cuda_linear_free(lin);
        cudaSetDevice(prev);
        cudaGetLastError();
        return e != cudaSuccess ? cuda_fail(e, "linear_create")
               : !fits ? fail(RABBIT_CUDA_ERR_UNSUPPORTED,
                              "linear_create: kernels built without 128 registers a thread")
                       : fail(RABBIT_CUDA_ERR_DEVICE,
                              "linear_create: the driver could not encode the weights' tensor map");
    }
    cudaSetDevice(prev);
    *out = lin;
    return ok();
}

int rabbit_cuda_linear_free(rabbit_cuda_linear *lin) {
    if (!lin) return ok();
    {
        DeviceScope scope(lin->device);
        if (lin->d_err) cudaFree(lin->d_err);
    }
    delete lin;
    return ok();
}

int rabbit_cuda_linear_dev(rabbit_cuda_linear *lin, const void *d_x, int64_t x_stride,
                           const float *d_x_scale, int64_t x_scale_stride, int out_dtype, void *d_y,
                           int64_t y_stride, int n_rows, void *stream) {
    if (!lin) return fail(RABBIT_CUDA_ERR_ARGS, "linear: NULL object");
    if (lin->d.n_experts != 1)
        return fail(RABBIT_CUDA_ERR_ARGS, "linear: the object has %d experts: rabbit_cuda_linear_grouped_dev",
                    lin->d.n_experts);
    return lin_run(lin, "linear", d_x, x_stride, n_rows, d_x_scale, x_scale_stride, nullptr, nullptr,
                   out_dtype, d_y, y_stride, n_rows, stream);
}

int rabbit_cuda_linear_grouped_dev(rabbit_cuda_linear *lin, const void *d_x, int64_t x_stride,
                                   int x_rows, const float *d_x_scale, int64_t x_scale_stride,
                                   const int *d_rows, const int *d_offsets, int out_dtype,
                                   void *d_y, int64_t y_stride, int n_rows, void *stream) {
    if (!lin) return fail(RABBIT_CUDA_ERR_ARGS, "linear_grouped: NULL object");
    if (!d_offsets) return fail(RABBIT_CUDA_ERR_ARGS, "linear_grouped: NULL offsets");
    return lin_run(lin, "linear_grouped", d_x, x_stride, x_rows, d_x_scale, x_scale_stride, d_rows,
                   d_offsets, out_dtype, d_y, y_stride, n_rows, stream);
}

int rabbit_cuda_linear_debug_withhold(rabbit_cuda_linear *lin) {
    if (!lin) return fail(RABBIT_CUDA_ERR_ARGS, "linear_debug_withhold: NULL object");
    lin->withhold.store(3);
    return ok();
}

int rabbit_cuda_linear_debug_withhold_cta(rabbit_cuda_linear *lin, int cta) {
    if (!lin || (cta & ~1))
        return fail(RABBIT_CUDA_ERR_ARGS, "linear_debug_withhold_cta: NULL object, or a CTA other than 0 and 1");
    lin->withhold.store(1 << cta);
    return ok();
}

int rabbit_cuda_linear_check(rabbit_cuda_linear *lin, void *stream) {
    if (!lin) return fail(RABBIT_CUDA_ERR_ARGS, "linear_check: NULL object");
    DeviceScope scope(lin->device);
    if (scope.status != RABBIT_CUDA_OK) return scope.status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int h = 0;
    RB_CUDA(cudaStreamSynchronize(s));
    {
        std::lock_guard<std::mutex> hold(lin->taking);
        k_linear_take<<<1, 1, 0, s>>>(lin->d_err);
        RB_CUDA(cudaGetLastError());
        RB_CUDA(cudaMemcpyAsync(&h, lin->d_err + 1, sizeof(int), cudaMemcpyDeviceToHost, s));
        RB_CUDA(cudaStreamSynchronize(s));
    }
    if (h == 0) return ok();
    return fail(h & RB_LIN_ERR_WAIT ? RABBIT_CUDA_ERR_TIMEOUT : RABBIT_CUDA_ERR_ARGS, "linear: %s%s%s%s%s",
                h & RB_LIN_ERR_WAIT ? "a bounded device wait ran out; " : "",
                h & RB_LIN_ERR_OPEN ? "copies or products did not end; " : "",
                h & (RB_LIN_ERR_OFFSETS | RB_LIN_ERR_ROWS) ? "out of range on the device:" : "",
                h & RB_LIN_ERR_OFFSETS ? " offsets" : "", h & RB_LIN_ERR_ROWS ? " rows" : "");
}

}  // extern "C"
