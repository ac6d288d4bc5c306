// rb_launch.h -- programmatic-dependent launches, and the device scope of an
// entry point that leaves the caller's current device as it found it.
#pragma once
#include <cuda_runtime.h>

#include "rb_runtime.h"

namespace rb {

// Launch `kern` so that it may start while the kernel before it on the stream
// drains; every thread of such a kernel calls wait_prerequisite() before it
// touches memory.
template <typename... Args>
inline cudaError_t launch_pdl(void (*kern)(Args...), dim3 grid, dim3 block, size_t smem,
                              cudaStream_t s, const Args &...args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Makes `device` current for the calling thread until the scope ends.
// Allocates nothing, so it may be used while a stream captures.
struct DeviceScope {
    int prev = -1, status = RABBIT_CUDA_OK;
    explicit DeviceScope(int device) {
        cudaError_t e = cudaGetDevice(&prev);
        if (e == cudaSuccess && prev != device) e = cudaSetDevice(device);
        else if (e == cudaSuccess) prev = -1;
        if (e != cudaSuccess) status = cuda_fail(e, "cudaSetDevice");
    }
    ~DeviceScope() {
        if (prev >= 0) cudaSetDevice(prev);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
    // Record a launch's result; the first failure stays.
    void launch(cudaError_t e, const char *what) {
        if (e != cudaSuccess && status == RABBIT_CUDA_OK) status = cuda_fail(e, what);
    }
    int done() const { return status == RABBIT_CUDA_OK ? ok() : status; }
};

}  // namespace rb
