// Host helpers of the C entry points.
#pragma once
#include <cuda_runtime.h>

namespace w4a16 {

// Device whose primary context this thread has made current through cudaSetDevice.
// A thread that never called it (a worker such as autograd's backward thread) reports
// device 0 from cudaGetDevice but has no current context yet, and driver entry points
// (cuTensorMapEncodeTiled) then fail with CUDA_ERROR_INVALID_CONTEXT.
inline thread_local int t_bound_device = -1;

// Switches to `dev` for the scope, with its context current, and restores the caller's
// device afterwards (the reference calls cudaSetDevice and leaves it changed,
// q4_matmul.cu:248,476).
struct DeviceGuard {
    int prev = -1;
    bool ok = true;
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev || t_bound_device != dev) {
            ok = cudaSetDevice(dev) == cudaSuccess;
            if (ok) t_bound_device = dev;
        }
    }
    ~DeviceGuard() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev && cudaSetDevice(prev) == cudaSuccess)
            t_bound_device = prev;
    }
};

}  // namespace w4a16
