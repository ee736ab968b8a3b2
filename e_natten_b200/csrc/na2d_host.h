// What the files with C entry points share on the host: the device of a call, errors, the launch counter.  Defined in na2d_api.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/na2d.h"

namespace na2d_ptx { struct ErrorState; }

namespace na2d_host {

// Makes `device` current for the scope and restores the previous device afterwards.
// cudaSetDevice is called even when `device` already is the thread's current device: a thread that
// has made no runtime call yet (an autograd worker thread, for one) reports device 0 as current
// without having its context bound, and the driver call that encodes tensor maps needs a bound
// context.
struct DeviceScope {
    int prev = -1;
    cudaError_t err = cudaSuccess;
    explicit DeviceScope(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess) err = cudaSetDevice(device);
    }
    ~DeviceScope() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

// Records the error's text for na2d_last_cuda_error; NA2D_ERR_CUDA.
int cuda_fail(cudaError_t e, const char* what);
// Failure of a launcher that encodes tensor maps: a runtime error or a failed encode.
int launch_fail(const char* what);
// Compute-capability check, cached per device.
int check_device(int device);
// The device's error state for kernels with waits (the device must be current).
int error_state(int device, const na2d_ptx::ErrorState** out);
void count_launches(int n);
int sm_count(int device);

// Runs `step` with the device current and checked.
template <typename F>
int on_device(int device, F&& step) {
    DeviceScope scope(device);
    if (scope.err != cudaSuccess) return cuda_fail(scope.err, "cudaSetDevice");
    const int rc = check_device(device);
    return rc != NA2D_OK ? rc : step();
}

// Element strides of a (B, heads, T, C) operand; all three zero means dense, and the stride of a dimension of extent 1 never reaches
// an address.
struct HeadStrides {
    long long b, n, t;
};
inline HeadStrides head_strides(const na2d_heads& x, int B, int heads, int T, int C) {
    const bool dense = x.stride_b == 0 && x.stride_n == 0 && x.stride_t == 0;
    HeadStrides s;
    s.t = dense || T == 1 ? C : x.stride_t;
    s.n = dense || heads == 1 ? (long long)T * s.t : x.stride_n;
    s.b = dense || B == 1 ? (long long)heads * s.n : x.stride_b;
    return s;
}

}  // namespace na2d_host
