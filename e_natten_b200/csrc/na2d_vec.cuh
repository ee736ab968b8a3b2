// Values of the three element types in vectors of 16, 8, 4 or 2 bytes, as fp32 in registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace na2d_vec {

template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ float narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

// N values of type T that lie together, aligned to their size.
template <typename T, int N>
struct Vec {
    using raw = typename Raw<N * (int)sizeof(T)>::type;
    union {
        raw bits;
        T at[N];
    };
    __device__ __forceinline__ Vec() {}
    __device__ __forceinline__ void load(const T* p) { bits = *reinterpret_cast<const raw*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<raw*>(p) = bits; }
    __device__ __forceinline__ void store_streaming(T* p) const { __stcs(reinterpret_cast<raw*>(p), bits); }       // not read again soon
    __device__ __forceinline__ void widened(float (&f)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = widen(at[i]);
    }
    __device__ __forceinline__ void round(const float (&f)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] = narrow<T>(f[i]);
    }
};

}  // namespace na2d_vec
