// Element types of the training operators: loads and stores of a few neighbouring values as fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "gridnerf_b200.h"

inline int gnr_type_size(int type) { return type == GNR_FP32 ? 4 : type == GNR_FP16 || type == GNR_BF16 ? 2 : 0; }

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N neighbouring values as one access of up to 16 bytes (two of them for 8 fp32 values).
template <typename T, int N> struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
  T v[N];
};

// Calls f(value of the C++ type that `type` names).
template <typename F> int gnr_with_type(int type, F f) {
  switch (type) {
    case GNR_FP32: return f(float());
    case GNR_FP16: return f(__half());
    case GNR_BF16: return f(__nv_bfloat16());
  }
  return -1;
}
