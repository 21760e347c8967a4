// Element types of the training operators: loads and stores of a few neighbouring values as fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

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

// N neighbouring values as the 32-bit words they lie in, converted where they are used: what a kernel keeps of loads in flight
// (16-bit values of a conditional load would each take a register).
template <typename T, int N, bool Words = (sizeof(T) * N >= 4)> struct Raw {
  uint32_t w[sizeof(T) * N / 4];
  __device__ __forceinline__ void load(const T* at) {
    if constexpr (sizeof(w) == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(at);
    } else if constexpr (sizeof(w) == 8) {
      const uint2 x = *reinterpret_cast<const uint2*>(at);
      w[0] = x.x, w[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < (int)sizeof(w) / 16; ++i) {
        const uint4 x = reinterpret_cast<const uint4*>(at)[i];
        w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
      }
    }
  }
  __device__ __forceinline__ float get(int k) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[k]);
    const uint32_t half = k & 1 ? w[k / 2] >> 16 : w[k / 2] & 0xffffu;
    if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(half << 16);
    return __half2float(__ushort_as_half((unsigned short)half));
  }
};
// 32 bytes on a 32-byte boundary in one access; load32 of memory that the kernel does not write
template <typename T, int N> __device__ __forceinline__ void load32(Raw<T, N>& x, const T* at) {
  static_assert(sizeof(x.w) == 32);
  asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(x.w[0]), "=r"(x.w[1]), "=r"(x.w[2]), "=r"(x.w[3]), "=r"(x.w[4]), "=r"(x.w[5]), "=r"(x.w[6]), "=r"(x.w[7])
      : "l"(at));
}
template <typename T, int N> __device__ __forceinline__ void store32(T* at, const Pack<T, N>& x) {
  static_assert(sizeof(x) == 32);
  uint32_t w[8];
  memcpy(w, &x, 32);
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
               "r"(w[6]), "r"(w[7])
               : "memory");
}

template <typename T, int N> struct Raw<T, N, false> {  // one 16-bit value
  T v;
  __device__ __forceinline__ void load(const T* at) { v = *at; }
  __device__ __forceinline__ float get(int) const { return to_float(v); }
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
