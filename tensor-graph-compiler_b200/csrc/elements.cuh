// Element types of the token-generation kernels: float32, bfloat16 and float16 values read and
// written as float32 (to 16 bits by rounding to nearest even, once, on the store).
#ifndef TGCB_ELEMENTS_CUH_
#define TGCB_ELEMENTS_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "tgcb.h"

namespace tgcb_elem {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// A 16-byte vector of T as floats.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  union {
    uint4 raw;
    T e[N];
  };
  __device__ Vec() {}
};

template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float* in) {
  Vec<T> v;
#pragma unroll
  for (int i = 0; i < Vec<T>::N; ++i) v.e[i] = from_float<T>(in[i]);
  *reinterpret_cast<uint4*>(p) = v.raw;
}

// Element i of an array whose type is known at run time (gains: few, and read once per row).
__device__ __forceinline__ float load_any(const void* p, int dtype, int i) {
  if (dtype == TGCB_F32) return static_cast<const float*>(p)[i];
  if (dtype == TGCB_BF16) return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_any(void* p, int dtype, int i, float x) {
  if (dtype == TGCB_F32)
    static_cast<float*>(p)[i] = x;
  else if (dtype == TGCB_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = from_float<__nv_bfloat16>(x);
  else
    static_cast<__half*>(p)[i] = from_float<__half>(x);
}

}  // namespace tgcb_elem

#endif  // TGCB_ELEMENTS_CUH_
