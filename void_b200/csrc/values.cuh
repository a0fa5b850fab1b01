// Elements of fp32, fp16 and bf16 rows as fp32 numbers, one by one or in 16-byte pieces.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace vb {

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The elements of a whole 16-byte piece as they lie.
template <typename T, int VEC = 16 / (int)sizeof(T)>
struct Piece {
  static_assert(VEC * sizeof(T) == 16, "a piece is 16 bytes");
  T v[VEC];
  __device__ __forceinline__ void load(const T* at) {
    const uint4 u = *reinterpret_cast<const uint4*>(at);
    memcpy(v, &u, 16);
  }
  __device__ __forceinline__ void store(T* at) const {
    uint4 u;
    memcpy(&u, v, 16);
    *reinterpret_cast<uint4*>(at) = u;
  }
  __device__ __forceinline__ float get(int e) const { return to_float<T>(v[e]); }
  __device__ __forceinline__ void set(int e, float x) { v[e] = from_float<T>(x); }
};
// One element of a vector of fp32, fp16 or bf16 numbers whose type the launch knows (VOID_ELEM_*).
__device__ __forceinline__ float element(const void* at, int elem, long long i) {
  if (elem == 0) return reinterpret_cast<const float*>(at)[i];
  return elem == 1 ? __half2float(reinterpret_cast<const __half*>(at)[i]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(at)[i]);
}
__device__ __forceinline__ void set_element(void* at, int elem, long long i, float v) {
  if (elem == 0) reinterpret_cast<float*>(at)[i] = v;
  else if (elem == 1) reinterpret_cast<__half*>(at)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(at)[i] = __float2bfloat16_rn(v);
}

// The same in two steps: the loads of several elements are on their way together, which a conversion behind each would prevent.
__device__ __forceinline__ uint32_t raw_element(const void* at, int elem, long long i) {
  return elem == 0 ? reinterpret_cast<const uint32_t*>(at)[i] : (uint32_t)reinterpret_cast<const uint16_t*>(at)[i];
}
__device__ __forceinline__ float of_raw(uint32_t u, int elem) {
  return elem == 0 ? __uint_as_float(u) : (elem == 1 ? __half2float(__ushort_as_half((unsigned short)u)) : __uint_as_float(u << 16));
}

}  // namespace vb
