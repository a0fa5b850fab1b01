// Backward pass of a linear layer's activation:  dz = g act'(z), and the column sums of dz, the bias's gradient, in the same pass.
//
// Memory bounds it: two matrices in, one out, 3 N M elements.  A block takes 128 rows (or fewer) of a slab of columns; a thread keeps
// eight columns, so the sums stay in its registers and meet in shared memory once per block.  Blocks leave one row of partial sums
// each, added afterwards in order: no atomics, the same result every time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/void_b200.h"
#include "epilogue.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace vb {

namespace {

// act'(z).  With s = sigmoid(w(z)): (z s)' = s + z s (1 - s) w'(z).
__device__ __forceinline__ float slope(float z, int act) {
  if (act == VOID_ACT_NONE) return 1.0f;
  if (act == VOID_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  // (kGelu1, kGelu3 and kSilu carry -log2(e), for a sigmoid of powers of two)
  const bool gelu = act == VOID_ACT_GELU;
  const float s = sigmoid_exp2(z * (gelu ? fmaf(z * z, kGelu3, kGelu1) : kSilu));
  const float inner = gelu ? fmaf(z * z, kGelu3 * (-3.0f / (float)kLog2e), kGelu1 * (-1.0f / (float)kLog2e)) : 1.0f;
  // (far out s is 0 or 1 to the last bit while z grows: nothing is left of the second term)
  const float rest = s * (1.0f - s);
  return rest > 0.0f ? fmaf(z * rest, inner, s) : s;
}

template <typename T> __device__ __forceinline__ float value(T v);
template <> __device__ __forceinline__ float value<float>(float v) { return v; }
template <> __device__ __forceinline__ float value<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float value<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr int kGradRows = 128, kGradThreads = 256;

struct ActivationGradParams {
  const void *g, *z;
  void* dz;
  float* partials;   // [row blocks][cols], or null
  long long ldg, ldz, lddz;
  int rows, cols, act;
};

// VEC: elements of a 16-byte piece of rows that lie on such boundaries, else 1.
template <typename T, int VEC>
__global__ void __launch_bounds__(kGradThreads) activation_grad_kernel(const __grid_constant__ ActivationGradParams p) {
  constexpr int WARPS = kGradThreads / 32;
  __shared__ float part[WARPS][32 * VEC];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = (blockIdx.x * 32 + lane) * VEC;
  const int r0 = blockIdx.y * kGradRows, r1 = r0 + kGradRows < p.rows ? r0 + kGradRows : p.rows;
  float s[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) s[e] = 0.0f;
  if (c0 < p.cols) {
#pragma unroll 4
    for (int r = r0 + warp; r < r1; r += WARPS) {
      const T *g = reinterpret_cast<const T*>(p.g) + (long long)r * p.ldg + c0, *z = reinterpret_cast<const T*>(p.z) + (long long)r * p.ldz + c0;
      T* dz = reinterpret_cast<T*>(p.dz) + (long long)r * p.lddz + c0;
      __align__(16) T gv[VEC], zv[VEC], o[VEC];
      if constexpr (VEC > 1) {
        *reinterpret_cast<uint4*>(gv) = *reinterpret_cast<const uint4*>(g);
        *reinterpret_cast<uint4*>(zv) = *reinterpret_cast<const uint4*>(z);
      } else {
        gv[0] = *g;
        zv[0] = *z;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = value<T>(gv[e]) * slope(value<T>(zv[e]), p.act);
        s[e] += d;
        o[e] = rounded<T>(d);
      }
      if constexpr (VEC > 1) *reinterpret_cast<uint4*>(dz) = *reinterpret_cast<const uint4*>(o);
      else *dz = o[0];
    }
  }
  grid_launch_dependents();
  if (p.partials == nullptr) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e) part[warp][lane * VEC + e] = s[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += kGradThreads) {
    const int c = blockIdx.x * 32 * VEC + i;
    if (c >= p.cols) continue;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum += part[w][i];
    p.partials[(size_t)blockIdx.y * (size_t)p.cols + c] = sum;
  }
}

// The row blocks' partial sums, in order: 32 columns and eight strands of blocks per block.
template <typename P>
__global__ void __launch_bounds__(256) partial_sums_kernel(const float* partials, int blocks, int cols, P* out) {
  __shared__ float part[8][32];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < cols)
#pragma unroll 4
    for (int k = warp; k < blocks; k += 8) s += partials[(size_t)k * (size_t)cols + c];
  part[warp][lane] = s;
  __syncthreads();
  grid_launch_dependents();
  if (warp == 0 && c < cols) {
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += part[k][lane];
    out[c] = rounded<P>(s);
  }
}

int row_blocks(int rows) { return (rows + kGradRows - 1) / kGradRows; }

template <typename T, typename P>
int activation_grad(const ActivationGradParams& p, P* dbias, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  auto on16 = [](const void* m, long long ld) { return (reinterpret_cast<uintptr_t>(m) & 15u) == 0 && ld % V == 0; };
  const bool wide = p.cols % V == 0 && on16(p.g, p.ldg) && on16(p.z, p.ldz) && on16(p.dz, p.lddz);
  const int blocks = row_blocks(p.rows);
  cudaError_t rc = cudaSuccess;
  if (blocks > 0) {
    if (wide) rc = launch_pdl(activation_grad_kernel<T, V>, dim3((unsigned)((p.cols + 32 * V - 1) / (32 * V)), (unsigned)blocks), kGradThreads, 0, st, p);
    else rc = launch_pdl(activation_grad_kernel<T, 1>, dim3((unsigned)((p.cols + 31) / 32), (unsigned)blocks), kGradThreads, 0, st, p);
  }
  if (rc == cudaSuccess && dbias != nullptr)
    rc = launch_pdl(partial_sums_kernel<P>, dim3((unsigned)((p.cols + 31) / 32)), 256, 0, st, p.partials, blocks, p.cols, dbias);
  return status_of(rc);
}

}  // namespace

}  // namespace vb

extern "C" {

size_t void_activation_grad_ws_bytes(int32_t rows, int32_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : (size_t)vb::row_blocks(rows) * (size_t)cols * sizeof(float);
}

int void_activation_grad(const void* g, int64_t ldg, const void* z, int64_t ldz, int32_t elem, int32_t rows, int32_t cols, int32_t act,
                         void* dz, int64_t lddz, void* dbias, int32_t bias_elem, void* ws, size_t ws_bytes, void_stream_t stream) {
  using namespace vb;
  if (elem < VOID_ELEM_F32 || elem > VOID_ELEM_BF16 || rows < 0 || cols < 0 || act < VOID_ACT_NONE || act > VOID_ACT_SILU) return VOID_ERR_BAD_ARG;
  if (ldg < cols || ldz < cols || lddz < cols) return VOID_ERR_BAD_ARG;
  if (dbias != nullptr && bias_elem != elem && bias_elem != VOID_ELEM_F32) return VOID_ERR_BAD_ARG;
  if (cols == 0 || (rows == 0 && dbias == nullptr)) return VOID_OK;
  if (rows > 0 && (g == nullptr || z == nullptr || dz == nullptr)) return VOID_ERR_BAD_ARG;
  if (row_blocks(rows) > 65535) return VOID_ERR_TOO_LARGE;
  if (dbias != nullptr && rows > 0 && (ws == nullptr || ws_bytes < void_activation_grad_ws_bytes(rows, cols))) return VOID_ERR_WORKSPACE;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  const ActivationGradParams p = {g, z, dz, dbias != nullptr ? reinterpret_cast<float*>(ws) : nullptr, ldg, ldz, lddz, rows, cols, act};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool wide_bias = bias_elem == VOID_ELEM_F32;
  if (elem == VOID_ELEM_F32) return activation_grad<float, float>(p, reinterpret_cast<float*>(dbias), st);
  if (elem == VOID_ELEM_F16)
    return wide_bias ? activation_grad<__half, float>(p, reinterpret_cast<float*>(dbias), st) : activation_grad<__half, __half>(p, reinterpret_cast<__half*>(dbias), st);
  return wide_bias ? activation_grad<__nv_bfloat16, float>(p, reinterpret_cast<float*>(dbias), st)
                   : activation_grad<__nv_bfloat16, __nv_bfloat16>(p, reinterpret_cast<__nv_bfloat16*>(dbias), st);
}

}  // extern "C"
