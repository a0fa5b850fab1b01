// Backward pass of a linear layer's activation:  dz = g act'(z), and the column sums of dz, the bias's gradient, in the same pass.
//
// Memory bounds it: two matrices in, one out, 3 N M elements.  A block takes 128 rows (or fewer) of a slab of columns; a thread keeps
// eight columns, so the sums stay in its registers and meet in shared memory once per block.  Blocks leave one row of partial sums
// each, added afterwards in order: no atomics, the same result every time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/void_b200.h"
#include "epilogue.cuh"
#include "experts.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace vb {

namespace {

// act'(z).  With s = sigmoid(w(z)): (z s)' = s + z s (1 - s) w'(z).
__device__ __forceinline__ float slope(float z, int act) {
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
struct RunsOfTokens {   // experts: a block takes a chunk of one expert's tokens (experts.cu)
  const int32_t* head;
  const int32_t* chunk_ptr;
  const int4* chunks;
};
struct NoRuns {};
template <bool RUNS>
using RunsIf = std::conditional_t<RUNS, RunsOfTokens, NoRuns>;

// VEC: elements of a 16-byte piece of rows that lie on such boundaries, else 1.
template <typename T, int VEC, bool RUNS>
__global__ void __launch_bounds__(kGradThreads) activation_grad_kernel(const __grid_constant__ ActivationGradParams p, const __grid_constant__ RunsIf<RUNS> runs) {
  constexpr int WARPS = kGradThreads / 32;
  __shared__ float part[WARPS][32 * VEC];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = (blockIdx.x * 32 + lane) * VEC;
  int r0 = blockIdx.y * kGradRows, r1 = r0 + kGradRows < p.rows ? r0 + kGradRows : p.rows;
  if constexpr (RUNS) {
    if ((int)blockIdx.y >= runs.head[0]) return;
    const int4 c = runs.chunks[blockIdx.y];
    r0 = c.y;
    r1 = c.z;
  }
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
        if (p.act != VOID_ACT_NONE) *reinterpret_cast<uint4*>(zv) = *reinterpret_cast<const uint4*>(z);
      } else {
        gv[0] = *g;
        if (p.act != VOID_ACT_NONE) zv[0] = *z;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = p.act != VOID_ACT_NONE ? value<T>(gv[e]) * slope(value<T>(zv[e]), p.act) : value<T>(gv[e]);
        s[e] += d;
        o[e] = rounded<T>(d);
      }
      if (p.dz == nullptr) continue;
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
// RUNS: the chunks of expert blockIdx.y.
template <typename P, bool RUNS>
__global__ void __launch_bounds__(256) partial_sums_kernel(const float* partials, int blocks, int cols, P* out, const __grid_constant__ RunsIf<RUNS> runs) {
  __shared__ float part[8][32];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  int first = 0;
  if constexpr (RUNS) {
    first = runs.chunk_ptr[blockIdx.y];
    blocks = runs.chunk_ptr[blockIdx.y + 1];
    out += (size_t)blockIdx.y * (size_t)cols;
  }
  float s = 0.0f;
  if (c < cols)
#pragma unroll 4
    for (int k = first + warp; k < blocks; k += 8) s += partials[(size_t)k * (size_t)cols + c];
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

// blocks: row blocks, or chunks there can be at most; experts: of runs
template <typename T, typename P, bool RUNS>
int activation_grad(const ActivationGradParams& p, const RunsIf<RUNS>& runs, int blocks, int experts, P* dbias, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  auto on16 = [](const void* m, long long ld) { return (reinterpret_cast<uintptr_t>(m) & 15u) == 0 && ld % V == 0; };
  const bool wide = p.cols % V == 0 && on16(p.g, p.ldg) && on16(p.z, p.ldz) && on16(p.dz, p.lddz);
  cudaError_t rc = cudaSuccess;
  if (blocks > 0) {
    if (wide)
      rc = launch_pdl(activation_grad_kernel<T, V, RUNS>, dim3((unsigned)((p.cols + 32 * V - 1) / (32 * V)), (unsigned)blocks), kGradThreads, 0, st, p, runs);
    else rc = launch_pdl(activation_grad_kernel<T, 1, RUNS>, dim3((unsigned)((p.cols + 31) / 32), (unsigned)blocks), kGradThreads, 0, st, p, runs);
  }
  if (rc == cudaSuccess && dbias != nullptr)
    rc = launch_pdl(partial_sums_kernel<P, RUNS>, dim3((unsigned)((p.cols + 31) / 32), (unsigned)experts), 256, 0, st, p.partials, blocks, p.cols, dbias, runs);
  return status_of(rc);
}
template <bool RUNS>
int activation_grad(const ActivationGradParams& p, const RunsIf<RUNS>& runs, int blocks, int experts, int elem, void* dbias, int bias_elem, cudaStream_t st) {
  using H = __half;
  using B = __nv_bfloat16;
  float* f = reinterpret_cast<float*>(dbias);
  if (elem == VOID_ELEM_F32) return activation_grad<float, float, RUNS>(p, runs, blocks, experts, f, st);
  if (elem == VOID_ELEM_F16)
    return bias_elem == VOID_ELEM_F32 ? activation_grad<H, float, RUNS>(p, runs, blocks, experts, f, st)
                                      : activation_grad<H, H, RUNS>(p, runs, blocks, experts, reinterpret_cast<H*>(dbias), st);
  return bias_elem == VOID_ELEM_F32 ? activation_grad<B, float, RUNS>(p, runs, blocks, experts, f, st)
                                    : activation_grad<B, B, RUNS>(p, runs, blocks, experts, reinterpret_cast<B*>(dbias), st);
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
  return activation_grad<false>(p, NoRuns{}, row_blocks(rows), 1, elem, dbias, bias_elem, reinterpret_cast<cudaStream_t>(stream));
}

size_t void_expert_activation_grad_ws_bytes(const void_experts* x, int32_t rows, int32_t cols) {
  if (x == nullptr || x->n_experts < 1 || x->chunk < 1 || rows <= 0 || cols <= 0) return 0;
  return (size_t)vb::plan_capacity(x->n_experts, rows, x->chunk) * (size_t)cols * sizeof(float);
}

int void_expert_activation_grad(const void* g, int64_t ldg, const void* z, int64_t ldz, int32_t elem, const void_experts* x, int32_t rows,
                                int32_t cols, int32_t act, void* dz, int64_t lddz, void* dbias, int32_t bias_elem, void* ws, size_t ws_bytes,
                                void_stream_t stream) {
  using namespace vb;
  if (x == nullptr || x->plan == nullptr || x->n_experts < 1 || x->chunk < 1) return VOID_ERR_BAD_ARG;
  if (elem < VOID_ELEM_F32 || elem > VOID_ELEM_BF16 || rows < 0 || cols < 0 || act < VOID_ACT_NONE || act > VOID_ACT_SILU) return VOID_ERR_BAD_ARG;
  if (ldg < cols || (z != nullptr && ldz < cols) || (dz != nullptr && lddz < cols)) return VOID_ERR_BAD_ARG;
  if (dbias != nullptr && bias_elem != elem && bias_elem != VOID_ELEM_F32) return VOID_ERR_BAD_ARG;
  if (cols == 0 || (rows == 0 && dbias == nullptr)) return VOID_OK;
  if (rows > 0 && (g == nullptr || (act != VOID_ACT_NONE && (z == nullptr || dz == nullptr)))) return VOID_ERR_BAD_ARG;
  const PlanView v = plan_of(*x, rows);
  if (v.capacity > 65535 || x->n_experts > 65535) return VOID_ERR_TOO_LARGE;
  if (dbias != nullptr && rows > 0 && (ws == nullptr || ws_bytes < void_expert_activation_grad_ws_bytes(x, rows, cols))) return VOID_ERR_WORKSPACE;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  const ActivationGradParams p = {g, z, dz, dbias != nullptr ? reinterpret_cast<float*>(ws) : nullptr, ldg, ldz, lddz, rows, cols, act};
  const RunsOfTokens runs = {v.head, v.chunk_ptr, v.chunks};
  return activation_grad<true>(p, runs, v.capacity, x->n_experts, elem, dbias, bias_elem, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
