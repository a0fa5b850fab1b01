// Layer norm over the features of each token, forward and backward:
//
//     xh = (x - mean) / sqrt(var + eps)          y = xh w + b                       per token, D features
//     gw = g w       dx = rstd (gw - mean(gw) - xh mean(gw xh))       dw = sum over tokens of g xh       db = sum over tokens of g
//
// Memory bounds both: 2 D elements per token forward (x, y), 3 D backward (g, x, dx).  A token's row stays in registers between its
// reductions, so it comes in once; the variance is the mean square of the centred values (two passes over registers: no
// cancellation for rows with a large mean).  All sums are fp32.  Backward, the block walks many rows and a thread keeps the same
// columns throughout, so the sums over tokens stay in its registers; they leave as one row of partial sums per block, which a second
// kernel adds in block order: no atomics, the result does not depend on which block ran when.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/void_b200.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace vb {

namespace {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC consecutive elements, moved in pieces of up to 16 bytes.
template <typename T, int VEC>
struct Pack {
  static constexpr int BYTES = (int)sizeof(T) * VEC, PIECE = BYTES < 16 ? BYTES : 16, N = BYTES / PIECE;
  T e[VEC];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (PIECE == 16) reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
      else e[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (PIECE == 16) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
      else p[i] = e[i];
    }
  }
} __attribute__((aligned(16)));

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the block; `s` has a word per warp and is free again behind the block's next barrier but one (callers alternate).
__device__ __forceinline__ float block_sum(float v, float* s) {
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  v = warp_sum(v);
  if (lane == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < warps ? s[lane] : 0.0f);
}

constexpr int kRowWarps = 4;   // rows of a block whose warps take a row each

struct NormParams {
  const void *x, *weight, *bias;
  void* y;
  float* stats;   // [2][rows]: mean, rstd; or null
  long long ldx, ldy, rows;
  int cols;
  float eps;
};

// WARP: a warp takes a row (kRowWarps of them per block), else the block does.
template <typename T, typename P, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kRowWarps : 1024) layer_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float sums[2][32];
  grid_dependency_wait();
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x, step = WARP ? 32 : blockDim.x;
  const long long row = WARP ? (long long)blockIdx.x * kRowWarps + (threadIdx.x >> 5) : (long long)blockIdx.x;
  if (WARP && row >= p.rows) return;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
  const P *w = reinterpret_cast<const P*>(p.weight), *b = reinterpret_cast<const P*>(p.bias);
  Pack<T, VEC> v[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (t + k * step) * VEC;
    if (i < p.cols) v[k].load(x + i);
  }
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if ((t + k * step) * VEC < p.cols)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += to_float(v[k].e[e]);
  const float n = (float)p.cols;
  const float mean = (WARP ? warp_sum(s) : block_sum(s, sums[0])) / n;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if ((t + k * step) * VEC < p.cols)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float c = to_float(v[k].e[e]) - mean;
        s = fmaf(c, c, s);
      }
  const float rstd = 1.0f / sqrtf((WARP ? warp_sum(s) : block_sum(s, sums[1])) / n + p.eps);
  if (p.stats != nullptr && t == 0) {
    p.stats[row] = mean;
    p.stats[p.rows + row] = rstd;
  }
  grid_launch_dependents();
  T* y = reinterpret_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (t + k * step) * VEC;
    if (i >= p.cols) continue;
    Pack<P, VEC> wv, bv;
    if (w != nullptr) wv.load(w + i);
    if (b != nullptr) bv.load(b + i);
    Pack<T, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float r = (to_float(v[k].e[e]) - mean) * rstd;
      if (w != nullptr) r *= to_float(wv.e[e]);
      if (b != nullptr) r += to_float(bv.e[e]);
      o.e[e] = from_float<T>(r);
    }
    o.store(y + i);
  }
}

// Rows longer than a block's registers: three passes, the second and third mostly from L2.
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(const __grid_constant__ NormParams p) {
  __shared__ float sums[2][32];
  grid_dependency_wait();
  const long long row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
  const P *w = reinterpret_cast<const P*>(p.weight), *b = reinterpret_cast<const P*>(p.bias);
  float s = 0.0f;
  for (int i = threadIdx.x * VEC; i < p.cols; i += 1024 * VEC) {
    Pack<T, VEC> v;
    v.load(x + i);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += to_float(v.e[e]);
  }
  const float n = (float)p.cols;
  const float mean = block_sum(s, sums[0]) / n;
  s = 0.0f;
  for (int i = threadIdx.x * VEC; i < p.cols; i += 1024 * VEC) {
    Pack<T, VEC> v;
    v.load(x + i);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float c = to_float(v.e[e]) - mean;
      s = fmaf(c, c, s);
    }
  }
  const float rstd = 1.0f / sqrtf(block_sum(s, sums[1]) / n + p.eps);
  if (p.stats != nullptr && threadIdx.x == 0) {
    p.stats[row] = mean;
    p.stats[p.rows + row] = rstd;
  }
  T* y = reinterpret_cast<T*>(p.y) + row * p.ldy;
  for (int i = threadIdx.x * VEC; i < p.cols; i += 1024 * VEC) {
    Pack<T, VEC> v, o;
    Pack<P, VEC> wv, bv;
    v.load(x + i);
    if (w != nullptr) wv.load(w + i);
    if (b != nullptr) bv.load(b + i);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float r = (to_float(v.e[e]) - mean) * rstd;
      if (w != nullptr) r *= to_float(wv.e[e]);
      if (b != nullptr) r += to_float(bv.e[e]);
      o.e[e] = from_float<T>(r);
    }
    o.store(y + i);
  }
  grid_launch_dependents();
}

struct NormGradParams {
  const void *g, *x, *weight;
  const float* stats;
  void* dx;         // or null
  float* partials;  // [blocks][2][cols]: sums of g xh and of g over the block's rows; or null
  long long ldg, ldx, lddx, rows;
  int cols;
};

// One barrier per row: both sums meet in it, in one of two places in turn.
__device__ __forceinline__ float2 block_sum2(float a, float b, float2* s) {
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  a = warp_sum(a);
  b = warp_sum(b);
  if (lane == 0) s[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  const float2 v = lane < warps ? s[lane] : make_float2(0.0f, 0.0f);
  return make_float2(warp_sum(v.x), warp_sum(v.y));
}

// (the next row's loads are in flight while this row's sums are taken, as far as registers reach)
template <typename T, typename P, int VEC, int NV>
__global__ void __launch_bounds__(1024) layer_norm_grad_kernel(const __grid_constant__ NormGradParams p) {
  constexpr int C = VEC * NV;
  __shared__ float2 sums[2][32];
  grid_dependency_wait();
  const int t = threadIdx.x, step = blockDim.x;
  const P* w = reinterpret_cast<const P*>(p.weight);
  float dw[C], db[C];
#pragma unroll
  for (int c = 0; c < C; ++c) dw[c] = db[c] = 0.0f;
  Pack<T, VEC> xv[NV], gv[NV];
  float mean = 0.0f, rstd = 0.0f;
  auto fetch = [&](long long row) {
    const T *x = reinterpret_cast<const T*>(p.x) + row * p.ldx, *g = reinterpret_cast<const T*>(p.g) + row * p.ldg;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (t + k * step) * VEC;
      if (i < p.cols) {
        xv[k].load(x + i);
        gv[k].load(g + i);
      }
    }
    mean = p.stats[row];
    rstd = p.stats[p.rows + row];
  };
  if (blockIdx.x < p.rows) fetch(blockIdx.x);
  int turn = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    float xh[C], gw[C], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (t + k * step) * VEC;
      Pack<P, VEC> wv;
      if (i < p.cols && w != nullptr) wv.load(w + i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int c = k * VEC + e;
        xh[c] = gw[c] = 0.0f;
        if (i < p.cols) {
          const float g = to_float(gv[k].e[e]);
          xh[c] = (to_float(xv[k].e[e]) - mean) * rstd;
          gw[c] = w != nullptr ? g * to_float(wv.e[e]) : g;
          dw[c] = fmaf(g, xh[c], dw[c]);
          db[c] += g;
          s1 += gw[c];
          s2 = fmaf(gw[c], xh[c], s2);
        }
      }
    }
    const float r = rstd;
    if (row + gridDim.x < p.rows) fetch(row + gridDim.x);
    if (p.dx == nullptr) continue;
    const float2 both = block_sum2(s1, s2, sums[turn]);
    const float n = (float)p.cols, m1 = both.x / n, m2 = both.y / n;
    T* dx = reinterpret_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (t + k * step) * VEC;
      if (i >= p.cols) continue;
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.e[e] = from_float<T>(r * (gw[k * VEC + e] - m1 - xh[k * VEC + e] * m2));
      o.store(dx + i);
    }
  }
  if (p.partials != nullptr) {
    float* out = p.partials + (size_t)blockIdx.x * 2 * (size_t)p.cols;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (t + k * step) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (i < p.cols) {
          out[i + e] = dw[k * VEC + e];
          out[(size_t)p.cols + i + e] = db[k * VEC + e];
        }
    }
  }
  grid_launch_dependents();
}

// Rows longer than that: dx by rows, then the sums over tokens by columns (a block takes 32 columns and a share of the rows).
template <typename T, typename P, int VEC>
__global__ void __launch_bounds__(1024) layer_norm_grad_long_kernel(const __grid_constant__ NormGradParams p) {
  __shared__ float2 sums[32];
  grid_dependency_wait();
  const long long row = blockIdx.x;
  const P* w = reinterpret_cast<const P*>(p.weight);
  const T *x = reinterpret_cast<const T*>(p.x) + row * p.ldx, *g = reinterpret_cast<const T*>(p.g) + row * p.ldg;
  const float mean = p.stats[row], rstd = p.stats[p.rows + row];
  float s1 = 0.0f, s2 = 0.0f;
  for (int i = threadIdx.x * VEC; i < p.cols; i += 1024 * VEC) {
    Pack<T, VEC> xv, gv;
    Pack<P, VEC> wv;
    xv.load(x + i);
    gv.load(g + i);
    if (w != nullptr) wv.load(w + i);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float gw = to_float(gv.e[e]) * (w != nullptr ? to_float(wv.e[e]) : 1.0f);
      s1 += gw;
      s2 = fmaf(gw, (to_float(xv.e[e]) - mean) * rstd, s2);
    }
  }
  const float2 both = block_sum2(s1, s2, sums);
  const float n = (float)p.cols, m1 = both.x / n, m2 = both.y / n;
  T* dx = reinterpret_cast<T*>(p.dx) + row * p.lddx;
  for (int i = threadIdx.x * VEC; i < p.cols; i += 1024 * VEC) {
    Pack<T, VEC> xv, gv, o;
    Pack<P, VEC> wv;
    xv.load(x + i);
    gv.load(g + i);
    if (w != nullptr) wv.load(w + i);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float gw = to_float(gv.e[e]) * (w != nullptr ? to_float(wv.e[e]) : 1.0f);
      o.e[e] = from_float<T>(rstd * (gw - m1 - (to_float(xv.e[e]) - mean) * rstd * m2));
    }
    o.store(dx + i);
  }
  grid_launch_dependents();
}
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(const __grid_constant__ NormGradParams p) {
  __shared__ float part[2][8][32];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float dw = 0.0f, db = 0.0f;
  if (c < p.cols)
    for (long long row = (long long)blockIdx.y * 8 + warp; row < p.rows; row += (long long)gridDim.y * 8) {
      const float g = to_float(reinterpret_cast<const T*>(p.g)[row * p.ldg + c]);
      const float x = to_float(reinterpret_cast<const T*>(p.x)[row * p.ldx + c]);
      dw = fmaf(g, (x - p.stats[row]) * p.stats[p.rows + row], dw);
      db += g;
    }
  part[0][warp][lane] = dw;
  part[1][warp][lane] = db;
  __syncthreads();
  if (warp < 2 && c < p.cols) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += part[warp][k][lane];
    p.partials[((size_t)blockIdx.y * 2 + warp) * (size_t)p.cols + c] = s;
  }
  grid_launch_dependents();
}

// The blocks' partial sums [blocks][2][cols], added in block order: 32 columns and eight strands of blocks per block.
template <typename P>
__global__ void __launch_bounds__(256) layer_norm_sums_kernel(const float* partials, int blocks, int cols, P* dweight, P* dbias) {
  __shared__ float part[8][32];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float s = 0.0f;
  if (c < cols)
#pragma unroll 8
    for (int k = warp; k < blocks; k += 8) s += partials[((size_t)k * 2 + which) * (size_t)cols + c];
  part[warp][lane] = s;
  __syncthreads();
  grid_launch_dependents();
  P* out = which == 0 ? dweight : dbias;
  if (warp == 0 && c < cols && out != nullptr) {
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += part[k][lane];
    out[c] = from_float<P>(s);
  }
}

constexpr int kMaxColumns = 16;   // columns of a thread in the fused backward kernel

// Threads that take a row of `pieces` pieces, nv each.
int row_threads(long long pieces, int nv) {
  const long long t = (pieces + nv - 1) / nv;
  return (int)((t + 31) / 32 * 32);
}
template <typename T, typename P, int VEC>
cudaError_t forward(const NormParams& p, int sms, cudaStream_t st) {
  const long long pieces = ((long long)p.cols + VEC - 1) / VEC;
  const bool few = p.rows <= 2ll * sms;   // rows that do not fill the machine: a piece per thread, so that the row's chain is short
  if (pieces <= 32 && !few)
    return launch_pdl(layer_norm_kernel<T, P, VEC, 1, true>, dim3((unsigned)((p.rows + kRowWarps - 1) / kRowWarps)), 32 * kRowWarps, 0, st, p);
  if (pieces <= 128 && !few)
    return launch_pdl(layer_norm_kernel<T, P, VEC, 4, true>, dim3((unsigned)((p.rows + kRowWarps - 1) / kRowWarps)), 32 * kRowWarps, 0, st, p);
  const dim3 grid((unsigned)p.rows);
  if (few && pieces <= 1024) return launch_pdl(layer_norm_kernel<T, P, VEC, 1, false>, grid, row_threads(pieces, 1), 0, st, p);
  if (pieces <= 4096) return launch_pdl(layer_norm_kernel<T, P, VEC, 4, false>, grid, row_threads(pieces, 4), 0, st, p);
  if (VEC == 1 && pieces <= 16384) return launch_pdl(layer_norm_kernel<T, P, VEC, (VEC == 1 ? 16 : 4), false>, grid, row_threads(pieces, 16), 0, st, p);
  return launch_pdl(layer_norm_long_kernel<T, P, VEC>, grid, 1024, 0, st, p);
}

int fused_blocks(long long rows, int threads, int sms) {
  const int per_sm = threads >= 1024 ? 1 : (1024 / threads < 16 ? 1024 / threads : 16);
  const long long most = (long long)sms * per_sm;
  return (int)(rows < most ? rows : most);
}
constexpr int kColumnBlocks = 64;   // shares of the rows in the backward pass of long rows

template <typename T, typename P, int VEC, int NV>
cudaError_t fused_backward(const NormGradParams& p, int threads, int blocks, cudaStream_t st) {
  return launch_pdl(layer_norm_grad_kernel<T, P, VEC, NV>, dim3((unsigned)blocks), threads, 0, st, p);
}
template <typename T, typename P, int VEC>
cudaError_t backward(const NormGradParams& p, int sms, P* dweight, P* dbias, cudaStream_t st) {
  const long long pieces = ((long long)p.cols + VEC - 1) / VEC;
  constexpr int MOST = VEC == 1 ? 8 : kMaxColumns / VEC;   // pieces of a thread
  cudaError_t rc = cudaSuccess;
  int blocks = 0;
  if (pieces <= 1024ll * MOST) {
    const int nv = pieces <= 1024 ? 1 : (pieces <= 2048 && MOST >= 2 ? 2 : (pieces <= 4096 && MOST >= 4 ? 4 : MOST));
    const int threads = row_threads(pieces, nv);
    blocks = fused_blocks(p.rows, threads, sms);
    if (p.rows > 0) {
      if (nv == 1) rc = fused_backward<T, P, VEC, 1>(p, threads, blocks, st);
      else if (nv == 2) rc = fused_backward<T, P, VEC, (MOST >= 2 ? 2 : 1)>(p, threads, blocks, st);
      else if (nv == 4) rc = fused_backward<T, P, VEC, (MOST >= 4 ? 4 : 1)>(p, threads, blocks, st);
      else rc = fused_backward<T, P, VEC, MOST>(p, threads, blocks, st);
    }
  } else {
    blocks = (int)((p.rows + 7) / 8 < kColumnBlocks ? (p.rows + 7) / 8 : kColumnBlocks);
    if (p.rows > 0 && p.dx != nullptr) rc = launch_pdl(layer_norm_grad_long_kernel<T, P, VEC>, dim3((unsigned)p.rows), 1024, 0, st, p);
    if (rc == cudaSuccess && p.rows > 0 && p.partials != nullptr)
      rc = launch_pdl(layer_norm_columns_kernel<T>, dim3((unsigned)((p.cols + 31) / 32), (unsigned)blocks), 256, 0, st, p);
  }
  if (rc == cudaSuccess && p.partials != nullptr)
    rc = launch_pdl(layer_norm_sums_kernel<P>, dim3((unsigned)((p.cols + 31) / 32), 2), 256, 0, st, p.partials, blocks, p.cols, dweight, dbias);
  return rc;
}

constexpr int kMostFeatures = 1 << 30;   // (column indexes are ints that step past the end)
size_t elem_size(int elem) { return elem == VOID_ELEM_F32 ? 4 : 2; }
bool aligned(const void* p, long long ld, int elem) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * (long long)elem_size(elem)) % 16 == 0;
}

}  // namespace

}  // namespace vb

// One instantiation per type of the tokens, type of the parameters and width of the accesses.
#define VB_NORM_TYPES(CALL)                                                                                          \
  (elem == VOID_ELEM_F32 ? CALL(float, float)                                                                         \
   : elem == VOID_ELEM_F16 ? (param_elem == VOID_ELEM_F16 ? CALL(__half, __half) : CALL(__half, float))               \
                           : (param_elem == VOID_ELEM_BF16 ? CALL(__nv_bfloat16, __nv_bfloat16) : CALL(__nv_bfloat16, float)))

extern "C" {

int void_layer_norm(const void* x, int32_t elem, int64_t ldx, int64_t rows, int32_t cols, const void* weight, const void* bias,
                    int32_t param_elem, float eps, void* y, int64_t ldy, float* stats, void_stream_t stream) {
  using namespace vb;
  if (elem < VOID_ELEM_F32 || elem > VOID_ELEM_BF16 || (param_elem != elem && param_elem != VOID_ELEM_F32)) return VOID_ERR_BAD_ARG;
  if (rows < 0 || cols <= 0 || ldx < cols || ldy < cols || !(eps >= 0.0f)) return VOID_ERR_BAD_ARG;
  if (rows > 0x7fffffffll || cols > kMostFeatures) return VOID_ERR_TOO_LARGE;
  if (rows == 0) return VOID_OK;
  if (x == nullptr || y == nullptr) return VOID_ERR_BAD_ARG;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  const NormParams p = {x, weight, bias, y, stats, ldx, ldy, rows, cols, eps};
  const bool wide = cols % (elem == VOID_ELEM_F32 ? 4 : 8) == 0 && aligned(x, ldx, elem) && aligned(y, ldy, elem) && aligned(weight, 0, param_elem) &&
                    aligned(bias, 0, param_elem);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define VB_CALL(T, P) (wide ? forward<T, P, 16 / (int)sizeof(T)>(p, dev.sms, st) : forward<T, P, 1>(p, dev.sms, st))
  return status_of(VB_NORM_TYPES(VB_CALL));
#undef VB_CALL
}

size_t void_layer_norm_grad_ws_bytes(int64_t rows, int32_t cols) {
  using namespace vb;
  if (rows <= 0 || cols <= 0) return 0;
  const DeviceInfo dev = device_info();
  const long long most = 16ll * (dev.ok ? dev.sms : 148);
  return (size_t)(rows < most ? rows : most) * 2 * (size_t)cols * sizeof(float);
}

int void_layer_norm_grad(const void* g, int64_t ldg, const void* x, int64_t ldx, int32_t elem, int64_t rows, int32_t cols,
                         const void* weight, int32_t param_elem, const float* stats, void* dx, int64_t lddx, void* dweight,
                         void* dbias, void* ws, size_t ws_bytes, void_stream_t stream) {
  using namespace vb;
  if (elem < VOID_ELEM_F32 || elem > VOID_ELEM_BF16 || (param_elem != elem && param_elem != VOID_ELEM_F32)) return VOID_ERR_BAD_ARG;
  if (rows < 0 || cols <= 0 || ldg < cols || ldx < cols || (dx != nullptr && lddx < cols)) return VOID_ERR_BAD_ARG;
  if (rows > 0x7fffffffll || cols > kMostFeatures) return VOID_ERR_TOO_LARGE;
  if (rows > 0 && (g == nullptr || x == nullptr || stats == nullptr)) return VOID_ERR_BAD_ARG;
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (!sums && (dx == nullptr || rows == 0)) return VOID_OK;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  if (sums && rows > 0 && (ws == nullptr || ws_bytes < void_layer_norm_grad_ws_bytes(rows, cols))) return VOID_ERR_WORKSPACE;
  float* partials = sums ? reinterpret_cast<float*>(rows > 0 ? ws : dweight) : nullptr;   // (no rows: not read)
  if (partials == nullptr && sums) partials = reinterpret_cast<float*>(dbias);
  const NormGradParams p = {g, x, weight, stats, dx, partials, ldg, ldx, lddx, rows, cols};
  const bool wide = cols % (elem == VOID_ELEM_F32 ? 4 : 8) == 0 && aligned(g, ldg, elem) && aligned(x, ldx, elem) &&
                    (dx == nullptr || aligned(dx, lddx, elem)) && aligned(weight, 0, param_elem);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define VB_CALL(T, P)                                                                                                                  \
  (wide ? backward<T, P, 16 / (int)sizeof(T)>(p, dev.sms, reinterpret_cast<P*>(dweight), reinterpret_cast<P*>(dbias), st)             \
        : backward<T, P, 1>(p, dev.sms, reinterpret_cast<P*>(dweight), reinterpret_cast<P*>(dbias), st))
  return status_of(VB_NORM_TYPES(VB_CALL));
#undef VB_CALL
}

}  // extern "C"
