// Layer norm over the features of each token, forward and backward:
//
//     xh = (x - mean) / sqrt(var + eps)          y = xh w + b                       per token, D features
//     gw = g w       dx = rstd (gw - mean(gw) - xh mean(gw xh))       dw = sum over tokens of g xh       db = sum over tokens of g
//
// Memory bounds both: 2 D elements per token forward (x, y), 3 D backward (g, x, dx).  On B200, of 6.5 TB/s of copies: 16384 x 4096 bf16 5.3
// TB/s forward (51 us) and 4.9 backward (82 us with the sums over tokens), 8192 x 8192 6.0 and 4.7, 3001 x 5003 fp32 4.5 and 4.1; a row per block,
// 2048 x 4096 bf16 2.9 and 1.8.  A token's row stays in registers between its
// reductions, so it comes in once; the variance is the mean square of the centred values (two passes over registers: no
// cancellation for rows with a large mean).  All sums are fp32.  Backward, the block walks many rows and a thread keeps the same
// columns throughout, so the sums over tokens stay in its registers; they leave as one row of partial sums per block, which a second
// kernel adds in block order: no atomics, the result does not depend on which block ran when.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

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
// Sum over the block; `s` has a word per warp and is free again behind the block's next barrier but one (callers alternate).  Few warps'
// sums are added by every thread for itself: broadcast reads, which do not wait for one another as the steps of a shuffle do.
__device__ __forceinline__ float block_sum(float v, float* s) {
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  v = warp_sum(v);
  if (lane == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (warps > 8) return warp_sum(lane < warps ? s[lane] : 0.0f);
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w)
    if (w < warps) v += s[w];
  return v;
}

constexpr int kRowWarps = 4;   // rows of a block whose warps take a row each

struct NormParams {
  const void *x, *weight, *bias;
  void* y;
  float* stats;   // [2][rows]: mean, rstd; or null
  long long ldx, ldy, rows;
  int cols;
  float eps;
  uint32_t slot_bytes;   // of a row in shared memory
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

// ------------------------------------------------------------------------------------------ many rows
// With enough rows to go round, blocks stay and walk the rows; the next rows are on their way to shared memory meanwhile (asynchronous
// copies, S - 1 rows ahead), and the parameters of a thread's columns stay in its registers.  Rows in whole 16-byte pieces: a thread
// copies and reads its own pieces only, so nothing but its own wait stands between a copy and its use.  Other rows start anywhere
// in such a piece; they come in the pieces they lie in (the first of which begins in the row before), a barrier later every thread reads
// its columns, element by element.
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, uint32_t bytes) {   // (of 16; the rest is zeroed)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// A row that starts anywhere, to shared memory; it then begins row_offset(row) bytes behind dst.
__device__ __forceinline__ uint32_t row_offset(const void* row) { return (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u); }
__device__ __forceinline__ void copy_row(uint32_t dst, const void* row, uint32_t bytes) {
  const uint32_t off = row_offset(row), end = off + bytes;
  const uint8_t* from = static_cast<const uint8_t*>(row) - off;
  for (uint32_t at = threadIdx.x * 16u; at < end; at += blockDim.x * 16u) copy_async(dst + at, from + at, end - at < 16u ? end - at : 16u);
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
// A thread's piece of shared memory.
template <typename T, int E>
struct Piece {
  static_assert(E == 1 || sizeof(T) * E == 16, "an element or 16 bytes");
  static constexpr int BYTES = (int)sizeof(T) * E, WORDS = (BYTES + 3) / 4;
  union { T e[E]; uint32_t w[WORDS]; };
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < WORDS; ++k) w[k] = 0u;
  }
  __device__ __forceinline__ void load_shared(uint32_t at) {
    if constexpr (BYTES == 16) {
      ld_shared_v4(at, *reinterpret_cast<uint32_t(*)[4]>(&w));
    } else if constexpr (BYTES == 4) {
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
    } else {
      uint16_t h;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at) : "memory");
      w[0] = h;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (BYTES == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (BYTES == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *p = e[0];
  }
  // elements i and i + 1
  __device__ __forceinline__ void set2(int i, float a, float b) {
    if constexpr (sizeof(T) == 4) { e[i] = from_float<T>(a); e[i + 1] = from_float<T>(b); }
    else if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i / 2]) : "f"(b), "f"(a));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i / 2]) : "f"(b), "f"(a));
  }
  __device__ __forceinline__ Piece() {}
};
// A thread's parameters: E of them from an index that is a multiple of E and inside; `absent` where there are none.
template <typename P, int E>
struct Params {
  Pack<P, E> v;
  __device__ __forceinline__ void load(const P* p, int i, int cols, float absent) {
#pragma unroll
    for (int e = 0; e < E; ++e) v.e[e] = from_float<P>(absent);
    if (p != nullptr && i < cols) v.load(p + i);
  }
  __device__ __forceinline__ float operator[](int e) const { return to_float(v.e[e]); }
};

// C: elements of a thread, in pieces of E; S: rows in shared memory; MOST: threads at most.  What bounds such a kernel beside memory is
// the number of its instructions (the two sums over a block take a hundred per warp and row whatever a thread has of the row), so a thread
// takes many elements and computes in pairs.  16384 x 4096 bf16, eight elements per thread and single operations: 72 us;
// parameters read for every row again: 72 us with fp32 ones, 60 with bf16; this way 51, at 0.67 instructions per clock and scheduler.
template <typename T, typename P, int E, int C, int S, int MOST>
__global__ void __launch_bounds__(MOST, MOST <= 256 ? (C > 16 ? 2 : 3) : (MOST <= 384 ? 2 : 1)) layer_norm_rows_kernel(const __grid_constant__ NormParams p) {
  constexpr int PIECE = (int)sizeof(T) * E, NV = C / E;
  constexpr bool WHOLE = PIECE == 16;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float4 joins[2][MOST / 32];
  grid_dependency_wait();
  const int t = threadIdx.x, step = blockDim.x, lane = t & 31, warps = step >> 5;
  // piece k of this thread in slot s: mine + s slot_bytes + k pitch (and the row's own offset)
  const uint32_t mine = smem_u32(ring) + (uint32_t)(t * PIECE), pitch = (uint32_t)(step * PIECE), slot_bytes = p.slot_bytes;
  const long long x_step = (long long)gridDim.x * p.ldx, y_step = (long long)gridDim.x * p.ldy;
  const T *x = reinterpret_cast<const T*>(p.x) + (long long)blockIdx.x * p.ldx, *ahead = x;
  int left = (int)((p.rows - blockIdx.x + gridDim.x - 1) / gridDim.x), asked = left;   // rows of this block, and those not yet asked for
  auto fetch = [&](int slot) {
    if (asked > 0) {
      if constexpr (WHOLE) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if ((t + k * step) * E < p.cols) copy_async(mine + (uint32_t)slot * slot_bytes + (uint32_t)k * pitch, ahead + (t + k * step) * E);
      } else {
        copy_row(smem_u32(ring) + (uint32_t)slot * slot_bytes, ahead, (uint32_t)(p.cols * (int)sizeof(T)));
      }
    }
    copies_commit();
    --asked;
    ahead += x_step;
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);
  Params<P, E> w[NV], bias[NV];
  int count = 0;   // elements of this thread, then of its warp
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    w[k].load(reinterpret_cast<const P*>(p.weight), (t + k * step) * E, p.cols, 1.0f);
    bias[k].load(reinterpret_cast<const P*>(p.bias), (t + k * step) * E, p.cols, 0.0f);
    if ((t + k * step) * E < p.cols) count += E;
  }
  const float of_warp = warp_sum((float)count), each_of_warp = of_warp > 0.0f ? 1.0f / of_warp : 0.0f, each = 1.0f / (float)p.cols;
  T* y = reinterpret_cast<T*>(p.y) + (long long)blockIdx.x * p.ldy + t * E;
  int slot = 0, turn = 0;
  long long row = blockIdx.x;
  for (; left > 0; --left, row += gridDim.x, x += x_step, y += y_step, turn ^= 1) {
    uint32_t at = mine + (uint32_t)slot * slot_bytes;
    if constexpr (WHOLE) {
      fetch(slot == 0 ? S - 1 : slot - 1);
      copies_wait<S - 1>();
    } else {
      copies_wait<S - 2>();
      __syncthreads();   // (the row is there for all threads, and none still reads the slot that is asked for next)
      fetch(slot == 0 ? S - 1 : slot - 1);
      at += row_offset(x);
    }
    f32x2 v[C / 2], s = pair(0.0f, 0.0f);
    float f[C], a, b;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      Piece<T, E> u;
      u.zero();
      if ((t + k * step) * E < p.cols) u.load_shared(at + (uint32_t)k * pitch);
#pragma unroll
      for (int e = 0; e < E; ++e) f[k * E + e] = to_float(u.e[e]);
    }
#pragma unroll
    for (int c = 0; c < C / 2; ++c) {
      v[c] = pair(f[2 * c], f[2 * c + 1]);
      s = add2(s, v[c]);
    }
    // mean and sum of squares about it, of the warp; then those of the block from the warps' (each square about its own mean, and the
    // means' distance from the common one: no differences of large sums)
    unpair(s, a, b);
    const float m = warp_sum(a + b) * each_of_warp;
    s = pair(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < C / 2; ++c) {
      const f32x2 d = add2(v[c], pair(-m, -m));
      if (E > 1) {
        if ((t + 2 * c / E * step) * E < p.cols) s = fma2(d, d, s);
      } else {
        unpair(d, a, b);
        s = fma2(d, pair(t + 2 * c * step < p.cols ? a : 0.0f, t + (2 * c + 1) * step < p.cols ? b : 0.0f), s);
      }
    }
    unpair(s, a, b);
    const float squares = warp_sum(a + b);
    if (lane == 0) joins[turn][t >> 5] = make_float4(m, of_warp, squares, 0.0f);
    __syncthreads();
    float mean = 0.0f, var = 0.0f;
    if (MOST <= 256) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < warps) {
          const float2 j = *reinterpret_cast<const float2*>(&joins[turn][i]);
          mean = fmaf(j.x, j.y, mean);
        }
      mean *= each;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < warps) {
          const float4 j = joins[turn][i];
          const float d = j.x - mean;
          var += fmaf(d * d, j.y, j.z);
        }
    } else {
      const float4 j = lane < warps ? joins[turn][lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      mean = warp_sum(j.x * j.y) * each;
      const float d = j.x - mean;
      var = warp_sum(fmaf(d * d, j.y, j.z));
    }
    const float rstd = 1.0f / sqrtf(var * each + p.eps);
    if (p.stats != nullptr && t == 0) {
      p.stats[row] = mean;
      p.stats[p.rows + row] = rstd;
    }
    const f32x2 shift = pair(-mean, -mean), scale = pair(rstd, rstd);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if ((t + k * step) * E >= p.cols) continue;
      Piece<T, E> o;
      if constexpr (E > 1) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          unpair(fma2(mul2(add2(v[(k * E + e) / 2], shift), scale), pair(w[k][e], w[k][e + 1]), pair(bias[k][e], bias[k][e + 1])), a, b);
          o.set2(e, a, b);
        }
      } else {
        o.e[0] = from_float<T>(fmaf((f[k] - mean) * rstd, w[k][0], bias[k][0]));
      }
      o.store(y + k * step * E);
    }
    slot = slot == S - 1 ? 0 : slot + 1;
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
  uint32_t slot_bytes;   // of a row in shared memory
};

// One barrier per row: both sums meet in it, in one of two places in turn.
__device__ __forceinline__ float2 block_sum2(float a, float b, float2* s) {
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  a = warp_sum(a);
  b = warp_sum(b);
  if (lane == 0) s[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 v = make_float2(0.0f, 0.0f);
  if (warps > 8) {
    if (lane < warps) v = s[lane];
    return make_float2(warp_sum(v.x), warp_sum(v.y));
  }
#pragma unroll
  for (int w = 0; w < 8; ++w)
    if (w < warps) {
      const float2 u = s[w];
      v.x += u.x;
      v.y += u.y;
    }
  return v;
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

// The same with rows on their way through shared memory, as layer_norm_rows_kernel has them: x and g of a row side by side.  In rows of
// up to 8192 elements a thread keeps its values between the row's sums and its result; in longer ones they are read again from there.
template <typename T, typename P, int E, int C, int S, int MOST>
__global__ void __launch_bounds__(MOST, MOST <= 256 ? 2 : 1) layer_norm_grad_rows_kernel(const __grid_constant__ NormGradParams p) {
  constexpr bool KEPT = C <= 16;   // whether a row's values stay in registers between its sums and its result
  constexpr int PIECE = (int)sizeof(T) * E, NV = C / E;
  constexpr bool WHOLE = PIECE == 16;
  constexpr int Q = E > 1 ? E / 2 : 1, R = 2 * Q / E, CHUNKS = C / (2 * Q);   // a chunk: Q pairs of R pieces
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float2 sums[2][32];
  grid_dependency_wait();
  const int t = threadIdx.x, step = blockDim.x;
  // a slot holds a row of x and then one of g
  const uint32_t mine = smem_u32(ring) + (uint32_t)(t * PIECE), pitch = (uint32_t)(step * PIECE), row_bytes = p.slot_bytes, slot_bytes = 2u * row_bytes;
  const T *x = reinterpret_cast<const T*>(p.x) + (long long)blockIdx.x * p.ldx, *g_row = reinterpret_cast<const T*>(p.g) + (long long)blockIdx.x * p.ldg;
  const T *ahead_x = x, *ahead_g = g_row;
  const long long x_step = (long long)gridDim.x * p.ldx, g_step = (long long)gridDim.x * p.ldg, dx_step = (long long)gridDim.x * p.lddx;
  int left = (int)((p.rows - blockIdx.x + gridDim.x - 1) / gridDim.x), asked = left;
  auto fetch = [&](int slot) {
    if (asked > 0) {
      const uint32_t to = (uint32_t)slot * slot_bytes;
      if constexpr (WHOLE) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if ((t + k * step) * E < p.cols) {
            copy_async(mine + to + (uint32_t)k * pitch, ahead_x + (t + k * step) * E);
            copy_async(mine + to + row_bytes + (uint32_t)k * pitch, ahead_g + (t + k * step) * E);
          }
      } else {
        copy_row(smem_u32(ring) + to, ahead_x, (uint32_t)(p.cols * (int)sizeof(T)));
        copy_row(smem_u32(ring) + to + row_bytes, ahead_g, (uint32_t)(p.cols * (int)sizeof(T)));
      }
    }
    copies_commit();
    --asked;
    ahead_x += x_step;
    ahead_g += g_step;
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);
  f32x2 dw[CHUNKS][Q], db[CHUNKS][Q];
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
    for (int q = 0; q < Q; ++q) dw[k][q] = db[k][q] = pair(0.0f, 0.0f);
  const float each = 1.0f / (float)p.cols;
  Params<P, E> w[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) w[k].load(reinterpret_cast<const P*>(p.weight), (t + k * step) * E, p.cols, 1.0f);
  int slot = 0, turn = 0;
  float mean = 0.0f, rstd = 0.0f;
  if (blockIdx.x < p.rows) {
    mean = p.stats[blockIdx.x];
    rstd = p.stats[p.rows + blockIdx.x];
  }
  // a chunk's gradients, unit values and weighted gradients; past the end of the row the gradients are zero, and so is what they bring
  auto chunk = [&](uint32_t at, uint32_t at_g, int c, float scale, float shift, f32x2 (&g)[Q], f32x2 (&xh)[Q], f32x2 (&gw)[Q]) {
    float gf[2 * Q], xf[2 * Q];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = c * R + r;
      Piece<T, E> xv, gv;
      xv.zero();
      gv.zero();
      if ((t + k * step) * E < p.cols) {
        xv.load_shared(at + (uint32_t)k * pitch);
        gv.load_shared(at_g + (uint32_t)k * pitch);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        gf[r * E + e] = to_float(gv.e[e]);
        xf[r * E + e] = to_float(xv.e[e]);
      }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      g[q] = pair(gf[2 * q], gf[2 * q + 1]);
      xh[q] = mul2(add2(pair(xf[2 * q], xf[2 * q + 1]), pair(shift, shift)), pair(scale, scale));
      gw[q] = mul2(g[q], pair(w[c * R + 2 * q / E][2 * q % E], w[c * R + (2 * q + 1) / E][(2 * q + 1) % E]));
    }
  };
  T* dx = reinterpret_cast<T*>(p.dx) + (long long)blockIdx.x * p.lddx + t * E;
  const float* stats = p.stats + blockIdx.x;
  for (; left > 0; --left, turn ^= 1, dx += dx_step, x += x_step, g_row += g_step) {
    uint32_t at = mine + (uint32_t)slot * slot_bytes, at_g = at + row_bytes;
    if constexpr (WHOLE) {
      fetch(slot == 0 ? S - 1 : slot - 1);
      copies_wait<S - 1>();
    } else {
      copies_wait<S - 2>();
      __syncthreads();
      fetch(slot == 0 ? S - 1 : slot - 1);
      at += row_offset(x);
      at_g += row_offset(g_row);
    }
    const float shift = -mean, scale = rstd;
    if (left > 1) {
      stats += gridDim.x;
      mean = stats[0];
      rstd = stats[p.rows];
    }
    f32x2 s1 = pair(0.0f, 0.0f), s2 = s1, g[Q], xh[KEPT ? CHUNKS : 1][Q], gw[KEPT ? CHUNKS : 1][Q];
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
      const int r = KEPT ? k : 0;
      chunk(at, at_g, k, scale, shift, g, xh[r], gw[r]);
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        dw[k][q] = fma2(g[q], xh[r][q], dw[k][q]);
        db[k][q] = add2(db[k][q], g[q]);
        s1 = add2(s1, gw[r][q]);
        s2 = fma2(gw[r][q], xh[r][q], s2);
      }
    }
    if (p.dx != nullptr) {
      float a, b, c, d;
      unpair(s1, a, b);
      unpair(s2, c, d);
      const float2 both = block_sum2(a + b, c + d, sums[turn]);
      // dx = rstd gw - rstd m1 - xh (rstd m2)
      const f32x2 m1 = pair(-both.x * each * scale, -both.x * each * scale), m2 = pair(-both.y * each * scale, -both.y * each * scale);
#pragma unroll
      for (int k = 0; k < CHUNKS; ++k) {
        const int r = KEPT ? k : 0;
        if (!KEPT) chunk(at, at_g, k, scale, shift, g, xh[r], gw[r]);
        Piece<T, E> o[R];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          unpair(fma2(xh[r][q], m2, fma2(gw[r][q], pair(scale, scale), m1)), a, b);
          if constexpr (E > 1) {
            o[0].set2(2 * q, a, b);
          } else {
            o[0].e[0] = from_float<T>(a);
            o[R - 1].e[0] = from_float<T>(b);
          }
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
          if ((t + (k * R + i) * step) * E < p.cols) o[i].store(dx + (k * R + i) * step * E);
      }
    }
    slot = slot == S - 1 ? 0 : slot + 1;
  }
  if (p.partials != nullptr) {
    float* out = p.partials + (size_t)blockIdx.x * 2 * (size_t)p.cols;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        float v[2], u[2];
        unpair(dw[k][q], v[0], v[1]);
        unpair(db[k][q], u[0], u[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = 2 * q + h, i = (t + (k * R + c / E) * step) * E + c % E;
          if (i < p.cols) {
            out[i] = v[h];
            out[(size_t)p.cols + i] = u[h];
          }
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
constexpr int kColumns = 16;   // elements of a thread in the kernels for many rows, or twice that
// Whether rows that are not in whole 16-byte pieces can be taken from such pieces all the same: the first row has to start on one, what
// lies before another row's first element in its piece is then the tensor's, too.
bool starts_on_piece(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool through_ring(long long rows, int cols, int sms) { return rows > 2ll * sms && cols > 64 * kColumns && cols <= 1024 * kColumns; }
// (forward a block has to walk a few rows before it gains on blocks of one row each: 4096 bf16, 2048 rows 9.8 and 9.2 us, 16384 rows 52 and
// 68; 5003 fp32, 3001 rows 33 and 46)
int forward_blocks_per_sm(int cols) { return cols <= 256 * kColumns ? 768 * kColumns / cols : (cols <= 512 * kColumns ? 2 : 1); }
// Blocks of a launch that fills the SMs: what registers (per_sm of them) and shared memory leave room for.
int resident_blocks(const DeviceInfo& dev, long long rows, int smem, int per_sm) {
  const int fit = (dev.smem_per_sm - 4096) / (smem + 2048);
  if (per_sm > fit) per_sm = fit;
  if (per_sm < 1) per_sm = 1;
  const long long most = (long long)dev.sms * per_sm;
  return (int)(rows < most ? rows : most);
}
template <typename T, int E, int C>
uint32_t ring_slot(int cols, int threads) {
  return sizeof(T) * E == 16 ? (uint32_t)(threads * C * (int)sizeof(T)) : (uint32_t)((cols * (int)sizeof(T) + 15 + 15) / 16 * 16);
}
template <typename T, typename P, int E, int C, int MOST>
cudaError_t forward_rows(NormParams p, const DeviceInfo& dev, cudaStream_t st) {
  constexpr int S = sizeof(T) == 4 && MOST > 256 ? 3 : 4;
  auto kernel = layer_norm_rows_kernel<T, P, E, C, S, MOST>;
  const int threads = row_threads((p.cols + E - 1) / E, C / E);
  p.slot_bytes = ring_slot<T, E, C>(p.cols, threads);
  const int smem = S * (int)p.slot_bytes;
  if (ensure_smem((const void*)kernel, smem)) return cudaErrorInvalidValue;
  const int per_sm = threads <= 256 ? (C > kColumns ? 512 : 768) / threads : (MOST <= 384 ? 2 : 1);
  return launch_pdl(kernel, dim3((unsigned)resident_blocks(dev, p.rows, smem, per_sm)), threads, smem, st, p);
}
// Rows of up to 4096 elements in threads of 16, longer ones in threads of 32 (bf16, GB/s: 4096 5190 and 5060, 8192 4390 and 4770, 16384
// 3890 and 5290).  Element by element it is a little better to keep 16 as long as two blocks fit an SM (fp32, 5003 elements, 3001 rows 28.4 and
// 26.4 us, 8000 rows 68.3 and 63.9).
template <typename T, typename P, int E>
cudaError_t forward_rows(const NormParams& p, const DeviceInfo& dev, cudaStream_t st) {
  if constexpr (E == 1)
    if (p.cols > 256 * kColumns && p.cols <= 384 * kColumns) return forward_rows<T, P, E, kColumns, 384>(p, dev, st);
  if (p.cols <= 256 * kColumns) return forward_rows<T, P, E, kColumns, 256>(p, dev, st);
  return p.cols <= 512 * kColumns ? forward_rows<T, P, E, 2 * kColumns, 256>(p, dev, st) : forward_rows<T, P, E, 2 * kColumns, 512>(p, dev, st);
}

template <typename T, typename P, int VEC>
cudaError_t forward(const NormParams& p, const DeviceInfo& dev, cudaStream_t st) {
  const int sms = dev.sms;
  const long long pieces = ((long long)p.cols + VEC - 1) / VEC;
  const bool few = p.rows <= 2ll * sms;   // rows that do not fill the machine: a piece per thread, so that the row's chain is short
  if ((VEC > 1 || starts_on_piece(p.x)) && through_ring(p.rows, p.cols, sms) && p.rows >= 6ll * sms * forward_blocks_per_sm(p.cols))
    return forward_rows<T, P, VEC>(p, dev, st);
  if (pieces <= 32 && !few)
    return launch_pdl(layer_norm_kernel<T, P, VEC, 1, true>, dim3((unsigned)((p.rows + kRowWarps - 1) / kRowWarps)), 32 * kRowWarps, 0, st, p);
  if (VEC == 1 && pieces > 128 && pieces <= 512 && !few)
    return launch_pdl(layer_norm_kernel<T, P, VEC, 16 / VEC, true>, dim3((unsigned)((p.rows + kRowWarps - 1) / kRowWarps)), 32 * kRowWarps, 0, st, p);
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
// (rows of up to 32 KB: three of them with their gradients fit an SM)
template <typename T, typename P, int E, int C, int MOST>
cudaError_t backward_rows(NormGradParams p, const DeviceInfo& dev, int* blocks, cudaStream_t st) {
  constexpr int S = C > kColumns || (sizeof(T) == 4 && MOST == 512) ? 3 : 4;
  auto kernel = layer_norm_grad_rows_kernel<T, P, E, C, S, MOST>;
  const int threads = row_threads((p.cols + E - 1) / E, C / E);
  p.slot_bytes = ring_slot<T, E, C>(p.cols, threads);
  const int smem = 2 * S * (int)p.slot_bytes;
  if (ensure_smem((const void*)kernel, smem)) return cudaErrorInvalidValue;
  *blocks = resident_blocks(dev, p.rows, smem, threads <= 256 ? 512 / threads : 1);
  return launch_pdl(kernel, dim3((unsigned)*blocks), threads, smem, st, p);
}
template <typename T, typename P, int E>
cudaError_t backward_rows(const NormGradParams& p, const DeviceInfo& dev, int* blocks, cudaStream_t st) {
  if (p.cols <= 256 * kColumns) return backward_rows<T, P, E, kColumns, 256>(p, dev, blocks, st);
  return p.cols <= 512 * kColumns ? backward_rows<T, P, E, kColumns, 512>(p, dev, blocks, st) : backward_rows<T, P, E, 2 * kColumns, 512>(p, dev, blocks, st);
}
template <typename T, typename P, int VEC>
cudaError_t backward(const NormGradParams& p, const DeviceInfo& dev, P* dweight, P* dbias, cudaStream_t st) {
  const int sms = dev.sms;
  const long long pieces = ((long long)p.cols + VEC - 1) / VEC;
  constexpr int MOST = VEC == 1 ? 8 : kMaxColumns / VEC;   // pieces of a thread
  cudaError_t rc = cudaSuccess;
  int blocks = 0;
  if ((VEC > 1 || (starts_on_piece(p.x) && starts_on_piece(p.g))) && through_ring(p.rows, p.cols, sms) && p.cols * (long long)sizeof(T) <= 32 * 1024) {
    rc = backward_rows<T, P, VEC>(p, dev, &blocks, st);
  } else if (pieces <= 1024ll * MOST) {
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
    // (the sums first: dx may take the place of g or x)
    if (p.rows > 0 && p.partials != nullptr)
      rc = launch_pdl(layer_norm_columns_kernel<T>, dim3((unsigned)((p.cols + 31) / 32), (unsigned)blocks), 256, 0, st, p);
    if (rc == cudaSuccess && p.rows > 0 && p.dx != nullptr) rc = launch_pdl(layer_norm_grad_long_kernel<T, P, VEC>, dim3((unsigned)p.rows), 1024, 0, st, p);
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
  const NormParams p = {x, weight, bias, y, stats, ldx, ldy, rows, cols, eps, 0u};
  const bool wide = cols % (elem == VOID_ELEM_F32 ? 4 : 8) == 0 && aligned(x, ldx, elem) && aligned(y, ldy, elem) && aligned(weight, 0, param_elem) &&
                    aligned(bias, 0, param_elem);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define VB_CALL(T, P) (wide ? forward<T, P, 16 / (int)sizeof(T)>(p, dev, st) : forward<T, P, 1>(p, dev, st))
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
  const NormGradParams p = {g, x, weight, stats, dx, partials, ldg, ldx, lddx, rows, cols, 0u};
  const bool wide = cols % (elem == VOID_ELEM_F32 ? 4 : 8) == 0 && aligned(g, ldg, elem) && aligned(x, ldx, elem) &&
                    (dx == nullptr || aligned(dx, lddx, elem)) && aligned(weight, 0, param_elem);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define VB_CALL(T, P)                                                                                                                  \
  (wide ? backward<T, P, 16 / (int)sizeof(T)>(p, dev, reinterpret_cast<P*>(dweight), reinterpret_cast<P*>(dbias), st)             \
        : backward<T, P, 1>(p, dev, reinterpret_cast<P*>(dweight), reinterpret_cast<P*>(dbias), st))
  return status_of(VB_NORM_TYPES(VB_CALL));
#undef VB_CALL
}

}  // extern "C"
