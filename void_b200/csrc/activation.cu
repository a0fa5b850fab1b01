// Backward pass of a linear layer's activation:  dz = g act'(z), and the column sums of dz, the bias's gradient, in the same pass.
//
// Memory bounds it: two matrices in, one out, 3 N M elements.  A block takes a share of the rows of a slab of columns; a thread keeps
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

// act'(z) of two values, of GELU and SiLU.  With s = sigmoid(w(z)): (z s)' = s + z s (1 - s) w'(z).
__device__ __forceinline__ f32x2 slopes(f32x2 z, int act) {
  float a, b;
  unpair(z, a, b);
  // (kGelu1, kGelu3 and kSilu carry -log2(e), for a sigmoid of powers of two)
  const bool gelu = act == VOID_ACT_GELU;
  const f32x2 square = mul2(z, z), one = pair(1.0f, 1.0f);
  const f32x2 w = mul2(z, gelu ? fma2(square, pair(kGelu3, kGelu3), pair(kGelu1, kGelu1)) : pair(kSilu, kSilu));
  constexpr float back = -1.0f / (float)kLog2e;
  const f32x2 inner = gelu ? fma2(square, pair(3.0f * kGelu3 * back, 3.0f * kGelu3 * back), pair(kGelu1 * back, kGelu1 * back)) : one;
  unpair(w, a, b);
  const float s0 = sigmoid_exp2(a), s1 = sigmoid_exp2(b);
  const f32x2 s = pair(s0, s1), rest = mul2(s, fma2(s, pair(-1.0f, -1.0f), one));
  float r0, r1;
  unpair(fma2(mul2(z, rest), inner, s), a, b);
  unpair(rest, r0, r1);
  // (far out s is 0 or 1 to the last bit while z grows: nothing is left of the second term)
  return pair(r0 > 0.0f ? a : s0, r1 > 0.0f ? b : s1);
}
// d act'(z).  Where ReLU has no slope nothing comes through, an infinite gradient no more than others.
__device__ __forceinline__ f32x2 through(f32x2 d, f32x2 z, int act) {
  if (act != VOID_ACT_RELU) return mul2(d, slopes(z, act));
  float a, b, da, db;
  unpair(z, a, b);
  unpair(d, da, db);
  return pair(a > 0.0f ? da : 0.0f, b > 0.0f ? db : 0.0f);
}

template <typename T> __device__ __forceinline__ float value(T v);
template <> __device__ __forceinline__ float value<float>(float v) { return v; }
template <> __device__ __forceinline__ float value<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float value<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr int kGradThreads = 256, kGradWarps = kGradThreads / 32, kRing = 4;
constexpr int kMostRows = 128 * 65535;

// (own pieces only: a thread's own wait is all that a copy needs before its use)
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

struct ActivationGradParams {
  const void *g, *z;
  void* dz;
  float* partials;   // [row blocks][cols], or null
  long long ldg, ldz, lddz;
  int rows, cols, act;
  int block_rows;    // rows of a block
};
struct RunsOfTokens {   // experts: a block takes a chunk of one expert's tokens (experts.cu)
  const int32_t* head;
  const int32_t* chunk_ptr;
  const int4* chunks;
};
struct NoRuns {};
template <bool RUNS>
using RunsIf = std::conditional_t<RUNS, RunsOfTokens, NoRuns>;

// VEC: elements of a 16-byte piece of rows that lie on such boundaries (the next rows' pieces are on their way to shared memory), else 1.
// 4096 x 4096 bf16, GELU: rows loaded four at a time into registers 28 us, 23 instructions per element; this way 21 (with the sums).
template <typename T, int VEC, bool RUNS>
__global__ void __launch_bounds__(kGradThreads, 4) activation_grad_kernel(const __grid_constant__ ActivationGradParams p, const __grid_constant__ RunsIf<RUNS> runs) {
  constexpr bool WIDE = VEC > 1;
  __shared__ float part[kGradWarps][32 * VEC];
  __shared__ __align__(16) uint8_t ring[WIDE ? kRing * 2 * kGradThreads * 16 : 16];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = (blockIdx.x * 32 + lane) * VEC;
  int r0 = blockIdx.y * p.block_rows, r1 = r0 + p.block_rows < p.rows ? r0 + p.block_rows : p.rows;
  if constexpr (RUNS) {
    if ((int)blockIdx.y >= runs.head[0]) return;
    const int4 c = runs.chunks[blockIdx.y];
    r0 = c.y;
    r1 = c.z;
  }
  const bool active = p.act != VOID_ACT_NONE;
  constexpr int PAIRS = WIDE ? VEC / 2 : 1;
  f32x2 s[PAIRS];
#pragma unroll
  for (int e = 0; e < PAIRS; ++e) s[e] = pair(0.0f, 0.0f);
  if (c0 < p.cols) {
    const T *g = reinterpret_cast<const T*>(p.g) + (long long)(r0 + warp) * p.ldg + c0, *z = reinterpret_cast<const T*>(p.z) + (long long)(r0 + warp) * p.ldz + c0;
    T* dz = reinterpret_cast<T*>(p.dz) + (long long)(r0 + warp) * p.lddz + c0;
    const long long g_step = kGradWarps * p.ldg, z_step = kGradWarps * p.ldz, dz_step = kGradWarps * p.lddz;
    int left = r1 - r0 > warp ? (r1 - r0 - warp + kGradWarps - 1) / kGradWarps : 0;
    if constexpr (WIDE) {
      const uint32_t mine = smem_u32(ring) + threadIdx.x * 16u;   // slot k: g at mine + 2 k THREADS 16, z behind it
      int asked = left;
      auto fetch = [&](int slot) {
        if (asked-- > 0) {
          const uint32_t to = mine + (uint32_t)slot * (2u * kGradThreads * 16u);
          copy_async(to, g);
          if (active) copy_async(to + kGradThreads * 16u, z);
        }
        copies_commit();
        g += g_step;
        z += z_step;
      };
#pragma unroll
      for (int k = 0; k < kRing - 1; ++k) fetch(k);
      for (int slot = 0; left > 0; --left, dz += dz_step, slot = (slot + 1) % kRing) {
        fetch((slot + kRing - 1) % kRing);
        copies_wait<kRing - 1>();
        union { uint32_t w[4]; T e[VEC]; } gv, zv;
        const uint32_t at = mine + (uint32_t)slot * (2u * kGradThreads * 16u);
        ld_shared_v4(at, gv.w);
        if (active) ld_shared_v4(at + kGradThreads * 16u, zv.w);
        f32x2 d[PAIRS];
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {
          d[e] = pair(value<T>(gv.e[2 * e]), value<T>(gv.e[2 * e + 1]));
          if (active) d[e] = through(d[e], pair(value<T>(zv.e[2 * e]), value<T>(zv.e[2 * e + 1])), p.act);
          s[e] = add2(s[e], d[e]);
        }
        if (p.dz == nullptr) continue;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int e = 0; e < PAIRS; ++e) zv.w[e] = half2_bits<std::is_same<T, __half>::value>(d[e]);
        } else {
#pragma unroll
          for (int e = 0; e < PAIRS; ++e) {
            float a, b;
            unpair(d[e], a, b);
            zv.w[2 * e] = __float_as_uint(a);
            zv.w[2 * e + 1] = __float_as_uint(b);
          }
        }
        *reinterpret_cast<uint4*>(dz) = make_uint4(zv.w[0], zv.w[1], zv.w[2], zv.w[3]);
      }
    } else {
      // two rows at a time, in a pair
      for (; left > 0; left -= 2, g += 2 * g_step, z += 2 * z_step, dz += 2 * dz_step) {
        const bool two = left > 1;
        f32x2 d = pair(value<T>(g[0]), two ? value<T>(g[g_step]) : 0.0f);
        if (active) d = through(d, pair(value<T>(z[0]), two ? value<T>(z[z_step]) : 0.0f), p.act);
        s[0] = add2(s[0], d);
        float a, b;
        unpair(d, a, b);
        if (p.dz != nullptr) {
          dz[0] = rounded<T>(a);
          if (two) dz[dz_step] = rounded<T>(b);
        }
      }
    }
  }
  grid_launch_dependents();
  if (p.partials == nullptr) return;
#pragma unroll
  for (int e = 0; e < PAIRS; ++e) {
    float a, b;
    unpair(s[e], a, b);
    if (WIDE) {
      part[warp][lane * VEC + 2 * e] = a;
      part[warp][lane * VEC + (2 * e + 1) % VEC] = b;
    } else {
      part[warp][lane] = a + b;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += kGradThreads) {
    const int c = blockIdx.x * 32 * VEC + i;
    if (c >= p.cols) continue;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kGradWarps; ++w) sum += part[w][i];
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

// Values of z that lie next to ReLU's border, computed again.  The slope there is a question of z's sign, and the tensor cores cut what they hold
// after every product that they add, by half of 2^-23 of it: of 45 million sums of rows of 3 to 107 tiles none was off by more than 3.2 times
// (tiles + 16) 2^-23 of what is typical of its token, the square of the mean root of |sum| over a strip of up to 256 columns (which one large value hardly
// moves).  The border is eight times that, and as many times four for the bias, which a sum that it cancels has grown to.  What lies inside, or is -0 (with_bias),
// is summed in 64 bits: of normal values one in sixty thousand for rows of 13 tiles, at most kMostDoubtful of a block's 8192 whatever the values are; those
// beyond, the last of the block, keep the sign they were summed to.  The order is that of tokens and columns: the same result every time.
// (What fp16 would round to zero has kept its sign, keep_sign.)  One value is summed by the block, eight of them by a warp each.
// us, forward pass with SiLU and with ReLU and this behind it, fp16, bias and residual: 4096^2, 90 %, 4096 tokens 63 and 87; 2048^2, 50 %, 512 tokens 14
// and 23; 14336 -> 14240, 76 %, 44 tokens 76 and 96 (mostly the way to the tiles of one or two values per block); 16 experts of 2048 -> 4096, 90 %, 8192 tokens bf16 82 and
// 121.  One output in 32 a thousand times the others, or one bias of each strip 3e4: 4 to 9 us more (a border relative to the strip's largest value: 25 ms).
__device__ __forceinline__ float sqrt_approx(float v) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr int kStrip = 256, kBorderWarps = 8, kBorderTokens = 4, kMostDoubtful = 256;   // columns of a block, its warps, tokens of a warp at a time
struct BorderParams {
  const void *x, *values, *bias;
  const int32_t *row_ptr, *block_indices, *tile_cols, *bounds;
  void* z;
  long long ldx, ldz;
  int N, M, K, nbr, n_experts, bias_dtype;
};
template <typename T>
__global__ void __launch_bounds__(32 * kBorderWarps) relu_border_kernel(const __grid_constant__ BorderParams p) {
  constexpr int BATCH = kBorderWarps * kBorderTokens;
  __shared__ uint16_t list[kMostDoubtful];   // (token of the batch) << 8 | column of the strip
  __shared__ int counts[kBorderWarps];
  __shared__ double sums[kBorderWarps];
  grid_dependency_wait();
  // strips of whole pieces of eight columns, none much narrower than the others: it would say little about what is typical
  const long long pieces = (p.M + 7) >> 3;
  const int strip = (int)(pieces * blockIdx.x / gridDim.x) * 8, strip_end = (int)(pieces * (blockIdx.x + 1) / gridDim.x) * 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m0 = strip + lane * 8;
  const int cols = m0 >= strip_end ? 0 : (p.M - m0 < 8 ? p.M - m0 : 8);
  int run_begin = 0, run_end = p.N, run = 0;   // of the token asked for last: tokens of its run, expert (-1: in no run)
  if (p.bounds != nullptr) run_end = 0;
  auto expert_of = [&](int n) {
    if (n >= run_begin && n < run_end) return run;
    const int before = p.bounds[0], behind = p.bounds[p.n_experts];
    if (n < before || n >= behind) {
      run = -1;
      run_begin = n < before ? 0 : behind;
      run_end = n < before ? before : p.N;
      return run;
    }
    int e = 0, hi = p.n_experts;   // the last whose run does not begin behind the token
    while (hi - e > 1) {
      const int mid = (e + hi) >> 1;
      if (p.bounds[mid] <= n) e = mid;
      else hi = mid;
    }
    run = e;
    run_begin = p.bounds[e];
    run_end = p.bounds[e + 1];
    return run;
  };
  auto bias_at = [&](size_t at) {
    return p.bias_dtype == VOID_OUT_F32 ? reinterpret_cast<const float*>(p.bias)[at]
                                        : f16_value(reinterpret_cast<const uint16_t*>(p.bias)[at], p.bias_dtype == VOID_OUT_F16);
  };
  // of the lane's columns, for the expert that the token belongs to: 2^-21 (tiles + 16); the biases, NaN (no comparison holds) where there are no tiles
  int held = -1;
  float unit = 0.0f, each = 0.0f, bias[8];
  auto take = [&](int e) {
    if (e < 0 || e == held) return;
    held = e;
    const int32_t* row = p.row_ptr + (size_t)e * p.nbr + (m0 >> 5);
    const int tiles = cols > 0 ? row[1] - row[0] : 0;
    unit = (float)(tiles + 16) * (1.0f / 2097152.0f);
    const int all = __reduce_add_sync(0xffffffffu, tiles > 0 ? cols : 0);
    each = all > 0 ? 1.0f / (float)all : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      bias[i] = tiles > 0 && i < cols ? (p.bias != nullptr ? bias_at((size_t)e * p.M + m0 + i) : 0.0f) : __int_as_float(0x7fffffff);
  };
  for (long long first = (long long)blockIdx.y * BATCH; first < p.N; first += (long long)gridDim.y * BATCH) {
    union { uint4 v; T t[8]; uint16_t bits[8]; } u[kBorderTokens];
#pragma unroll
    for (int k = 0; k < kBorderTokens; ++k) {
      const long long n = first + warp * kBorderTokens + k;
      u[k].v = make_uint4(0u, 0u, 0u, 0u);
      if (cols > 0 && n < p.N) u[k].v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.z) + n * p.ldz + m0);
    }
    uint32_t doubtful = 0u;   // bit 8 k + i: column i of token k
#pragma unroll
    for (int k = 0; k < kBorderTokens; ++k) {
      const long long n = first + warp * kBorderTokens + k;
      const int e = n < p.N ? expert_of((int)n) : -1;
      take(e);
      if (e < 0) continue;
      float root = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = fabsf(value<T>(u[k].t[i]) - bias[i]);
        if (s < 1e30f) root += sqrt_approx(s);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) root += __shfl_xor_sync(0xffffffffu, root, o);
      root *= each;
      const float typical = unit * 2.0f * root * root;
#pragma unroll
      for (int i = 0; i < 8; ++i)   // (of the zeros only -0)
        if (fabsf(value<T>(u[k].t[i])) < fmaf(unit, fabsf(bias[i]), typical) && u[k].bits[i] != 0) doubtful |= 1u << (8 * k + i);
    }
    if (!__syncthreads_or(doubtful != 0u)) continue;
    int place[kBorderTokens], found = 0;   // in the warp's part of the list: token by token
#pragma unroll
    for (int k = 0; k < kBorderTokens; ++k) {
      const int mine = __popc((doubtful >> (8 * k)) & 255u);
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int before = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += before;
      }
      place[k] = found + upto - mine;
      found += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) counts[warp] = found;
    __syncthreads();
    int base = 0, count = 0;
#pragma unroll
    for (int w = 0; w < kBorderWarps; ++w) {
      if (w < warp) base += counts[w];
      count += counts[w];
    }
    if (count > kMostDoubtful) count = kMostDoubtful;
#pragma unroll
    for (int k = 0; k < kBorderTokens; ++k)
      for (uint32_t bits = (doubtful >> (8 * k)) & 255u, at = (uint32_t)(base + place[k]); bits != 0u; bits &= bits - 1u, ++at)
        if (at < (uint32_t)kMostDoubtful) list[at] = (uint16_t)((warp * kBorderTokens + k) << 8 | (lane * 8 + __ffs(bits) - 1));
    __syncthreads();
    for (int c = 0, share; c < count; c += kBorderWarps / share) {
      const int left = count - c;
      share = left >= 8 ? 1 : (left >= 4 ? 2 : (left >= 2 ? 4 : 8));   // warps of a value, which take its tiles in turn
      const int v = list[c + warp / share], part = warp % share;
      const int n = (int)(first + (v >> 8)), m = strip + (v & 255), e = expert_of(n);
      const int32_t* row = p.row_ptr + (size_t)e * p.nbr + (m >> 5);
      const T *x = reinterpret_cast<const T*>(p.x) + (long long)n * p.ldx, *values = reinterpret_cast<const T*>(p.values) + (m & 31) * 32 + lane;
      double s = 0.0;
      const int end = row[1];
      for (int t = row[0] + part; t < end; t += 4 * share) {
        float a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = t + i * share < end;
          const int k = in ? p.tile_cols[t + i * share] * 32 + lane : p.K;
          a[i] = in ? value<T>(values[(size_t)p.block_indices[t + i * share] * 1024]) : 0.0f;
          b[i] = k < p.K ? value<T>(x[k]) : 0.0f;
          if (k >= p.K) a[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s += (double)a[i] * (double)b[i];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (share > 1) {
        if (lane == 0) sums[warp] = s;
        __syncthreads();
      }
      if (part == 0 && lane == 0) {
        for (int w = 1; w < share; ++w) s += sums[warp + w];
        if (p.bias != nullptr) s += (double)bias_at((size_t)e * p.M + m);
        union { uint16_t bits; T t; } r;
        r.t = rounded<T>((float)s);
        if (s != 0.0 && (r.bits & 0x7fffu) == 0) r.bits = s > 0.0 ? 0x0001u : 0x8001u;   // (the sign is what is asked for)
        reinterpret_cast<T*>(p.z)[(long long)n * p.ldz + m] = r.t;
      }
      if (share > 1) __syncthreads();
    }
    __syncthreads();   // (the list is read to its end before a warp writes the next)
  }
  grid_launch_dependents();
}

// Rows of a block: as many blocks as the SMs hold, or of a few rows per warp.
int rows_per_block(int rows, int cols) {
  const DeviceInfo dev = device_info();
  const int slabs = (cols + 255) / 256, most = 4 * (dev.ok ? dev.sms : 148) / slabs;
  const int even = (rows + (most > 0 ? most : 1) - 1) / (most > 0 ? most : 1), least = 4 * kGradWarps;
  return even > least ? even : least;
}
int row_blocks(int rows, int cols) { return (rows + rows_per_block(rows, cols) - 1) / rows_per_block(rows, cols); }

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
  return rows <= 0 || cols <= 0 ? 0 : (size_t)vb::row_blocks(rows, cols) * (size_t)cols * sizeof(float);
}

int void_activation_grad(const void* g, int64_t ldg, const void* z, int64_t ldz, int32_t elem, int32_t rows, int32_t cols, int32_t act,
                         void* dz, int64_t lddz, void* dbias, int32_t bias_elem, void* ws, size_t ws_bytes, void_stream_t stream) {
  using namespace vb;
  if (elem < VOID_ELEM_F32 || elem > VOID_ELEM_BF16 || rows < 0 || cols < 0 || act < VOID_ACT_NONE || act > VOID_ACT_SILU) return VOID_ERR_BAD_ARG;
  if (ldg < cols || ldz < cols || lddz < cols) return VOID_ERR_BAD_ARG;
  if (dbias != nullptr && bias_elem != elem && bias_elem != VOID_ELEM_F32) return VOID_ERR_BAD_ARG;
  if (cols == 0 || (rows == 0 && dbias == nullptr)) return VOID_OK;
  if (rows > 0 && (g == nullptr || z == nullptr || dz == nullptr)) return VOID_ERR_BAD_ARG;
  if (rows > kMostRows) return VOID_ERR_TOO_LARGE;
  if (dbias != nullptr && rows > 0 && (ws == nullptr || ws_bytes < void_activation_grad_ws_bytes(rows, cols))) return VOID_ERR_WORKSPACE;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  const ActivationGradParams p = {g, z, dz, dbias != nullptr ? reinterpret_cast<float*>(ws) : nullptr, ldg, ldz, lddz, rows, cols, act, rows_per_block(rows, cols)};
  return activation_grad<false>(p, NoRuns{}, row_blocks(rows, cols), 1, elem, dbias, bias_elem, reinterpret_cast<cudaStream_t>(stream));
}

int void_relu_border(const void* x, int64_t ldx, const void* values, const int32_t* row_ptr, const int32_t* block_indices, const int32_t* tile_cols,
                     int32_t M, int32_t K, int32_t N, int32_t kind, const void* bias, int32_t bias_dtype, void* z, int64_t ldz, const void_experts* experts,
                     void_stream_t stream) {
  using namespace vb;
  if (kind != VOID_KIND_F16 && kind != VOID_KIND_BF16) return VOID_ERR_BAD_ARG;
  if (M < 0 || K < 0 || N < 0 || ldx < K || ldz < M || bias_dtype < VOID_OUT_F32 || bias_dtype > VOID_OUT_BF16) return VOID_ERR_BAD_ARG;
  if (experts != nullptr && (experts->plan == nullptr || experts->offset_bytes != 0 || experts->n_experts < 1)) return VOID_ERR_BAD_ARG;
  if (M == 0 || N == 0 || K == 0) return VOID_OK;
  if (x == nullptr || values == nullptr || row_ptr == nullptr || block_indices == nullptr || tile_cols == nullptr || z == nullptr) return VOID_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(z) & 15u) != 0 || ldz % 8 != 0) return VOID_ERR_ALIGN;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  const BorderParams p = {x, values, bias, row_ptr, block_indices, tile_cols, experts != nullptr ? plan_of(*experts, N).bounds : nullptr, z, ldx, ldz,
                          N, M, K, (M + 31) / 32, experts != nullptr ? experts->n_experts : 0, bias_dtype};
  const int turns = (N + kBorderWarps * kBorderTokens - 1) / (kBorderWarps * kBorderTokens);
  const dim3 grid((unsigned)((M + kStrip - 1) / kStrip), (unsigned)(turns < 65535 ? turns : 65535));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return status_of(kind == VOID_KIND_F16 ? launch_pdl(relu_border_kernel<__half>, grid, 32 * kBorderWarps, 0, st, p)
                                         : launch_pdl(relu_border_kernel<__nv_bfloat16>, grid, 32 * kBorderWarps, 0, st, p));
}

size_t void_expert_activation_grad_ws_bytes(const void_experts* x, int32_t rows, int32_t cols) {
  if (x == nullptr || x->n_experts < 1 || x->chunk < 1 || rows <= 0 || cols <= 0) return 0;
  return (size_t)vb::plan_capacity(x->n_experts, rows, x->chunk) * (size_t)cols * sizeof(float);
}

int void_expert_activation_grad(const void* g, int64_t ldg, const void* z, int64_t ldz, int32_t elem, const void_experts* x, int32_t rows,
                                int32_t cols, int32_t act, void* dz, int64_t lddz, void* dbias, int32_t bias_elem, void* ws, size_t ws_bytes,
                                void_stream_t stream) {
  using namespace vb;
  if (x == nullptr || x->plan == nullptr || x->offset_bytes != 0 || x->n_experts < 1 || x->chunk < 1) return VOID_ERR_BAD_ARG;
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
  const ActivationGradParams p = {g, z, dz, dbias != nullptr ? reinterpret_cast<float*>(ws) : nullptr, ldg, ldz, lddz, rows, cols, act, 0};
  const RunsOfTokens runs = {v.head, v.chunk_ptr, v.chunks};
  return activation_grad<true>(p, runs, v.capacity, x->n_experts, elem, dbias, bias_elem, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
