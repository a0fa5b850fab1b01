// Linear layers whose weights are dense e4m3 matrices with a scale for each block of 128 x 128, on tokens in e4m3 with a scale for each
// token's 128 features:
//
//     out[t, m] = act( sum_b sx[t, b] sa[m / 128, b] sum_{k in block b} x[t, k] a[m, k]  + bias[m] ) + residual[t, m]
//
// of one matrix, or of the matrices of experts for tokens sorted by expert.  The scales differ from block to block of k, so every block's product is
// an accumulator of its own, which eight warps read back, multiply by sx sa and add in registers, while the tensor cores fill the other of two.
//
// Up to 64 tokens (of experts: up to 48 or 24 on average, by the size of their matrices) the product is computed transposed (fp8_block_kernel): 128 features are the lanes of tensor memory and
// the tokens its columns, in sixteens, so a short run costs what its tokens cost and the weights stream once; sx sa is one number per column.  More
// tokens (fp8_wide_kernel) are the lanes, 128 of them, and 256 features the columns, so that sx sa is one number of a thread's own.
//
// With fewer work items than SMs, the blocks of k are dealt to a cluster of CTAs, whose partial sums meet through shared memory, added in the
// order of the CTAs.
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <stdint.h>
#include <string.h>

#include "../../include/void_b200.h"
#include "epilogue.cuh"
#include "experts.cuh"
#include "kinds.cuh"
#include "launch.cuh"
#include "pipeline.cuh"
#include "ptx.cuh"
#include "values.cuh"

namespace vb {

namespace {

constexpr int kBlock = 128;          // features of a block, and of a work item
constexpr int kTokenBox = 32;        // tokens that one copy brings
constexpr unsigned kEvery = 0xffffffffu;

// ------------------------------------------------------------------------------------------ quantisers
struct QuantParams {
  const void* x;
  long long ldx, ldq, scale_row, scale_col;
  long long rows;
  int cols;
  uint8_t* q;
  float* scales;
};
// The smallest power of two that keeps numbers up to `amax` within e4m3's 448 = 1.75 * 2^8, and its reciprocal: no rounding but that to
// e4m3 itself.  bits: of amax, so that NaN is larger than all; a block that holds one, or an infinity, gets a scale of NaN.
__device__ __forceinline__ float block_scale(uint32_t bits, float& inverse) {
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < -100 ? -100 : e;
  inverse = __int_as_float((127 - e) << 23);
  if (bits >= 0x7f800000u) {
    inverse = 0.0f;
    return __int_as_float(0x7fc00000);
  }
  return __int_as_float((127 + e) << 23);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

constexpr int kQuantThreads = 256;

// The largest magnitude of 16-bit numbers as their bits, two at a time (NaN above infinity above all others).
__device__ __forceinline__ uint32_t magnitudes(uint32_t pair16) { return pair16 & 0x7fff7fffu; }
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <typename T>
__device__ __forceinline__ uint32_t bits_of_half(uint32_t h);   // of the fp32 number that a 16-bit magnitude stands for
template <>
__device__ __forceinline__ uint32_t bits_of_half<__nv_bfloat16>(uint32_t h) { return h << 16; }
template <>
__device__ __forceinline__ uint32_t bits_of_half<__half>(uint32_t h) { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h))) & 0x7fffffffu; }

// A scale per row and 128 columns.  Rows in 16-byte pieces: 128 columns lie in 16 lanes (fp32: 32), a warp has `HELD` groups of 512 bytes of a
// row at a time on their way; others element by element.  blockIdx.y: part of the columns.  8192 x 8192 bf16: 35 us, 5.7 TB/s (fp32 maxima and a division for
// every piece's place: 57).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kQuantThreads) quant_rows_kernel(const __grid_constant__ QuantParams p) {
  constexpr int VEC = WIDE ? 16 / (int)sizeof(T) : 4, HELD = WIDE ? 4 : 2;
  constexpr int LANES = kBlock / VEC;   // of a block of 128 columns: 16 or 32
  constexpr int STEP = 32 * VEC;
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, c0 = (int)blockIdx.y * (STEP * HELD);
  for (long long row = (long long)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5); row < p.rows; row += (long long)gridDim.x * (kQuantThreads / 32)) {
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
    uint8_t* q = p.q + row * p.ldq;
    float* scales = p.scales + row * p.scale_row;
    if constexpr (WIDE) {
      uint4 raw[HELD];
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        const int c = c0 + h * STEP + lane * VEC;
        raw[h] = c < p.cols ? *reinterpret_cast<const uint4*>(x + c) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        uint32_t most;
        if constexpr (VEC == 8) {
          most = max_halves(max_halves(magnitudes(raw[h].x), magnitudes(raw[h].y)), max_halves(magnitudes(raw[h].z), magnitudes(raw[h].w)));
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) most = max_halves(most, __shfl_xor_sync(kEvery, most, o));
          most = bits_of_half<T>(max(most & 0xffffu, most >> 16));
        } else {
          most = max(max(raw[h].x & 0x7fffffffu, raw[h].y & 0x7fffffffu), max(raw[h].z & 0x7fffffffu, raw[h].w & 0x7fffffffu));
          most = __reduce_max_sync(kEvery, most);
        }
        float inverse;
        const float scale = block_scale(most, inverse);
        const int c = c0 + h * STEP + lane * VEC;
        if (c < p.cols) {
          if (lane % LANES == 0) scales[(long long)(c / kBlock) * p.scale_col] = scale;
          Piece<T, VEC> piece;
          memcpy(piece.v, &raw[h], 16);
          uint32_t w[VEC / 4];
#pragma unroll
          for (int k = 0; k < VEC / 4; ++k)
            w[k] = e4m3x2(piece.get(4 * k) * inverse, piece.get(4 * k + 1) * inverse) | e4m3x2(piece.get(4 * k + 2) * inverse, piece.get(4 * k + 3) * inverse) << 16;
          if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q + c) = make_uint2(w[0], w[1]);
          else *reinterpret_cast<uint32_t*>(q + c) = w[0];
        }
      }
    } else {
      float v[HELD][VEC];
#pragma unroll
      for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int c = c0 + h * STEP + e * 32 + lane;
          v[h][e] = c < p.cols ? to_float<T>(x[c]) : 0.0f;
        }
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) most = max(most, magnitude(v[h][e]));
        most = __reduce_max_sync(kEvery, most);
        float inverse;
        const float scale = block_scale(most, inverse);
        const int first = c0 + h * STEP;
        if (first < p.cols && lane == 0) scales[(long long)(first / kBlock) * p.scale_col] = scale;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int c = first + e * 32 + lane;
          if (c < p.cols) q[c] = (uint8_t)e4m3x2(v[h][e] * inverse, 0.0f);
        }
      }
    }
  }
}

// A scale per 128 x 128, a block each (weights, once, so that it is simple: x twice, element by element).  8192 x 8192 bf16 125 us, where memory would take
// 31: waits for loads (12 of 19 cycles per instruction), 66.8 million instructions of warps.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quant_blocks_kernel(const __grid_constant__ QuantParams p) {
  __shared__ uint32_t most_of[kQuantThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const long long r0 = (long long)blockIdx.y * kBlock;
  const int c = blockIdx.x * kBlock + (threadIdx.x & 127);
  uint32_t most = 0;
  for (int r = threadIdx.x >> 7; r < kBlock; r += 2)
    if (r0 + r < p.rows && c < p.cols) most = max(most, magnitude(to_float<T>(reinterpret_cast<const T*>(p.x)[(r0 + r) * p.ldx + c])));
  most = __reduce_max_sync(kEvery, most);
  if ((threadIdx.x & 31) == 0) most_of[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQuantThreads / 32; ++w) most = max(most, most_of[w]);
  float inverse;
  const float scale = block_scale(most, inverse);
  if (threadIdx.x == 0) p.scales[(long long)blockIdx.y * p.scale_row + (long long)blockIdx.x * p.scale_col] = scale;
  for (int r = threadIdx.x >> 7; r < kBlock; r += 2)
    if (r0 + r < p.rows && c < p.cols)
      p.q[(r0 + r) * p.ldq + c] = (uint8_t)e4m3x2(to_float<T>(reinterpret_cast<const T*>(p.x)[(r0 + r) * p.ldx + c]) * inverse, 0.0f);
}

template <typename T>
int quant_of_type(const QuantParams& p, int block_rows, int sms, cudaStream_t st) {
  if (block_rows == kBlock) {
    const long long down = (p.rows + kBlock - 1) / kBlock;
    if (down > 65535) return VOID_ERR_TOO_LARGE;
    return status_of(launch_pdl(quant_blocks_kernel<T>, dim3((unsigned)((p.cols + kBlock - 1) / kBlock), (unsigned)down), kQuantThreads, 0, st, p));
  }
  constexpr int VEC = 16 / (int)sizeof(T);
  const bool wide = p.cols % VEC == 0 && ((reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)(p.ldx * sizeof(T))) & 15u) == 0 &&
                    ((reinterpret_cast<uintptr_t>(p.q) | (uintptr_t)p.ldq) & 7u) == 0;
  const int step = wide ? 32 * VEC * 4 : 32 * 4 * 2;
  const long long parts = (p.cols + (long long)step - 1) / step, blocks = (p.rows + kQuantThreads / 32 - 1) / (kQuantThreads / 32);
  if (parts > 65535) return VOID_ERR_TOO_LARGE;
  const dim3 grid((unsigned)(blocks < 0x7fffffffll ? blocks : 0x7fffffffll), (unsigned)parts);
  return status_of(wide ? launch_pdl(quant_rows_kernel<T, true>, grid, kQuantThreads, 0, st, p) : launch_pdl(quant_rows_kernel<T, false>, grid, kQuantThreads, 0, st, p));
}

// ------------------------------------------------------------------------------------------ products
constexpr int kThreads = 384;         // copies, products, scales (2), then eight warps that add up
constexpr int kAdders = 8, kFirstAdder = 4;
constexpr int kMaxRing = 12, kScaleSlots = 8;

struct Fp8Params {
  int M, K, N, k_blocks, m_tiles;
  int chunk, n_chunks, group;     // one matrix: tokens of an item, items along the tokens, and of them those taken together
  const int32_t *head, *bounds;   // experts: the plan of experts.cu
  const int4* chunks;
  const void* offsets;            // or, of up to 32 experts, the runs' offsets themselves
  int offset_bytes, n_experts, zero_rest;
  const float* a_scale;
  long long as_row, as_col, as_expert;
  const float* x_scale;
  long long xs_row, xs_col;
  const void* bias;
  int bias_elem;
  const void* residual;
  long long ldr;
  int residual_elem;
  void* out;
  long long ldc;
  int out_elem, act;
  int splits;                     // CTAs of a cluster, which share an item's blocks of k
  int stages;
  int32_t* status;
  int wait_limit_ms, drop_first;  // drop_first: test hook, the first stage is never filled
};
struct __align__(8) Fp8Bars {
  uint64_t full[kMaxRing], empty[kMaxRing];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t scale_full[kScaleSlots], scale_empty[kScaleSlots];
};
struct Item {
  int m, n0, n1, expert;
};
// The plan of up to 32 experts, which a warp makes for its CTA from the offsets (RunTable): a launch less.
struct Runs {
  int begin[32], end[32], first[32];   // tokens; chunks before the run's
  int total;                           // chunks in all
};
// Behind the wait on the kernel before; for all threads.
__device__ __forceinline__ void find_runs(const Fp8Params& p, Runs& runs) {
  if (p.offsets == nullptr) return;
  if (threadIdx.x < 32) {
    ExpertParams x = {};
    x.offsets = p.offsets;
    x.offset_bytes = p.offset_bytes;
    x.chunk = p.chunk;
    x.n_experts = p.n_experts;
    const RunTable table(x, p.N);
    runs.begin[threadIdx.x] = table.begin;
    runs.end[threadIdx.x] = table.end;
    runs.first[threadIdx.x] = table.first;
    if (threadIdx.x == 0) runs.total = table.total;
    if (blockIdx.x == 0 && table.bad && p.status != nullptr) atomicCAS(p.status, 0, kStatusBadOffsets);
  }
  __syncthreads();
}
__device__ __forceinline__ int items_of(const Fp8Params& p, const Runs& runs) {
  return (p.offsets != nullptr ? runs.total : (p.head != nullptr ? p.head[0] : p.n_chunks)) * p.m_tiles;
}
// Items that follow one another share tokens or weights: of one matrix, `group` chunks of tokens meet every piece of features.
__device__ __forceinline__ Item item_at(const Fp8Params& p, const Runs& runs, int i) {
  Item t;
  if (p.offsets != nullptr) {
    const int c = i / p.m_tiles;
    int e = 0;   // the last expert whose first chunk is not behind it
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (e + o < p.n_experts && runs.first[e + o] <= c) e += o;
    t.m = i - c * p.m_tiles;
    t.expert = e;
    t.n0 = runs.begin[e] + (c - runs.first[e]) * p.chunk;
    t.n1 = min(t.n0 + p.chunk, runs.end[e]);
    return t;
  }
  if (p.head != nullptr) {
    const int c = i / p.m_tiles;
    const int4 chunk = p.chunks[c];
    t.m = i - c * p.m_tiles;
    t.expert = chunk.x;
    t.n0 = chunk.y;
    t.n1 = chunk.z;
    return t;
  }
  const int per = p.group * p.m_tiles, g = i / per, first = g * p.group, wide = p.n_chunks - first < p.group ? p.n_chunks - first : p.group;
  const int rest = i - g * per;
  t.m = rest / wide;
  t.expert = 0;
  t.n0 = (first + rest - t.m * wide) * p.chunk;
  t.n1 = t.n0 + p.chunk < p.N ? t.n0 + p.chunk : p.N;
  return t;
}
__device__ __forceinline__ uint32_t cluster_address(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void store_result(const Fp8Params& p, long long token, int m, float v) {
  const long long at = token * p.ldc + m;
  if (p.out_elem == VOID_ELEM_F32) {
    reinterpret_cast<float*>(p.out)[at] = v;
  } else {
    const unsigned short h = p.out_elem == VOID_ELEM_F16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
    reinterpret_cast<unsigned short*>(p.out)[at] = h;
  }
}

// Zeros for tokens in no run.
__device__ __forceinline__ void zero_tokens_in_no_run(const Fp8Params& p, const Runs& runs) {
  if ((p.head == nullptr && p.offsets == nullptr) || !p.zero_rest) return;
  const int low = p.offsets != nullptr ? runs.begin[0] : p.bounds[0], high = p.offsets != nullptr ? runs.end[p.n_experts - 1] : p.bounds[p.n_experts];
  for (int r = (int)blockIdx.x; r < low + p.N - high; r += (int)gridDim.x) {
    const long long token = r < low ? r : high + r - low;
    for (int m = threadIdx.x; m < p.M; m += kThreads) store_result(p, token, m, 0.0f);
  }
}

// Few tokens: the weights are read once and that is all.  8 tokens, 8192 x 8192: 16.5 us (4.1 TB/s): 0.8 until the first copies are asked for, 2 to the first
// block, 12.5 of streaming, 2.5 for the sums of a cluster; 16384 x 16384: 48 (5.6 TB/s).  Weights asked for by prefetches ahead of the wait on the kernel
// before: 18.2 to 20.8 with the quantiser in front, against 18.5 without.
// NT: tokens of an item at most.
constexpr int kFewCtas = 2;   // of an SM
template <int NT>
__global__ void __launch_bounds__(kThreads, kFewCtas) fp8_block_kernel(const __grid_constant__ Fp8Params p, const __grid_constant__ CUtensorMap map_a,
                                                                       const __grid_constant__ CUtensorMap map_x) {
  static_assert(NT == 32 || NT == 64, "a warp reads 16 or 32 columns back at once");
  constexpr int CG = NT / 2;   // columns of an adding warp
  constexpr uint32_t kStageA = kBlock * kBlock, kStage = kStageA + NT * kBlock;
  constexpr uint32_t kTmem = NT * 2;
  extern __shared__ uint8_t raw[];
  __shared__ Fp8Bars bars;
  __shared__ __align__(16) float scale_ring[kScaleSlots][NT];
  __shared__ uint32_t tmem_s;
  __shared__ int ctl_s[2];
  __shared__ Runs runs;
  volatile int* ctl = ctl_s;
  const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    ctl_s[0] = 0;
    ctl_s[1] = p.wait_limit_ms;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&bars.full[s]), 1);
      mbar_init(smem_u32(&bars.empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&bars.acc_full[s]), 1);
      mbar_init(smem_u32(&bars.acc_empty[s]), kAdders);
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      mbar_init(smem_u32(&bars.scale_full[s]), 1);
      mbar_init(smem_u32(&bars.scale_empty[s]), kAdders);
    }
    fence_mbar_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_s), kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  const int rank = p.splits > 1 ? (int)cluster_rank() : 0;
  const int b0 = (int)((long long)p.k_blocks * rank / p.splits), b1 = (int)((long long)p.k_blocks * (rank + 1) / p.splits);
  grid_dependency_wait();
  find_runs(p, runs);
  const int step = (int)gridDim.x / p.splits, begin = (int)blockIdx.x / p.splits, end = items_of(p, runs);
  // With several CTAs per item a launch has a cluster for every item, so that the ring is free when the sums meet in its place.
  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool first = true;
    for (int i = begin; i < end && !ctl[0]; i += step) {
      const Item t = item_at(p, runs, i);
      const int boxes = (t.n1 - t.n0 + kTokenBox - 1) / kTokenBox;
      for (int b = b0; b < b1; ++b) {
        if (!mbar_wait_warp(smem_u32(&bars.empty[stage]), phase ^ 1u, ctl)) break;
        const bool drop = first && p.drop_first != 0;
        first = false;
        if (lane == 0 && !drop) {
          const uint32_t full = smem_u32(&bars.full[stage]);
          mbar_expect_tx(full, kStageA + (uint32_t)boxes * (kTokenBox * kBlock));
          tma_load_3d(ring + (uint32_t)stage * kStage, &map_a, b * kBlock, t.m * kBlock, t.expert, full);
        }
        __syncwarp();
        if (lane >= 1 && lane <= boxes && !drop)
          tma_load_2d(ring + (uint32_t)stage * kStage + kStageA + (uint32_t)(lane - 1) * (kTokenBox * kBlock), &map_x, b * kBlock, t.n0 + (lane - 1) * kTokenBox,
                      smem_u32(&bars.full[stage]));
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    constexpr uint64_t kDescHi = smem_desc_hi(16, 1024, kLayoutSw128);
    const bool leader = elect_one();
    int stage = 0;
    uint32_t phase = 0, it = 0;
    bool ok = true;
    for (int i = begin; i < end && ok; i += step) {
      const Item t = item_at(p, runs, i);
      const uint32_t idesc = instr_desc(1, 0, 0, 0, 0, 128, (uint32_t)(t.n1 - t.n0 + 15) & ~15u);
      for (int b = b0; b < b1; ++b, ++it) {
        const uint32_t slot = it & 1u;
        ok = mbar_wait_warp(smem_u32(&bars.acc_empty[slot]), ((it >> 1) & 1u) ^ 1u, ctl) && mbar_wait_warp(smem_u32(&bars.full[stage]), phase, ctl);
        if (!ok) break;
        tc_fence_after();
        const uint32_t at = ring + (uint32_t)stage * kStage;
        const uint64_t da = smem_desc(kDescHi, at), db = smem_desc(kDescHi, at + kStageA);
#pragma unroll
        for (int k = 0; k < 4; ++k)   // 32 features each: 32 bytes further in rows of 128
          issue_mma<VOID_KIND_F8E4M3>(leader, tmem + slot * NT, da + 2 * k, db + 2 * k, idesc, k > 0);
        tc_commit_if(leader, smem_u32(&bars.empty[stage]));
        tc_commit_if(leader, smem_u32(&bars.acc_full[slot]));
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp < kFirstAdder) {
    // The products of both scales, every other block of k for either warp; those of the next block are on their way meanwhile.
    constexpr int PER = NT / 32;
    uint32_t it0 = 0;
    bool ok = true;
    for (int i = begin; i < end && ok; i += step) {
      const Item t = item_at(p, runs, i);
      const float* sa = p.a_scale + t.expert * p.as_expert + t.m * p.as_row;
      const float* sx = p.x_scale + (long long)t.n0 * p.xs_row;
      float next[PER], next_a = 0.0f;
      auto fetch = [&](int b) {
        next_a = sa[b * p.as_col];
#pragma unroll
        for (int k = 0; k < PER; ++k) next[k] = t.n0 + lane + 32 * k < t.n1 ? sx[(lane + 32 * k) * p.xs_row + b * p.xs_col] : 0.0f;
      };
      // (block b is iteration it0 + b - b0 of the CTA)
      int b = b0 + (int)(((it0 & 1u) ^ (uint32_t)(warp - 2)) & 1u);
      if (b < b1) fetch(b);
      for (; b < b1; b += 2) {
        const uint32_t it = it0 + (uint32_t)(b - b0), slot = it % kScaleSlots;
        float now[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) now[k] = next[k] * next_a;
        if (b + 2 < b1) fetch(b + 2);
        ok = mbar_wait_warp(smem_u32(&bars.scale_empty[slot]), ((it / kScaleSlots) & 1u) ^ 1u, ctl);
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < PER; ++k) scale_ring[slot][lane + 32 * k] = now[k];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars.scale_full[slot]));
      }
      it0 += (uint32_t)(b1 - b0);
    }
  } else {
    const int quad = warp & 3, c0 = ((warp - kFirstAdder) >> 2) * CG;
    uint32_t it = 0;
    bool ok = true;
    for (int i = begin; i < end && ok; i += step) {
      const Item t = item_at(p, runs, i);
      const int n = t.n1 - t.n0, m = t.m * kBlock + quad * 32 + lane;
      const uint32_t bias_raw = p.bias != nullptr && m < p.M ? raw_element(p.bias, p.bias_elem, (long long)t.expert * p.M + m) : 0u;
      f32x2 sum[CG / 2];
#pragma unroll
      for (int c = 0; c < CG / 2; ++c) sum[c] = pair(0.0f, 0.0f);
      for (int b = b0; b < b1; ++b, ++it) {
        const uint32_t slot = it & 1u, ring_slot = it % kScaleSlots;
        ok = mbar_wait_warp(smem_u32(&bars.scale_full[ring_slot]), (it / kScaleSlots) & 1u, ctl) &&
             mbar_wait_warp(smem_u32(&bars.acc_full[slot]), (it >> 1) & 1u, ctl);
        if (!ok) break;
        tc_fence_after();
        if (c0 < n) {
          const uint32_t from = tmem + slot * NT + (uint32_t)c0 + ((uint32_t)(quad * 32) << 16);
          uint32_t r[CG];
          if constexpr (CG == 32) tmem_ld_32x32(from, r);
          else tmem_ld_32x16p(from, r);
          tmem_ld_wait();
          const float4* s4 = reinterpret_cast<const float4*>(&scale_ring[ring_slot][c0]);
#pragma unroll
          for (int c = 0; c < CG / 4; ++c) {
            const float4 s = s4[c];
            sum[2 * c] = fma2(pair(__uint_as_float(r[4 * c]), __uint_as_float(r[4 * c + 1])), pair(s.x, s.y), sum[2 * c]);
            sum[2 * c + 1] = fma2(pair(__uint_as_float(r[4 * c + 2]), __uint_as_float(r[4 * c + 3])), pair(s.z, s.w), sum[2 * c + 1]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&bars.acc_empty[slot]));
          mbar_arrive(smem_u32(&bars.scale_empty[ring_slot]));
        }
      }
      if (!ok) break;
      if (p.splits > 1) {
        float* part = reinterpret_cast<float*>(raw + (ring - smem_u32(raw)));   // [tokens][128]
#pragma unroll
        for (int c = 0; c < CG / 2; ++c) {
          float a, d;
          unpair(sum[c], a, d);
          if (c0 + 2 * c < n) part[(c0 + 2 * c) * kBlock + quad * 32 + lane] = a;
          if (c0 + 2 * c + 1 < n) part[(c0 + 2 * c + 1) * kBlock + quad * 32 + lane] = d;
        }
        break;   // (one item per cluster)
      }
      if (m < p.M && c0 < n) {
        const float bias = of_raw(bias_raw, p.bias_elem);
        f32x2 y[CG / 2];
#pragma unroll
        for (int c = 0; c < CG / 2; ++c) y[c] = add2(sum[c], pair(bias, bias));
        activate<CG / 2>(y, p.act);
        const long long token = t.n0 + c0;
#pragma unroll
        for (int h = 0; h < CG; h += 8) {   // eight residuals on their way together
          uint32_t res[8];
#pragma unroll
          for (int c = 0; c < 8; ++c)
            res[c] = p.residual != nullptr && c0 + h + c < n ? raw_element(p.residual, p.residual_elem, (token + h + c) * p.ldr + m) : 0u;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float a, d;
            unpair(y[(h + c) / 2], a, d);
            float v = c % 2 ? d : a;
            if (p.residual != nullptr) v += of_raw(res[c], p.residual_elem);
            if (c0 + h + c < n) store_result(p, token + h + c, m, v);
          }
        }
      }
      __syncwarp();
    }
  }
  if (p.splits > 1) {
    __syncwarp();
    cluster_meet();
    if (begin < end && warp >= kFirstAdder) {
      constexpr int HELD = 4;   // tokens whose sums and residuals are on their way together
      const Item t = item_at(p, runs, begin);
      const int n = t.n1 - t.n0, quad = warp & 3, side = (warp - kFirstAdder) >> 2, m = t.m * kBlock + quad * 32 + lane;
      const int share = (n + p.splits - 1) / p.splits, c1 = min(n, (rank + 1) * share);
      const uint32_t bias_raw = p.bias != nullptr && m < p.M ? raw_element(p.bias, p.bias_elem, (long long)t.expert * p.M + m) : 0u;
      for (int c0 = rank * share + side; c0 < c1; c0 += 2 * HELD) {
        uint32_t res[HELD];
        float v[HELD];
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
          v[k] = 0.0f;
          res[k] = p.residual != nullptr && m < p.M && c0 + 2 * k < c1 ? raw_element(p.residual, p.residual_elem, (long long)(t.n0 + c0 + 2 * k) * p.ldr + m) : 0u;
        }
#pragma unroll 2
        for (int q = 0; q < p.splits; ++q) {
          float part[HELD];
#pragma unroll
          for (int k = 0; k < HELD; ++k)
            part[k] = ld_cluster(cluster_address(ring + (uint32_t)(min(c0 + 2 * k, c1 - 1) * kBlock + quad * 32 + lane) * 4u, (uint32_t)q));
#pragma unroll
          for (int k = 0; k < HELD; ++k) v[k] += part[k];
        }
#pragma unroll
        for (int k = 0; k < HELD; ++k)
          if (m < p.M && c0 + 2 * k < c1) {
            float y = activate(v[k] + of_raw(bias_raw, p.bias_elem), p.act);
            if (p.residual != nullptr) y += of_raw(res[k], p.residual_elem);
            store_result(p, t.n0 + c0 + 2 * k, m, y);
          }
      }
    }
    __syncwarp();
    cluster_meet();   // (nobody leaves while others read its sums)
  }
  zero_tokens_in_no_run(p, runs);
  grid_launch_dependents();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (ctl_s[0]) {   // let copies that may still be in flight land before shared memory is given back
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {
    }
    if (tid == 0 && p.status != nullptr) atomicCAS(p.status, 0, kStatusTimeout);
    __syncthreads();
  }
  if (warp == 1) tmem_dealloc(tmem, kTmem);
}

// ------------------------------------------------------------------------------------------ many tokens
// Tokens are the lanes here, 256 features the columns: a thread that adds up has one token and one block of 128 features, so that both
// scales are one number of its own, and its results are 128 neighbours in memory.  Eight warps read an accumulator back and add it while the
// tensor cores fill the other one; they hold 128 sums a thread, which takes registers from the other warps (setmaxnreg).
//
// 8192 tokens, 8192 x 8192, bf16 with residual: 605 us at 1.97 GHz (1.82 PFLOP/s), 747 under the power cap (1.61 GHz, 989 W).  Its parts by themselves, in
// copies of the kernel: products 319, copies 371 (48 KB for every 128 x 256 x 128), both 478 (they share the bandwidth of shared memory), adding 390 to
// 490, all without the way out 561.  With features in the lanes and tokens in the columns, the scales read from shared memory: 1680.
// Taken back: two SMs for one item (cta_group::2; 32 KB a block, but accumulators handed back across SMs, of which there are only two: 1088); sixteen
// adding warps of 64 columns (641); two accumulators of 128 columns each for every block (695: products of 128 columns are bound by shared memory);
// the next block's first columns asked for ahead of the last of this one (823: registers are moved); pairs of numbers in one instruction (635).
constexpr int kWideTokens = 128, kWideFeatures = 256;
constexpr int kWideAhead = 4;                 // scales that are on their way, blocks of k
constexpr int kWidePitch = kWideFeatures + 4; // of partial sums in shared memory: 16-byte pieces of eight rows meet all banks
constexpr int kCopier = 8, kIssuer = 9, kBiasWarp = 10;
constexpr uint32_t kWideStage = (kWideTokens + kWideFeatures) * kBlock;
struct __align__(8) WideBars {
  uint64_t full[kMaxRing], empty[kMaxRing];
  uint64_t acc_full[2], acc_empty[2], bias_full[2], bias_empty[2];
};
__device__ __forceinline__ uint32_t pack2(float a, float b, int elem) {
  uint32_t r;
  if (elem == VOID_ELEM_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// Adds 16 residuals, a piece of 32 bytes or (fp32) two, to 16 results.
__device__ __forceinline__ void add_residual(float (&y)[16], const uint32_t (&u)[8], const uint32_t (&v)[8], int elem) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (elem == VOID_ELEM_F32) {
      y[k] += __uint_as_float(u[k]);
      y[8 + k] += __uint_as_float(v[k]);
    } else if (elem == VOID_ELEM_F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
      y[2 * k] += f.x;
      y[2 * k + 1] += f.y;
    } else {
      y[2 * k] += __uint_as_float(u[k] << 16);
      y[2 * k + 1] += __uint_as_float(u[k] & 0xffff0000u);
    }
  }
}
// 16 neighbouring results of a row that lies on 32 bytes.
__device__ __forceinline__ void store16(const Fp8Params& p, long long token, int m, const float (&y)[16]) {
  const long long at = token * p.ldc + m;
  uint32_t u[8];
  if (p.out_elem == VOID_ELEM_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = __float_as_uint(y[8 * h + k]);
      st_global_v8(reinterpret_cast<float*>(p.out) + at + 8 * h, u);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = pack2(y[2 * k], y[2 * k + 1], p.out_elem);
    st_global_v8(reinterpret_cast<uint16_t*>(p.out) + at, u);
  }
}

// 64 results of a row that lies on 32 bytes, and their residuals: four pieces of 32 bytes, or (fp32) twice four, fetched here.
template <class FETCH>
__device__ __forceinline__ void add_residuals(f32x2 (&y)[32], uint32_t (&u)[4][8], int elem, FETCH fetch) {
  if (elem == VOID_ELEM_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      fetch(32 * h);
#pragma unroll
      for (int k = 0; k < 16; ++k) y[16 * h + k] = add2(y[16 * h + k], pair(__uint_as_float(u[k / 4][2 * (k % 4)]), __uint_as_float(u[k / 4][2 * (k % 4) + 1])));
    }
  } else if (elem == VOID_ELEM_F16) {
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[k / 8][k % 8]));
      y[k] = add2(y[k], pair(f.x, f.y));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 32; ++k) y[k] = add2(y[k], pair(__uint_as_float(u[k / 8][k % 8] << 16), __uint_as_float(u[k / 8][k % 8] & 0xffff0000u)));
  }
}
__device__ __forceinline__ void store64(const Fp8Params& p, long long token, int m, const f32x2 (&y)[32]) {
  const long long at = token * p.ldc + m;
  uint32_t u[8];
  float a, b;
  if (p.out_elem == VOID_ELEM_F32) {
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      unpair(y[k], a, b);
      u[2 * (k % 4)] = __float_as_uint(a);
      u[2 * (k % 4) + 1] = __float_as_uint(b);
      if (k % 4 == 3) st_global_v8(reinterpret_cast<float*>(p.out) + at + 8 * (k / 4), u);
    }
  } else if (p.out_elem == VOID_ELEM_F16) {
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      unpair(y[k], a, b);
      u[k % 8] = pack2(a, b, VOID_ELEM_F16);
      if (k % 8 == 7) st_global_v8(reinterpret_cast<uint16_t*>(p.out) + at + 16 * (k / 8), u);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      unpair(y[k], a, b);
      u[k % 8] = pack2(a, b, VOID_ELEM_BF16);
      if (k % 8 == 7) st_global_v8(reinterpret_cast<uint16_t*>(p.out) + at + 16 * (k / 8), u);
    }
  }
}

// A cluster's sums meet: its tokens are dealt to the CTAs, halves of their rows to the adding warps, features to lanes.  The pieces of four halves, of one CTA
// after the other, are on their way together.  Four features of a lane lie side by side, or (LOOSE) 32 apart, so that neighbours in memory are
// neighbouring lanes' either way.
template <bool LOOSE>
__device__ __forceinline__ void add_parts(const Fp8Params& p, const Item& t, uint32_t ring, int rank, int warp, int lane) {
  constexpr int HELD = 4, APART = LOOSE ? 32 : 1;
  const int n = t.n1 - t.n0, share = (n + p.splits - 1) / p.splits, r0 = rank * share, r1 = min(n, r0 + share), units = (r1 - r0) * 2;
  const int half = warp & 1, f0 = half * kBlock + (LOOSE ? lane : 4 * lane), m = t.m * kWideFeatures + f0;
  bool in[4];
  uint32_t bias[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    in[c] = m + c * APART < p.M;
    bias[c] = in[c] && p.bias != nullptr ? raw_element(p.bias, p.bias_elem, (long long)t.expert * p.M + m + c * APART) : 0u;
  }
  const bool whole = !LOOSE && m + 4 <= p.M;   // (then rows lie on 32 bytes: four results are one store)
  for (int u0 = warp; u0 < units; u0 += kAdders * HELD) {   // (units of one warp are all first halves, or all second ones)
    float y[HELD][4];
    uint32_t res[HELD][4];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int u = u0 + k * kAdders;
      const long long at = (long long)(t.n0 + r0 + u / 2) * p.ldr + m;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        y[k][c] = 0.0f;
        res[k][c] = 0u;
      }
      if (p.residual == nullptr || u >= units) continue;
      if (whole && p.residual_elem != VOID_ELEM_F32) {
        const uint2 v = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.residual) + at);
        res[k][0] = v.x & 0xffffu; res[k][1] = v.x >> 16; res[k][2] = v.y & 0xffffu; res[k][3] = v.y >> 16;
      } else if (whole) {
        const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p.residual) + at);
        res[k][0] = v.x; res[k][1] = v.y; res[k][2] = v.z; res[k][3] = v.w;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (in[c]) res[k][c] = raw_element(p.residual, p.residual_elem, at + c * APART);
      }
    }
#pragma unroll 2
    for (int q = 0; q < p.splits; ++q) {
      float part[HELD][4];
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        const int row = r0 + min(u0 + k * kAdders, units - 1) / 2;
        const uint32_t from = cluster_address(ring + (uint32_t)(row * kWidePitch + f0) * 4u, (uint32_t)q);
        if constexpr (LOOSE) {
#pragma unroll
          for (int c = 0; c < 4; ++c) part[k][c] = ld_cluster(from + 128u * c);
        } else {
          const float4 v = ld_cluster4(from);
          part[k][0] = v.x; part[k][1] = v.y; part[k][2] = v.z; part[k][3] = v.w;
        }
      }
#pragma unroll
      for (int k = 0; k < HELD; ++k)
#pragma unroll
        for (int c = 0; c < 4; ++c) y[k][c] += part[k][c];
    }
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int u = u0 + k * kAdders;
      if (u >= units) continue;
      f32x2 z[2];
#pragma unroll
      for (int c = 0; c < 2; ++c)
        z[c] = add2(pair(y[k][2 * c], y[k][2 * c + 1]), pair(of_raw(bias[2 * c], p.bias_elem), of_raw(bias[2 * c + 1], p.bias_elem)));
      activate<2>(z, p.act);
      float v[4];
      unpair(z[0], v[0], v[1]);
      unpair(z[1], v[2], v[3]);
      if (p.residual != nullptr) {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] += of_raw(res[k][c], p.residual_elem);
      }
      const long long token = t.n0 + r0 + u / 2, at = token * p.ldc + m;
      if (whole && p.out_elem == VOID_ELEM_F32)
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
      else if (whole)
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at) = make_uint2(pack2(v[0], v[1], p.out_elem), pack2(v[2], v[3], p.out_elem));
      else
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (in[c]) store_result(p, token, m + c * APART, v[c]);
    }
  }
}

// LOOSE: rows of results or residuals that do not lie on 32 bytes.
template <bool LOOSE>
__global__ void __launch_bounds__(kThreads, 1) fp8_wide_kernel(const __grid_constant__ Fp8Params p, const __grid_constant__ CUtensorMap map_a,
                                                               const __grid_constant__ CUtensorMap map_x) {
  constexpr int COLS = kBlock;    // of an adding warp
  extern __shared__ uint8_t raw[];
  __shared__ WideBars bars;
  __shared__ __align__(16) float bias_s[2][kWideFeatures];
  __shared__ float strips[kAdders][32 * 17];   // results of a warp on their way from lanes that are tokens to lanes that are features
  __shared__ uint32_t tmem_s;
  __shared__ int ctl_s[2];
  __shared__ Runs runs;
  volatile int* ctl = ctl_s;
  const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    ctl_s[0] = 0;
    ctl_s[1] = p.wait_limit_ms;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&bars.full[s]), 1);
      mbar_init(smem_u32(&bars.empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&bars.acc_full[s]), 1);
      mbar_init(smem_u32(&bars.acc_empty[s]), kAdders);
      mbar_init(smem_u32(&bars.bias_full[s]), 1);
      mbar_init(smem_u32(&bars.bias_empty[s]), kAdders);
    }
    fence_mbar_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_x);
  }
  if (warp == kIssuer) {
    tmem_alloc(smem_u32(&tmem_s), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  grid_dependency_wait();
  find_runs(p, runs);

  const int rank = p.splits > 1 ? (int)cluster_rank() : 0;
  const int b0 = (int)((long long)p.k_blocks * rank / p.splits), b1 = (int)((long long)p.k_blocks * (rank + 1) / p.splits);
  const int step = (int)gridDim.x / p.splits, begin = (int)blockIdx.x / p.splits, end = items_of(p, runs);
  // (4 * 56 + 8 * 224 = 12 * 168, what the block was launched with)
  if (warp >= kAdders) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  if (warp == kCopier) {
    int stage = 0;
    uint32_t phase = 0;
    bool first = true;
    for (int i = begin; i < end && !ctl[0]; i += step) {
      const Item t = item_at(p, runs, i);
      const int m0 = t.m * kWideFeatures, halves = p.M - m0 > kBlock ? 2 : 1, boxes = (t.n1 - t.n0 + kTokenBox - 1) / kTokenBox;
      for (int b = b0; b < b1; ++b) {
        if (!mbar_wait_warp(smem_u32(&bars.empty[stage]), phase ^ 1u, ctl)) break;
        const bool drop = first && p.drop_first != 0;
        first = false;
        if (lane == 0 && !drop) {
          const uint32_t full = smem_u32(&bars.full[stage]), at = ring + (uint32_t)stage * kWideStage + kWideTokens * kBlock;
          mbar_expect_tx(full, (uint32_t)(halves * kBlock + boxes * kTokenBox) * kBlock);
          for (int h = 0; h < halves; ++h) tma_load_3d(at + (uint32_t)h * (kBlock * kBlock), &map_a, b * kBlock, m0 + h * kBlock, t.expert, full);
        }
        __syncwarp();
        if (lane >= 1 && lane <= boxes && !drop)
          tma_load_2d(ring + (uint32_t)stage * kWideStage + (uint32_t)(lane - 1) * (kTokenBox * kBlock), &map_x, b * kBlock, t.n0 + (lane - 1) * kTokenBox,
                      smem_u32(&bars.full[stage]));
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == kIssuer) {
    constexpr uint64_t kDescHi = smem_desc_hi(16, 1024, kLayoutSw128);
    const bool leader = elect_one();
    int stage = 0;
    uint32_t phase = 0, it = 0;
    bool ok = true;
    for (int i = begin; i < end && ok; i += step) {
      const Item t = item_at(p, runs, i);
      const uint32_t idesc = instr_desc(1, 0, 0, 0, 0, kWideTokens, p.M - t.m * kWideFeatures > kBlock ? kWideFeatures : kBlock);
      for (int b = b0; b < b1; ++b, ++it) {
        const uint32_t slot = it & 1u;
        ok = mbar_wait_warp(smem_u32(&bars.full[stage]), phase, ctl) && mbar_wait_warp(smem_u32(&bars.acc_empty[slot]), ((it >> 1) & 1u) ^ 1u, ctl);
        if (!ok) break;
        tc_fence_after();
        const uint32_t at = ring + (uint32_t)stage * kWideStage;
        const uint64_t dx = smem_desc(kDescHi, at), da = smem_desc(kDescHi, at + kWideTokens * kBlock);
#pragma unroll
        for (int k = 0; k < 4; ++k)   // 32 features each: 32 bytes further in rows of 128
          issue_mma<VOID_KIND_F8E4M3>(leader, tmem + slot * kWideFeatures, dx + 2 * k, da + 2 * k, idesc, k > 0);
        tc_commit_if(leader, smem_u32(&bars.empty[stage]));
        tc_commit_if(leader, smem_u32(&bars.acc_full[slot]));
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == kBiasWarp) {   // biases of an item, asked for while the one before is multiplied
    uint32_t it = 0;
    for (int i = begin; i < end && p.splits == 1; i += step, ++it) {
      const Item t = item_at(p, runs, i);
      float v[kWideFeatures / 32];
#pragma unroll
      for (int k = 0; k < kWideFeatures / 32; ++k) {
        const int m = t.m * kWideFeatures + lane + 32 * k;
        v[k] = p.bias != nullptr && m < p.M ? element(p.bias, p.bias_elem, (long long)t.expert * p.M + m) : 0.0f;
      }
      if (!mbar_wait_warp(smem_u32(&bars.bias_empty[it & 1u]), ((it >> 1) & 1u) ^ 1u, ctl)) break;
#pragma unroll
      for (int k = 0; k < kWideFeatures / 32; ++k) bias_s[it & 1u][lane + 32 * k] = v[k];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars.bias_full[it & 1u]));
    }
  } else if (warp < kAdders) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int quad = warp & 3, side = warp >> 2;
    uint32_t it = 0, item = 0;
    bool ok = true;
    for (int i = begin; i < end && ok; i += step, ++item) {
      const Item t = item_at(p, runs, i);
      const int n = t.n1 - t.n0, token = quad * 32 + lane, m0 = t.m * kWideFeatures + side * COLS;
      const bool mine = token < n, any = m0 < p.M && quad * 32 < n;   // (any: of what this warp reads back)
      const long long row = t.n0 + token;
      const float* sx = p.x_scale + row * p.xs_row;
      const float* sa = p.a_scale + t.expert * p.as_expert + (long long)(2 * t.m + side) * p.as_row;
      float ahead_x[kWideAhead], ahead_a[kWideAhead], scale[kWideAhead];
      auto fetch = [&](int b) {
#pragma unroll
        for (int k = 0; k < kWideAhead; ++k) {
          const bool in = mine && any && b + k < b1;
          ahead_x[k] = in ? sx[(long long)(b + k) * p.xs_col] : 0.0f;
          ahead_a[k] = in ? sa[(long long)(b + k) * p.as_col] : 0.0f;
        }
      };
      fetch(b0);
      if (mine && any && p.residual != nullptr) {   // on its way into the second cache while the products are made
        const int es = p.residual_elem == VOID_ELEM_F32 ? 4 : 2, bytes = (p.M - m0 < COLS ? p.M - m0 : COLS) * es;
        const uint8_t* from = reinterpret_cast<const uint8_t*>(p.residual) + (row * p.ldr + m0) * es;
        for (int at = 0; at < bytes; at += 128) prefetch_l2(from + at);
      }
      float sum[COLS];   // (pairs of numbers in one instruction, which read three pairs of registers: 635 us for 8192^3 against 605)
#pragma unroll
      for (int c = 0; c < COLS; ++c) sum[c] = 0.0f;
      for (int b = b0; b < b1 && ok; b += kWideAhead) {
#pragma unroll
        for (int k = 0; k < kWideAhead; ++k) scale[k] = ahead_x[k] * ahead_a[k];
        if (b + kWideAhead < b1) fetch(b + kWideAhead);
#pragma unroll 1
        for (int k = 0; k < kWideAhead && b + k < b1; ++k, ++it) {
          const uint32_t slot = it & 1u;
          const float s = scale[0];
#pragma unroll
          for (int q = 0; q + 1 < kWideAhead; ++q) scale[q] = scale[q + 1];
          ok = mbar_wait_warp(smem_u32(&bars.acc_full[slot]), (it >> 1) & 1u, ctl);
          if (!ok) break;
          tc_fence_after();
          auto hand_back = [&] {   // all is read back: the next product may begin
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars.acc_empty[slot]));
          };
          if (any) {
            const uint32_t from = tmem + slot * kWideFeatures + (uint32_t)(side * COLS) + ((uint32_t)(quad * 32) << 16);
            uint32_t r[2][32];
            tmem_ld_32x32(from, r[0]);
#pragma unroll
            for (int g = 0; g < COLS / 32; ++g) {
              tmem_ld_wait();
              if (g + 1 < COLS / 32) tmem_ld_32x32(from + 32u * (g + 1), r[(g + 1) & 1]);
              else hand_back();
#pragma unroll
              for (int c = 0; c < 32; ++c) sum[32 * g + c] = fmaf(__uint_as_float(r[g & 1][c]), s, sum[32 * g + c]);
            }
          } else {
            hand_back();
          }
        }
      }
      if (!ok) break;
      if (p.splits > 1) {
        float* part = reinterpret_cast<float*>(raw + (ring - smem_u32(raw))) + token * kWidePitch + side * COLS;   // [tokens][features]
        if (mine && any) {
#pragma unroll
          for (int c = 0; c < COLS; c += 4) *reinterpret_cast<float4*>(part + c) = make_float4(sum[c], sum[c + 1], sum[c + 2], sum[c + 3]);
        }
        break;   // (one item per cluster)
      }
      ok = mbar_wait_warp(smem_u32(&bars.bias_full[item & 1u]), (item >> 1) & 1u, ctl);
      if (!ok) break;
      if (any) {
        const float4* bias = reinterpret_cast<const float4*>(&bias_s[item & 1u][side * COLS]);
        const int pieces = p.residual_elem == VOID_ELEM_F32 ? 2 : 1;   // of 32 bytes, of 16 residuals
        const uint8_t* from = reinterpret_cast<const uint8_t*>(p.residual) + (row * p.ldr + m0) * (pieces == 2 ? 4 : 2);
        uint32_t res[4][8];   // four pieces of residuals on their way together: of 64 results, or (fp32) of 32
        auto fetch_residuals = [&](int c0, int width) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (mine && m0 + (c0 + q * width) / 16 * 16 + 16 <= p.M) ld_global_v8(from + (c0 + q * width) / width * 32, res[q]);
        };
#pragma unroll
        for (int h = 0; h < COLS; h += 64) {
          if (!LOOSE && p.residual != nullptr && pieces == 1) fetch_residuals(h, 16);
          if (!LOOSE && m0 + h + 64 <= p.M) {   // 64 results step by step: two warps of a scheduler wait for each other's instructions, and each for its own
            f32x2 y[32];
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const float4 v = bias[h / 4 + c];
              y[2 * c] = add2(pair(sum[h + 4 * c], sum[h + 4 * c + 1]), pair(v.x, v.y));
              y[2 * c + 1] = add2(pair(sum[h + 4 * c + 2], sum[h + 4 * c + 3]), pair(v.z, v.w));
            }
            activate<32>(y, p.act);
            if (p.residual != nullptr) add_residuals(y, res, p.residual_elem, [&](int c) { fetch_residuals(h + c, 8); });
            if (mine) store64(p, row, m0 + h, y);
            continue;
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (!LOOSE && p.residual != nullptr && pieces == 2 && q % 2 == 0) fetch_residuals(h + 16 * q, 8);
            const int c0 = h + 16 * q, m = m0 + c0;
            f32x2 y2[8];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float4 v = bias[c0 / 4 + c];
              y2[2 * c] = add2(pair(sum[c0 + 4 * c], sum[c0 + 4 * c + 1]), pair(v.x, v.y));
              y2[2 * c + 1] = add2(pair(sum[c0 + 4 * c + 2], sum[c0 + 4 * c + 3]), pair(v.z, v.w));
            }
            activate<8>(y2, p.act);
            float y[16];
#pragma unroll
            for (int c = 0; c < 8; ++c) unpair(y2[c], y[2 * c], y[2 * c + 1]);
            if (!LOOSE && m + 16 <= p.M) {
              if (p.residual != nullptr) add_residual(y, pieces == 2 ? res[q % 2 * 2] : res[q], res[q % 2 * 2 + 1], p.residual_elem);
              if (mine) store16(p, row, m, y);
            } else if (m < p.M) {   // two rows at a time, 16 lanes each
              float* strip = strips[warp];
              __syncwarp();
#pragma unroll
              for (int c = 0; c < 16; ++c) strip[lane * 17 + c] = y[c];
              __syncwarp();
              const int col = lane & 15;
              // (loops that stay loops: unrolled for every group of columns, this code is read from memory for each item)
              const int first = lane >> 4, rows_left = m + col < p.M ? n - quad * 32 : 0;
              const long long at = row - lane + first;
#pragma unroll 1
              for (int k0 = 0; k0 < 32; k0 += 16) {
                uint32_t raw_res[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  raw_res[k] = p.residual != nullptr && k0 + 2 * k + first < rows_left ? raw_element(p.residual, p.residual_elem, (at + k0 + 2 * k) * p.ldr + m + col) : 0u;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  float v = strip[(k0 + 2 * k + first) * 17 + col];
                  if (p.residual != nullptr) v += of_raw(raw_res[k], p.residual_elem);
                  if (k0 + 2 * k + first < rows_left) store_result(p, at + k0 + 2 * k, m + col, v);
                }
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars.bias_empty[item & 1u]));
    }
    if (p.splits > 1) {
      __syncwarp();
      cluster_meet();
      if (begin < end) add_parts<LOOSE>(p, item_at(p, runs, begin), ring, rank, warp, lane);
    }
  }
  if (p.splits > 1) {   // (the adding warps have met the others already)
    __syncwarp();
    if (warp >= kAdders) cluster_meet();
    cluster_meet();   // (nobody leaves while others read its sums)
  }
  zero_tokens_in_no_run(p, runs);
  grid_launch_dependents();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (ctl_s[0]) {   // let copies that may still be in flight land before shared memory is given back
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {
    }
    if (tid == 0 && p.status != nullptr) atomicCAS(p.status, 0, kStatusTimeout);
    __syncthreads();
  }
  if (warp == kIssuer) tmem_dealloc(tmem, 512);
}

bool rows_map(CUtensorMap* m, const void* at, long long ld, long long expert, int K, int rows, int experts, int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = get_encode();
  if (enc == nullptr) return false;
  const cuuint64_t gdim[3] = {(cuuint64_t)K, (cuuint64_t)rows, (cuuint64_t)experts};
  const cuuint64_t gstride[2] = {(cuuint64_t)ld, (cuuint64_t)expert};
  const cuuint32_t box[3] = {(cuuint32_t)kBlock, (cuuint32_t)box_rows, 1};
  const cuuint32_t estride[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, experts > 0 ? 3 : 2, const_cast<void*>(at), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How many clusters of `splits` such CTAs a device holds at a time: a cluster lies within one of its groups of SMs, so some SMs are left over (36
// clusters of four CTAs, one per SM, took two turns where 33 fit).  For kernels that hold tensor memory
// the runtime answers for one CTA per SM.
int clusters_at_once(const void* kernel, int splits, int smem) {
  struct Rec { const void* fn; int dev, splits, smem, clusters; };
  static Rec recs[256];
  static int n_recs = 0;
  static std::mutex mu;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < n_recs; ++i)
    if (recs[i].fn == kernel && recs[i].dev == dev && recs[i].splits == splits && recs[i].smem == smem) return recs[i].clusters;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)splits);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) return 0;
  if (n_recs < 256) recs[n_recs++] = {kernel, dev, splits, smem, clusters};
  return clusters;
}
// Launch with `splits` CTAs per item, in clusters: as many as there are SMs for, as long as every CTA has four blocks of k, or places (`ctas` per SM) if
// it still has `least`.  us in graphs with one CTA per SM and with two, by the blocks that each then has.  Items of 32 tokens (least 32), 8 tokens: 16 blocks
// 8192^2 17.2 17.5, 4096 -> 16384 15.6 17.2; 32 blocks 16384 -> 8192 29.4 26.8, 8192 -> 12288 23.8 22.0; 64 blocks 16384^2 49.5 47.9.  Items of 64 (16), 64 tokens: 4 blocks
// 4096^2 12.2 14.1; 8 blocks 8192 -> 4096 15.8 17.6, 4096 -> 8192 16.6 15.2; 16 blocks 8192^2 23.5 20.7, 4096 -> 16384 21.6 21.9, 16384 -> 4096 22.6 24.1; 32 blocks 16384 -> 8192
// 37.9 31.1; 64 blocks 16384^2 63.9 55.5.
cudaError_t launch_split(void (*kernel)(Fp8Params, CUtensorMap, CUtensorMap), Fp8Params& p, const CUtensorMap& a, const CUtensorMap& x, long long items,
                         const DeviceInfo& dev, int ctas, int least, int smem, cudaStream_t st) {
  const long long places = (long long)dev.sms * ctas;
  int splits = 1;
  for (int s = 8; s > 1 && splits == 1; --s)
    if (p.k_blocks >= 4 * s && (items * s <= dev.sms || (items * s <= places && p.k_blocks >= least * s)) &&
        items <= ctas * clusters_at_once(reinterpret_cast<const void*>(kernel), s, smem))
      splits = s;
  p.splits = splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(splits > 1 ? items * splits : (items < places ? items : places)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p, a, x);
}
// Stages of a ring in the shared memory that `ctas` CTAs leave each other.
int ring_stages(const DeviceInfo& dev, int ctas, int stage_bytes, int fixed) {
  fixed += 64 + 1024 + 1024;   // (alignment, and what the system keeps of a CTA's)
  int stages = (dev.smem_per_sm / ctas - fixed) / stage_bytes;
  const int most = (dev.max_smem - fixed) / stage_bytes;
  if (stages > most) stages = most;
  return stages > kMaxRing ? kMaxRing : stages;
}
template <int NT>
int launch_few(Fp8Params p, const CUtensorMap& a, const CUtensorMap& x, long long items, const DeviceInfo& dev, cudaStream_t st) {
  constexpr int kStage = kBlock * kBlock + NT * kBlock;
  static_assert(NT * kBlock * 4 <= 2 * kStage, "the partial sums lie in the ring");
  p.stages = ring_stages(dev, kFewCtas, kStage, (int)(sizeof(Fp8Bars) + sizeof(Runs)) + kScaleSlots * NT * 4);
  const int smem = p.stages * kStage + 1024;
  if (p.stages < 2) return VOID_ERR_SHAPE;
  if (ensure_smem(reinterpret_cast<const void*>(fp8_block_kernel<NT>), smem) != 0) return VOID_ERR_CUDA;
  return status_of(launch_split(fp8_block_kernel<NT>, p, a, x, items, dev, kFewCtas, NT == 32 ? 32 : 16, smem, st));
}
template <bool LOOSE>
int launch_wide(Fp8Params p, const CUtensorMap& a, const CUtensorMap& x, long long items, const DeviceInfo& dev, cudaStream_t st) {
  constexpr int kStage = (int)kWideStage;
  p.stages = ring_stages(dev, 1, kStage, (int)(sizeof(WideBars) + sizeof(Runs)) + 2 * kWideFeatures * 4 + kAdders * 32 * 17 * 4);
  const int smem = p.stages * kStage + 1024;
  if (p.stages * kStage < kWideTokens * kWidePitch * 4) return VOID_ERR_SHAPE;
  if (ensure_smem(reinterpret_cast<const void*>(fp8_wide_kernel<LOOSE>), smem) != 0) return VOID_ERR_CUDA;
  return status_of(launch_split(fp8_wide_kernel<LOOSE>, p, a, x, items, dev, 1, 4, smem, st));
}
// Rows of results and residuals in pieces of 32 bytes.
bool on_32_bytes(const void* at, long long ld, int elem) { return ((reinterpret_cast<uintptr_t>(at) | (uintptr_t)(ld * (elem == VOID_ELEM_F32 ? 4 : 2))) & 31u) == 0; }

int fp8_linear(const void_fp8_args* a, const void_experts* x, cudaStream_t st) {
  if (a == nullptr || a->M < 0 || a->K < 0 || a->N < 0) return VOID_ERR_BAD_ARG;
  if (a->out_elem < VOID_ELEM_F32 || a->out_elem > VOID_ELEM_BF16 || a->bias_elem < VOID_ELEM_F32 || a->bias_elem > VOID_ELEM_BF16 ||
      a->residual_elem < VOID_ELEM_F32 || a->residual_elem > VOID_ELEM_BF16 || a->act < VOID_ACT_NONE || a->act > VOID_ACT_SILU)
    return VOID_ERR_BAD_ARG;
  if (a->M == 0 || a->N == 0) return VOID_OK;
  // (K: an item's time has to stay within the limit of the kernels' waits; M, N: places behind the last item are numbers, too)
  if (a->K > 1 << 28 || a->M > 0x7fffff00 || a->N > 0x40000000) return VOID_ERR_TOO_LARGE;
  if (a->out == nullptr || a->K == 0 || a->a == nullptr || a->x == nullptr || a->a_scale == nullptr || a->x_scale == nullptr) return VOID_ERR_BAD_ARG;
  if (x != nullptr && (x->n_experts < 1 || x->plan == nullptr || (x->offset_bytes != 0 && ((x->offset_bytes != 4 && x->offset_bytes != 8) || x->n_experts > 32)) || (x->chunk != 32 && x->chunk != 64 && x->chunk != 128)))
    return VOID_ERR_BAD_ARG;
  if (a->ldc < a->M || (a->residual != nullptr && a->ldr < a->M)) return VOID_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a->a) & 15u) != 0 || (reinterpret_cast<uintptr_t>(a->x) & 15u) != 0 || (a->lda & 15) != 0 || (a->ldx & 15) != 0 ||
      a->lda < a->K || a->ldx < a->K || (x != nullptr && ((a->expert_stride & 15) != 0 || a->expert_stride < 0 || (reinterpret_cast<uintptr_t>(x->plan) & (x->offset_bytes != 0 ? x->offset_bytes - 1u : 15u)) != 0)))
    return VOID_ERR_ALIGN;
  auto bytes_of = [](int elem) { return elem == VOID_ELEM_F32 ? 4 : 2; };
  if (!lies_on(a->a_scale, 4) || !lies_on(a->x_scale, 4) || !lies_on(a->status, 4) || !lies_on(a->bias, bytes_of(a->bias_elem)) ||
      !lies_on(a->residual, bytes_of(a->residual_elem)) || !lies_on(a->out, bytes_of(a->out_elem)))
    return VOID_ERR_ALIGN;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  Fp8Params p = {};
  p.M = a->M; p.K = a->K; p.N = a->N;
  p.k_blocks = (a->K + kBlock - 1) / kBlock;
  p.a_scale = a->a_scale; p.as_row = a->a_scale_row; p.as_col = a->a_scale_col; p.as_expert = a->a_scale_expert;
  p.x_scale = a->x_scale; p.xs_row = a->x_scale_row; p.xs_col = a->x_scale_col;
  p.bias = a->bias; p.bias_elem = a->bias_elem;
  p.residual = a->residual; p.ldr = a->ldr; p.residual_elem = a->residual_elem;
  p.out = a->out; p.ldc = a->ldc; p.out_elem = a->out_elem; p.act = a->act;
  p.status = a->status;
  p.wait_limit_ms = (a->test_hooks & 0xffff) ? (a->test_hooks & 0xffff) : kDefaultWaitLimitMs;
  p.drop_first = (a->test_hooks >> 16) & 1;
  // Up to 64 tokens lie in the columns of the tensor memory, more of them in its lanes.
  const int chunk = x != nullptr ? x->chunk : (a->N <= 32 ? 32 : (a->N <= 64 ? 64 : kWideTokens));
  const bool wide = chunk == kWideTokens;
  p.m_tiles = wide ? (a->M + kWideFeatures - 1) / kWideFeatures : (a->M + kBlock - 1) / kBlock;
  long long chunks;
  if (x != nullptr) {
    const PlanView v = plan_of(*x, a->N);
    if (x->offset_bytes != 0) {
      p.offsets = x->plan;
      p.offset_bytes = x->offset_bytes;
    } else {
      p.head = v.head; p.bounds = v.bounds; p.chunks = v.chunks;
    }
    p.chunk = chunk;
    p.n_experts = x->n_experts;
    p.zero_rest = x->zero_rest;
    chunks = v.capacity;
  } else {
    p.chunk = chunk;
    chunks = p.n_chunks = (int)(((long long)a->N + chunk - 1) / chunk);
    p.group = 16;   // 8192^3, us by groups of 1, 4, 16, 32, 64: 610 588 581 575 604; 4096 tokens, 4096 -> 16384 330 314 310 309 310; fewer tokens or features: no matter
  }
  const long long items = chunks * p.m_tiles;
  if (items > 0x3fffffff) return VOID_ERR_TOO_LARGE;
  CUtensorMap map_a, map_x;
  const int experts = x != nullptr ? x->n_experts : 1;
  if (!rows_map(&map_a, a->a, a->lda, x != nullptr ? a->expert_stride : (a->lda * a->M + 15) / 16 * 16, a->K, a->M, experts, kBlock) ||
      !rows_map(&map_x, a->x, a->ldx, 0, a->K, a->N, 0, kTokenBox))
    return VOID_ERR_TENSOR_MAP;
  if (wide) {
    const bool loose = !on_32_bytes(a->out, a->ldc, a->out_elem) || (a->residual != nullptr && !on_32_bytes(a->residual, a->ldr, a->residual_elem));
    return loose ? launch_wide<true>(p, map_a, map_x, items, dev, st) : launch_wide<false>(p, map_a, map_x, items, dev, st);
  }
  if (chunk == 32) return launch_few<32>(p, map_a, map_x, items, dev, st);
  return launch_few<64>(p, map_a, map_x, items, dev, st);
}

}  // namespace

}  // namespace vb

extern "C" {

int void_quant_fp8_blocks(const void* x, int32_t elem, int64_t ldx, int64_t rows, int32_t cols, int32_t block_rows, void* q, int64_t ldq, float* scales,
                          int64_t scale_row, int64_t scale_col, void_stream_t stream) {
  using namespace vb;
  if (rows < 0 || cols < 0 || elem < VOID_ELEM_F32 || elem > VOID_ELEM_BF16 || (block_rows != 1 && block_rows != kBlock)) return VOID_ERR_BAD_ARG;
  if (rows > 1 && (ldx < cols || ldq < cols)) return VOID_ERR_SHAPE;
  if (rows == 0 || cols == 0) return VOID_OK;
  if (x == nullptr || q == nullptr || scales == nullptr) return VOID_ERR_BAD_ARG;
  if (!lies_on(x, elem == VOID_ELEM_F32 ? 4 : 2) || !lies_on(scales, 4)) return VOID_ERR_ALIGN;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  QuantParams p = {};
  p.x = x; p.ldx = ldx; p.ldq = ldq; p.scale_row = scale_row; p.scale_col = scale_col; p.rows = rows; p.cols = cols;
  p.q = reinterpret_cast<uint8_t*>(q); p.scales = scales;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (elem == VOID_ELEM_F32) return quant_of_type<float>(p, block_rows, dev.sms, st);
  return elem == VOID_ELEM_F16 ? quant_of_type<__half>(p, block_rows, dev.sms, st) : quant_of_type<__nv_bfloat16>(p, block_rows, dev.sms, st);
}

int void_fp8_linear(const void_fp8_args* args, const void_experts* experts, void_stream_t stream) {
  return vb::fp8_linear(args, experts, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
