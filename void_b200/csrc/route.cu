// Tokens on their way to the experts and back:
//
//   router     the k largest of a token's scores, and w = softmax of them (over the chosen ones, or over all)
//              ds_i = p_i (g_i - sum_j g_j p_j)
//   sort       row of every choice (token t, slot j) when all are sorted by expert, in the order of the tokens
//   dispatch   xs[row(t, j)] = x[t]
//   combine    y[t] = r[t] + sum_j w[t, j] ys[row(t, j)]
//              dys[row(t, j)] = w[t, j] dy[t],  dw[t, j] = <dy[t], ys[row(t, j)]>; dispatch's gradient is combine without weights
//
// A choice of no expert (an id outside [0, experts)) is dropped: it has row -1, brings nothing into the sum, and leaves a row behind the last
// run, which dispatch and combine's gradient fill with zeros.  All sums are fp32 and taken in the order of the slots; nothing depends on the
// order in which blocks ran.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/void_b200.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "values.cuh"

namespace vb {

namespace {

constexpr unsigned kAll = 0xffffffffu;
inline int elem_size(int elem) { return elem == VOID_ELEM_F32 ? 4 : 2; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// ------------------------------------------------------------------------------------------ router
// Numbers as unsigned ones of the same order: NaN above all, -0 the same as 0, 0 for what is taken or not there.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kKeyOfMinusInfinity = 0x007fffffu;

struct RouteParams {
  const void* scores;
  long long lds, rows;
  int experts, top, normalize;
  int32_t* chosen;    // forward
  float* weights;
  const float* g;     // backward
  long long ldg;
  void* ds;
  long long ldd;
};
constexpr int kRouteWarps = 4;

// A warp per token, expert e in lane e % 32.  A slot takes two warp-wide reductions in hardware: the largest key, then the lowest index
// that has it.  The backward pass chooses again, from the scores: what it keeps of the forward pass is nothing that a caller could change.
// A few tokens are a launch and one trip to memory (1.5 us in a graph); 16384 tokens, eight of 128 fp32 scores, take 12 us where their 8 MB take 1.3, the gradient
// 14: instructions bound it (9.7 and 12.8 million of warps, issued in 73 and 75 % of cycles; a lane that keeps its best and looks again only when that is
// taken: 13.6).
template <typename T, int PER_LANE, bool GRAD>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const __grid_constant__ RouteParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  for (long long t = (long long)blockIdx.x * kRouteWarps + (threadIdx.x >> 5); t < p.rows; t += (long long)gridDim.x * kRouteWarps) {
    const T* row = reinterpret_cast<const T*>(p.scores) + t * p.lds;
    float s[PER_LANE];
    uint32_t key[PER_LANE];
#pragma unroll
    for (int v = 0; v < PER_LANE; ++v) {
      const int e = lane + 32 * v;
      s[v] = e < p.experts ? to_float<T>(row[e]) : -INFINITY;
    }
    float slot_grad = 0.0f;
    if constexpr (GRAD) slot_grad = lane < p.top ? p.g[t * p.ldg + lane] : 0.0f;
#pragma unroll
    for (int v = 0; v < PER_LANE; ++v) key[v] = lane + 32 * v < p.experts ? order_key(s[v]) : 0u;
    int taken = 0, id = -1;   // id, score: of the slot that is this lane's
    float score = 0.0f, largest = 0.0f;
    for (int j = 0; j < p.top; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int v = 0; v < PER_LANE; ++v) best = key[v] > best ? key[v] : best;
      best = __reduce_max_sync(kAll, best);
      if (best <= kKeyOfMinusInfinity) break;   // (an expert whose score is -infinity is never chosen)
      uint32_t at = kAll;
#pragma unroll
      for (int v = PER_LANE - 1; v >= 0; --v) at = key[v] == best ? (uint32_t)(lane + 32 * v) : at;
      at = __reduce_min_sync(kAll, at);
#pragma unroll
      for (int v = 0; v < PER_LANE; ++v) key[v] = at == (uint32_t)(lane + 32 * v) ? 0u : key[v];
      if (j == 0) largest = of_key(best);
      if (lane == j) {
        id = (int)at;
        score = of_key(best);
      }
      ++taken;
    }
    const float mine = lane < taken ? expf(score - largest) : 0.0f;
    float total;
    if (p.normalize) {
      total = warp_sum(mine);
    } else {
      float part = 0.0f;
#pragma unroll
      for (int v = 0; v < PER_LANE; ++v) {
        s[v] = taken > 0 ? expf(s[v] - largest) : 0.0f;
        part += s[v];
      }
      total = warp_sum(part);
    }
    const float w = lane < taken ? mine / total : 0.0f;
    if constexpr (!GRAD) {
      if (lane < p.top) {
        p.chosen[t * p.top + lane] = id;
        p.weights[t * p.top + lane] = w;
      }
    } else {
      const float mean = warp_sum(lane < taken ? slot_grad * w : 0.0f);
      float d[PER_LANE];
#pragma unroll
      for (int v = 0; v < PER_LANE; ++v) d[v] = p.normalize || taken == 0 ? 0.0f : s[v] / total * -mean;
      for (int j = 0; j < taken; ++j) {
        const int at = __shfl_sync(kAll, id, j);
        const float value = __shfl_sync(kAll, w * (slot_grad - mean), j);
#pragma unroll
        for (int v = 0; v < PER_LANE; ++v) d[v] = at == lane + 32 * v ? value : d[v];
      }
      T* out = reinterpret_cast<T*>(p.ds) + t * p.ldd;
#pragma unroll
      for (int v = 0; v < PER_LANE; ++v)
        if (lane + 32 * v < p.experts) out[lane + 32 * v] = from_float<T>(d[v]);
    }
  }
}

template <typename T, bool GRAD>
int route_of_type(const RouteParams& p, int sms, cudaStream_t st) {
  const long long blocks = (p.rows + kRouteWarps - 1) / kRouteWarps;
  const int grid = (int)(blocks < 16ll * sms ? blocks : 16ll * sms), threads = 32 * kRouteWarps;
  const int per_lane = (p.experts + 31) / 32;
  if (per_lane <= 1) return status_of(launch_pdl(route_kernel<T, 1, GRAD>, grid, threads, 0, st, p));
  if (per_lane <= 2) return status_of(launch_pdl(route_kernel<T, 2, GRAD>, grid, threads, 0, st, p));
  if (per_lane <= 4) return status_of(launch_pdl(route_kernel<T, 4, GRAD>, grid, threads, 0, st, p));
  if (per_lane <= 8) return status_of(launch_pdl(route_kernel<T, 8, GRAD>, grid, threads, 0, st, p));
  if (per_lane <= 16) return status_of(launch_pdl(route_kernel<T, 16, GRAD>, grid, threads, 0, st, p));
  return status_of(launch_pdl(route_kernel<T, 32, GRAD>, grid, threads, 0, st, p));
}
template <bool GRAD>
int route_launch(const RouteParams& p, int elem, cudaStream_t st) {
  if (p.rows < 0 || p.experts < 1 || p.top < 1 || elem < VOID_ELEM_F32 || elem > VOID_ELEM_BF16) return VOID_ERR_BAD_ARG;
  if (p.top > p.experts || p.lds < 0 || (p.rows > 1 && GRAD && (p.ldd < p.experts || p.ldg < 0))) return VOID_ERR_SHAPE;
  if (p.experts > 1024 || p.top > 32 || p.rows > 0x7fffffffll) return VOID_ERR_TOO_LARGE;
  if (p.rows == 0) return VOID_OK;
  if (p.scores == nullptr || (GRAD ? p.g == nullptr || p.ds == nullptr : p.chosen == nullptr || p.weights == nullptr)) return VOID_ERR_BAD_ARG;
  if (!lies_on(p.scores, elem_size(elem)) || !lies_on(p.ds, elem_size(elem)) || !lies_on(p.g, 4) || !lies_on(p.chosen, 4) || !lies_on(p.weights, 4)) return VOID_ERR_ALIGN;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  if (elem == VOID_ELEM_F32) return route_of_type<float, GRAD>(p, dev.sms, st);
  return elem == VOID_ELEM_F16 ? route_of_type<__half, GRAD>(p, dev.sms, st) : route_of_type<__nv_bfloat16, GRAD>(p, dev.sms, st);
}

// ------------------------------------------------------------------------------------------ sort
// A counting sort that keeps the order of the choices within an expert: a warp ranks 32 choices at once by asking which lanes have the same
// expert, 32 warps meet in a table of their counts, and the CTAs of a cluster add up each other's.  More choices than one cluster holds in registers
// (32768) are dealt to blocks in order, which a launch of its own counts first.  In graphs, us: 1024 choices of 64 experts 3.4, 9003 of 17 5.1, 32768 of 64 5.9 (by
// the two launches 12), 131072 of 128 10.9 (by one cluster, 16 choices a thread, 15.5): latency, a few barriers and trips to memory.
constexpr int kSortThreads = 1024, kSortSteps = 4, kSortTile = kSortThreads * kSortSteps;
constexpr int kMaxSortExperts = 1024;
constexpr int kSortCluster = 8, kMostInCluster = kSortCluster * kSortTile;

struct SortParams {
  const void* experts;
  long long count, share;   // choices, and of one block (a multiple of a tile)
  int n_experts, pitch;     // pitch: entries between the warps' counts in shared memory
  int32_t* table;           // [blocks][experts] counts
  int32_t* offsets;
  int32_t* position;
};
template <typename I>
__device__ __forceinline__ int expert_of(const void* experts, long long i, int n_experts) {
  const long long e = (long long)reinterpret_cast<const I*>(experts)[i];
  return e < 0 || e >= n_experts ? -1 : (int)e;
}
// Sum of the values of the threads before, for the whole block; `s` has a word per warp.
__device__ __forceinline__ int sum_before(int v, int32_t* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(kAll, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) s[warp] = upto;
  __syncthreads();
  int first = upto - v;
  for (int w = 0; w < warp; ++w) first += s[w];
  return first;
}
// Lanes with the same expert as this one (a dropped choice: any): a vote for each bit of the number.  __match_any_sync takes a step for every expert that
// there is: 32768 choices of 64 experts 7.4 us that way.
__device__ __forceinline__ unsigned same_expert(int expert, int bits) {
  unsigned same = __ballot_sync(kAll, expert >= 0);
  for (int b = 0; b < bits; ++b) {
    const unsigned set = __ballot_sync(kAll, expert >> b & 1);
    same &= (expert >> b & 1) ? set : ~set;
  }
  return same;
}
template <typename I>
__device__ __forceinline__ void count_choices(const SortParams& p, long long begin, long long end, int32_t* counts) {
  for (int e = threadIdx.x; e < p.n_experts; e += blockDim.x) counts[e] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (long long i = begin + threadIdx.x; i - lane < end; i += blockDim.x) {
    const int e = i < end ? expert_of<I>(p.experts, i, p.n_experts) : -1;
    const unsigned same = same_expert(e, 32 - __clz(p.n_experts - 1));
    if (e >= 0 && lane == __ffs(same) - 1) atomicAdd(&counts[e], __popc(same));   // (whole numbers: any order gives the same)
  }
  __syncthreads();
}

// Ranks of a warp's choices among its own, and their counts in the warp's row of the table.
template <int STEPS>
__device__ __forceinline__ void rank_choices(const int (&expert)[STEPS], int (&rank)[STEPS], uint16_t* counts, int n_experts) {
  const int lane = threadIdx.x & 31, bits = 32 - __clz(n_experts - 1);
  unsigned mates[STEPS];
#pragma unroll
  for (int k = 0; k < STEPS; ++k) mates[k] = same_expert(expert[k], bits);
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const unsigned same = mates[k];
    const int ahead = expert[k] >= 0 ? counts[expert[k]] : 0;
    __syncwarp();
    if (expert[k] >= 0 && lane == __ffs(same) - 1) counts[expert[k]] = (uint16_t)(ahead + __popc(same));
    __syncwarp();
    rank[k] = ahead + __popc(same & ((1u << lane) - 1u));
  }
}
// Counts of the warps before, in the place of every warp's own (a warp adds up an expert's), and of all.
__device__ __forceinline__ void add_up_warps(uint16_t* warp_counts, int pitch, int n_experts, int32_t* totals) {
  const int lane = threadIdx.x & 31;
  for (int e = threadIdx.x >> 5; e < n_experts; e += kSortThreads / 32) {
    const int c = warp_counts[lane * pitch + e];
    int sum = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(kAll, sum, o);
      if (lane >= o) sum += u;
    }
    warp_counts[lane * pitch + e] = (uint16_t)(sum - c);
    if (lane == 31) totals[e] = sum;
  }
}

// All choices by one cluster, STEPS of them in a thread's registers.
template <typename I, int STEPS>
__global__ void __launch_bounds__(kSortThreads) sort_cluster_kernel(const __grid_constant__ SortParams p) {
  extern __shared__ uint16_t warp_counts[];   // [32][pitch]
  __shared__ int32_t totals[kMaxSortExperts], base[kMaxSortExperts], warp_total[32];
  const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, blocks = (int)gridDim.x;
  for (int i = tid; i < 16 * p.pitch; i += kSortThreads) reinterpret_cast<uint32_t*>(warp_counts)[i] = 0u;
  grid_dependency_wait();
  grid_launch_dependents();
  const long long begin = (long long)blockIdx.x * p.share, end = begin + p.share < p.count ? begin + p.share : p.count;
  const long long from = begin + warp * (32 * STEPS) + lane;
  int expert[STEPS], rank[STEPS];
#pragma unroll
  for (int k = 0; k < STEPS; ++k) expert[k] = from + 32 * k < end ? expert_of<I>(p.experts, from + 32 * k, p.n_experts) : -1;
  __syncthreads();
  rank_choices<STEPS>(expert, rank, warp_counts + warp * p.pitch, p.n_experts);
  __syncthreads();
  add_up_warps(warp_counts, p.pitch, p.n_experts, totals);
  cluster.sync();
  int total = 0, before = 0;
  if (tid < p.n_experts) {
#pragma unroll
    for (int b = 0; b < kSortCluster; ++b)
      if (b < blocks) {
        const int c = *cluster.map_shared_rank(totals + tid, b);
        total += c;
        before += b < (int)blockIdx.x ? c : 0;
      }
  }
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  const int first = sum_before(total, warp_total);
  if (tid < p.n_experts) base[tid] = first + before;
  if (blockIdx.x == 0) {
    if (tid < p.n_experts) p.offsets[tid] = first;
    if (tid == p.n_experts - 1) p.offsets[p.n_experts] = first + total;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const long long i = from + 32 * k;
    if (i < end) p.position[i] = expert[k] >= 0 ? base[expert[k]] + warp_counts[warp * p.pitch + expert[k]] + rank[k] : -1;
  }
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");   // (no CTA leaves while others read its counts)
}

template <typename I>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const __grid_constant__ SortParams p) {
  __shared__ int32_t counts[kMaxSortExperts];
  grid_dependency_wait();
  grid_launch_dependents();
  const long long begin = (long long)blockIdx.x * p.share, end = begin + p.share < p.count ? begin + p.share : p.count;
  count_choices<I>(p, begin, end, counts);
  for (int e = threadIdx.x; e < p.n_experts; e += blockDim.x) p.table[(long long)blockIdx.x * p.n_experts + e] = counts[e];
}

template <typename I>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const __grid_constant__ SortParams p) {
  extern __shared__ uint16_t warp_counts[];   // [32][pitch]
  __shared__ int32_t base[kMaxSortExperts];   // rows of the experts before, and of this expert's choices in blocks and tiles before
  __shared__ int32_t warp_total[32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long begin = (long long)blockIdx.x * p.share, end = begin + p.share < p.count ? begin + p.share : p.count;
  int total = 0, before = 0;
  if (tid < p.n_experts) {
#pragma unroll 8
    for (int b = 0; b < (int)gridDim.x; ++b) {
      const int c = p.table[(long long)b * p.n_experts + tid];
      total += c;
      before += b < (int)blockIdx.x ? c : 0;
    }
  }
  const int first = sum_before(total, warp_total);
  if (tid < p.n_experts) base[tid] = first + before;
  if (blockIdx.x == 0) {
    if (tid < p.n_experts) p.offsets[tid] = first;
    if (tid == p.n_experts - 1) p.offsets[p.n_experts] = first + total;
  }
  uint16_t* counts = warp_counts + warp * p.pitch;
  for (long long tile = begin; tile < end; tile += kSortTile) {
    for (int i = tid; i < 16 * p.pitch; i += kSortThreads) reinterpret_cast<uint32_t*>(warp_counts)[i] = 0u;
    __syncthreads();
    int expert[kSortSteps], rank[kSortSteps];
    const long long from = tile + (long long)warp * (32 * kSortSteps) + lane;
#pragma unroll
    for (int k = 0; k < kSortSteps; ++k) expert[k] = from + 32 * k < end ? expert_of<I>(p.experts, from + 32 * k, p.n_experts) : -1;
    rank_choices<kSortSteps>(expert, rank, counts, p.n_experts);
    __syncthreads();
    add_up_warps(warp_counts, p.pitch, p.n_experts, reinterpret_cast<int32_t*>(warp_counts + 32 * p.pitch));
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortSteps; ++k) {
      const long long i = from + 32 * k;
      if (i < end) p.position[i] = expert[k] >= 0 ? base[expert[k]] + counts[expert[k]] + rank[k] : -1;
    }
    __syncthreads();
    for (int e = tid; e < p.n_experts; e += kSortThreads) base[e] += reinterpret_cast<int32_t*>(warp_counts + 32 * p.pitch)[e];
    __syncthreads();
  }
}

// Blocks of a sort that one cluster does not hold, and the choices of one.
inline int sort_blocks(long long count, int sms) {
  const long long tiles = (count + kSortTile - 1) / kSortTile;
  return (int)(tiles < 1 ? 1 : (tiles < sms ? tiles : sms));
}
inline long long sort_share(long long count, int blocks) {
  const long long tiles = (count + kSortTile - 1) / kSortTile;
  return (tiles + blocks - 1) / blocks * kSortTile;
}
constexpr int kMaxSortBlocks = 256;

// ------------------------------------------------------------------------------------------ rows of tokens
constexpr int kRowThreads = 256;
static_assert(VOID_MOST_FEATURES == 65535 * kRowThreads * 4 - 8, "blocks along a row of fp32 that lies anyhow");
// 16-byte pieces of a row that one thread holds at a time.
template <bool WIDE>
constexpr int kHeld = WIDE ? 2 : 1;
// Choices that the sort's own block is not worth a launch for: every warp ranks its token's choices by counting, and one block counts what comes before every
// expert, eight experts at a time, so that the form's time grows with either number.  us of the one launch, in graphs (2048 bf16 features): 32 choices of 64
// experts 3.5, 128 5.1, 256 8.2; 512 choices of 8 3.6, 64 5.4, 128 7.4, 192 9.4; 1024 of 8 5.3, 32 6.5, 64 8.0, 256 17.0, 1024 53.  Behind the sort all of them take 4.5 to 6.7
// (1024 experts 10.7), but called one after another 8.3, for the host has two launches to make (one: 6.0).  The border is where the one launch takes as long as that.
constexpr int kFewChoices = 1024;
inline bool few_choices(long long count, int n_experts) { return count <= kFewChoices && 5ll * n_experts + count <= 1280; }

struct RowParams {
  const void* x;            // tokens (dispatch), rows (combine, its gradient)
  long long ldx;
  const void* g;            // combine's gradient: dy
  long long ldg;
  const void* residual;
  long long ldr;
  int residual_elem;
  const void* weights;      // [tokens][top], or null: ones
  int weight_elem;
  const int32_t* position;  // [tokens][top]
  const int32_t* used;      // rows in runs
  long long tokens, rows;   // rows: tokens * top
  int cols, top;
  void* out;                // rows (dispatch, gradient; may be null), tokens (combine)
  long long ldo;
  void* dw;                 // gradient of the weights, of their type, or null
  int zero_rest;
  // dispatch that sorts by itself
  const void* experts;
  int32_t *offsets, *positions;
  int n_experts;
};
// Whether a choice has a row; positions are not trusted.
__device__ __forceinline__ bool has_row(const RowParams& p, int row) { return row >= 0 && row < p.rows; }

// The 16-byte pieces of a row, from column `first` (at most 0) on, whatever address that is: WIDE, rows that lie in 16-byte pieces (first is 0), one
// load each; others from the one or two aligned pieces that hold them, shifted (all threads of a row by the same).  No piece is read that has no byte
// of the row in it; what is not the row's is anything.  In two steps, so that several loads are on their way together: the shift waits for its own.
template <typename T, bool WIDE>
struct Row {
  using Wanted = Piece<T, 16 / sizeof(T)>;
  struct Raw {
    Wanted piece;
  };
  const T* row;
  __device__ __forceinline__ Row(const T* at, int, int) : row(at) {}
  __device__ __forceinline__ void load(Raw& raw, int i) const { raw.piece.load(row + i * (16 / (int)sizeof(T))); }
  __device__ __forceinline__ Wanted get(const Raw& raw) const { return raw.piece; }
};
template <typename T>
struct Row<T, false> {
  using Wanted = Piece<T, 16 / sizeof(T)>;
  struct Raw {
    uint4 u, v;
  };
  const uint4* base;
  int shift, low, high;   // bytes; aligned pieces [low, high) hold the row
  __device__ __forceinline__ Row(const T* row, int first, int cols) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row) + (intptr_t)first * (intptr_t)sizeof(T), start = at & ~(uintptr_t)15;
    base = reinterpret_cast<const uint4*>(start);
    shift = (int)(at & 15u);
    const long long lead = (long long)(reinterpret_cast<uintptr_t>(row) - start);
    low = (int)(lead >> 4);
    high = (int)((lead + (long long)cols * (int)sizeof(T) + 15) >> 4);
  }
  __device__ __forceinline__ void load(Raw& raw, int i) const {
    raw.u = raw.v = make_uint4(0, 0, 0, 0);
    if (i >= low && i < high) raw.u = base[i];
    if (shift != 0 && i + 1 >= low && i + 1 < high) raw.v = base[i + 1];
  }
  __device__ __forceinline__ Wanted get(const Raw& raw) const {
    uint32_t w[8] = {raw.u.x, raw.u.y, raw.u.z, raw.u.w, raw.v.x, raw.v.y, raw.v.z, raw.v.w};
    if (shift & 8) {   // (branches: all threads take the same)
#pragma unroll
      for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
    }
    if (shift & 4) {
#pragma unroll
      for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
    }
    if (sizeof(T) == 2 && (shift & 2)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
    }
    Wanted piece;
    memcpy(piece.v, w, 16);
    return piece;
  }
};
// The pieces of a row that is written begin at its aligned addresses, so the first may lie partly ahead of the row (c < 0), and the last behind it.
template <typename T, bool WIDE>
__device__ __forceinline__ int first_piece(const T* row) {
  return WIDE ? 0 : -(int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
}
template <typename T, bool WIDE>
__device__ __forceinline__ void store_piece(const Piece<T, 16 / sizeof(T)>& piece, T* row, int c, int cols) {
  constexpr int VEC = 16 / (int)sizeof(T);
  if (WIDE || (c >= 0 && c + VEC <= cols)) {
    piece.store(row + c);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (c + e >= 0 && c + e < cols) row[c + e] = piece.v[e];
  }
}

// Zeros in the rows behind the last run, dealt to the launch's blocks; pieces [first, end) of each.
template <typename T, bool WIDE>
__device__ __forceinline__ void zero_rest(const RowParams& p, long long used, int first, int end) {
  constexpr int VEC = 16 / (int)sizeof(T);
  Piece<T, VEC> zero;
#pragma unroll
  for (int e = 0; e < VEC; ++e) zero.set(e, 0.0f);
  for (long long r = (used < 0 ? 0 : used) + blockIdx.x; r < p.rows; r += gridDim.x) {
    T* row = reinterpret_cast<T*>(p.out) + r * p.ldo;
    for (int i = first + threadIdx.x; i < end; i += kRowThreads) {
      const int c = first_piece<T, WIDE>(row) + i * VEC;
      if (c < p.cols) store_piece<T, WIDE>(zero, row, c, p.cols);
    }
  }
}

// Memory bounds it: 8192 x 4096 bf16 to four experts each 54 us behind the sort, 336 MB at 6.2 TB/s; rows that lie anyhow (4095) 78.
// Token by token, so that x is read once; a token's copies go where its choices were sorted to.  blockIdx.y: part of the columns.
// SORT (few choices): the rows are not known yet, each is the number of choices that come before it.
template <typename T, bool WIDE, typename I, bool SORT>
__global__ void __launch_bounds__(kRowThreads) dispatch_kernel(const __grid_constant__ RowParams p) {
  constexpr int VEC = 16 / (int)sizeof(T), U = kHeld<WIDE>;
  __shared__ int32_t ids[SORT ? kFewChoices : 1];
  __shared__ int32_t place[SORT ? kFewChoices : 1];   // of this token's choices
  __shared__ int32_t rows_used;
  grid_dependency_wait();
  grid_launch_dependents();
  const int i0 = blockIdx.y * (kRowThreads * U);   // the block's pieces
  const T* x = reinterpret_cast<const T*>(p.x);
  T* out = reinterpret_cast<T*>(p.out);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if constexpr (SORT) {
    for (int i = threadIdx.x; i < (int)p.rows; i += kRowThreads) ids[i] = expert_of<I>(p.experts, i, p.n_experts);
    if (threadIdx.x == 0) rows_used = 0;
    __syncthreads();
    if (warp == 0) {
      int n = 0;
      for (int i = lane; i < (int)p.rows; i += 32) n += ids[i] >= 0;
      n = __reduce_add_sync(kAll, n);
      if (lane == 0) rows_used = n;
    }
    if (blockIdx.x == 0 && blockIdx.y == 0) {
      for (int e = warp; e <= p.n_experts; e += kRowThreads / 32) {
        int n = 0;
        for (int i = lane; i < (int)p.rows; i += 32) n += ids[i] >= 0 && ids[i] < e;
        n = __reduce_add_sync(kAll, n);
        if (lane == 0) p.offsets[e] = n;
      }
    }
  }
  for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    typename Row<T, WIDE>::Raw raw[U];
    if constexpr (WIDE) {   // (else every copy's pieces are others)
      const Row<T, WIDE> token(x + t * p.ldx, 0, p.cols);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kRowThreads + threadIdx.x;
        if (i * VEC < p.cols) token.load(raw[u], i);
      }
    }
    if constexpr (SORT) {
      __syncthreads();
      for (int j = warp; j < p.top; j += kRowThreads / 32) {
        const int me = (int)t * p.top + j, e = ids[me];
        int n = 0;
        for (int i = lane; i < (int)p.rows; i += 32) n += ids[i] >= 0 && (ids[i] < e || (ids[i] == e && i < me));
        n = __reduce_add_sync(kAll, n);
        if (lane == 0) {
          place[j] = e >= 0 ? n : -1;
          if (blockIdx.y == 0) p.positions[me] = place[j];
        }
      }
      __syncthreads();
    }
    for (int j = 0; j < p.top; ++j) {
      const int row = SORT ? place[j] : p.position[t * p.top + j];
      if (!has_row(p, row)) continue;
      T* to = out + (long long)row * p.ldo;
      const int first = first_piece<T, WIDE>(to);
      const Row<T, WIDE> token(x + t * p.ldx, first, p.cols);
      if constexpr (!WIDE) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * kRowThreads + threadIdx.x;
          if (first + i * VEC < p.cols) token.load(raw[u], i);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = first + (i0 + u * kRowThreads + threadIdx.x) * VEC;
        if (c < p.cols) store_piece<T, WIDE>(token.get(raw[u]), to, c, p.cols);
      }
    }
  }
  if (p.zero_rest) {
    if constexpr (SORT) __syncthreads();
    zero_rest<T, WIDE>(p, SORT ? rows_used : *p.used, i0, i0 + kRowThreads * U);
  }
}

constexpr int kTogether = 4;   // rows of a token whose loads are in flight together

// Memory bounds it: 8192 x 4096 bf16, four rows a token, 57.5 us, 5.8 TB/s.  Rows that lie anyhow (4095) 101, element by element 197; of 16-bit elements two rows
// at a time, four take registers that warps in flight need (124).

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kRowThreads) combine_kernel(const __grid_constant__ RowParams p) {
  constexpr int VEC = 16 / (int)sizeof(T), U = kHeld<WIDE>, TOGETHER = WIDE || sizeof(T) == 4 ? kTogether : 2;
  grid_dependency_wait();
  grid_launch_dependents();
  const int i0 = blockIdx.y * (kRowThreads * U);
  const T* ys = reinterpret_cast<const T*>(p.x);
  T* out = reinterpret_cast<T*>(p.out);
  for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    T* to = out + t * p.ldo;
    const int first = first_piece<T, WIDE>(to);
    float sum[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[u][e] = 0.0f;
    for (int j0 = 0; j0 < p.top; j0 += TOGETHER) {
      int row[TOGETHER];
      float w[TOGETHER];
#pragma unroll
      for (int k = 0; k < TOGETHER; ++k) {
        const bool in = j0 + k < p.top;
        row[k] = in ? p.position[t * p.top + j0 + k] : -1;
        if (!has_row(p, row[k])) row[k] = -1;
        w[k] = in && p.weights != nullptr ? element(p.weights, p.weight_elem, t * p.top + j0 + k) : 1.0f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kRowThreads + threadIdx.x;
        if (first + i * VEC >= p.cols) continue;
        typename Row<T, WIDE>::Raw raw[TOGETHER];
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
          if (row[k] >= 0) Row<T, WIDE>(ys + (long long)row[k] * p.ldx, first, p.cols).load(raw[k], i);
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
          if (row[k] >= 0) {   // (a dropped choice's weight may be anything)
            const Piece<T, VEC> piece = Row<T, WIDE>(ys + (long long)row[k] * p.ldx, first, p.cols).get(raw[k]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[u][e] = fmaf(w[k], piece.get(e), sum[u][e]);
          }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kRowThreads + threadIdx.x, c = first + i * VEC;
      if (c >= p.cols) continue;
      if (p.residual != nullptr) {
        if (p.residual_elem == VOID_ELEM_F32 && sizeof(T) != 4) {
          const float* r = reinterpret_cast<const float*>(p.residual) + t * p.ldr + c;
          if constexpr (WIDE) {
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
              const float4 v = *reinterpret_cast<const float4*>(r + e);
              sum[u][e] += v.x; sum[u][e + 1] += v.y; sum[u][e + 2] += v.z; sum[u][e + 3] += v.w;
            }
          } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
              if (c + e >= 0 && c + e < p.cols) sum[u][e] += r[e];
          }
        } else {
          const Row<T, WIDE> residual(reinterpret_cast<const T*>(p.residual) + t * p.ldr, first, p.cols);
          typename Row<T, WIDE>::Raw raw;
          residual.load(raw, i);
          const Piece<T, VEC> r = residual.get(raw);
#pragma unroll
          for (int e = 0; e < VEC; ++e) sum[u][e] += r.get(e);
        }
      }
      Piece<T, VEC> y;
#pragma unroll
      for (int e = 0; e < VEC; ++e) y.set(e, sum[u][e]);
      store_piece<T, WIDE>(y, to, c, p.cols);
    }
  }
}

// A block per token: dy is read once (and again from the first cache for more than four choices), the rows of its choices meet it.  8192 x 4096 bf16, four
// rows a token, 93 us, 6.5 TB/s.  Rows that lie anyhow (not WIDE) are taken one by one, each with its own pieces (4095: 178; with two pieces of a row on their way
// 267 to 353, for their registers).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kRowThreads, WIDE ? 4 : 5) combine_grad_kernel(const __grid_constant__ RowParams p) {
  constexpr int VEC = 16 / (int)sizeof(T), TOGETHER = kTogether;
  __shared__ float part[TOGETHER][kRowThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const T *ys = reinterpret_cast<const T*>(p.x), *g = reinterpret_cast<const T*>(p.g);
  T* out = reinterpret_cast<T*>(p.out);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    for (int j0 = 0; j0 < p.top; j0 += TOGETHER) {
      int row[TOGETHER];
      float w[TOGETHER], dot[TOGETHER];
#pragma unroll
      for (int k = 0; k < TOGETHER; ++k) {
        const bool in = j0 + k < p.top;
        row[k] = in ? p.position[t * p.top + j0 + k] : -1;
        if (!has_row(p, row[k])) row[k] = -1;
        w[k] = in && p.weights != nullptr ? element(p.weights, p.weight_elem, t * p.top + j0 + k) : 1.0f;
        dot[k] = 0.0f;
      }
      auto store_grad = [&](const Piece<T, VEC>& d, int k, int c) {
        Piece<T, VEC> q;
#pragma unroll
        for (int e = 0; e < VEC; ++e) q.set(e, w[k] * d.get(e));
        store_piece<T, WIDE>(q, out + (long long)row[k] * p.ldo, c, p.cols);
      };
      if constexpr (WIDE) {
#pragma unroll 2
        for (int c = (int)threadIdx.x * VEC; c < p.cols; c += kRowThreads * VEC) {
          Piece<T, VEC> d, y[TOGETHER];
          d.load(g + t * p.ldg + c);
          if (p.dw != nullptr) {
#pragma unroll
            for (int k = 0; k < TOGETHER; ++k)
              if (row[k] >= 0) y[k].load(ys + (long long)row[k] * p.ldx + c);
          }
#pragma unroll
          for (int k = 0; k < TOGETHER; ++k) {
            if (row[k] < 0) continue;
            if (p.dw != nullptr) {
#pragma unroll
              for (int e = 0; e < VEC; ++e) dot[k] = fmaf(d.get(e), y[k].get(e), dot[k]);
            }
            if (out != nullptr) store_grad(d, k, c);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k) {
          if (row[k] < 0) continue;
          const T* from = ys + (long long)row[k] * p.ldx;
          const int first = first_piece<T, WIDE>(out != nullptr ? out + (long long)row[k] * p.ldo : from);
          float sum = 0.0f;
          const Row<T, WIDE> dy(g + t * p.ldg, first, p.cols), y_row(from, first, p.cols);
#pragma unroll 1
          for (int i = threadIdx.x; first + i * VEC < p.cols; i += kRowThreads) {
            typename Row<T, WIDE>::Raw raw_d, raw_y;
            dy.load(raw_d, i);
            if (p.dw != nullptr) y_row.load(raw_y, i);
            const Piece<T, VEC> d = dy.get(raw_d);
            const int c = first + i * VEC;
            if (out != nullptr) store_grad(d, k, c);
            if (p.dw != nullptr) {
              const Piece<T, VEC> y = y_row.get(raw_y);
              if (c >= 0 && c + VEC <= p.cols) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum = fmaf(d.get(e), y.get(e), sum);
              } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                  if (c + e >= 0 && c + e < p.cols) sum = fmaf(d.get(e), y.get(e), sum);
              }
            }
          }
          dot[k] = sum;
        }
      }
      if (p.dw != nullptr) {
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k) {
          const float s = warp_sum(dot[k]);
          if (lane == 0) part[k][warp] = s;
        }
        __syncthreads();
        if (threadIdx.x < TOGETHER && j0 + (int)threadIdx.x < p.top) {
          float s = 0.0f;
#pragma unroll
          for (int i = 0; i < kRowThreads / 32; ++i) s += part[threadIdx.x][i];
          set_element(p.dw, p.weight_elem, t * p.top + j0 + threadIdx.x, s);
        }
        __syncthreads();
      }
    }
  }
  if (out != nullptr && p.zero_rest) zero_rest<T, WIDE>(p, *p.used, 0, (p.cols + VEC - 1) / VEC + 1);
}

// Whether rows of `elem_bytes` elements lie in whole 16-byte pieces.
inline bool in_pieces(const void* at, long long ld, int elem_bytes) { return ((reinterpret_cast<uintptr_t>(at) | (uintptr_t)(ld * elem_bytes)) & 15u) == 0; }

enum class RowOp { Dispatch, DispatchSort32, DispatchSort64, Combine, CombineGrad };
template <typename T, bool WIDE>
cudaError_t launch_rows(RowOp op, const RowParams& p, int sms, cudaStream_t st) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const long long pieces = ((long long)p.cols + VEC - 1) / VEC + (WIDE ? 0 : 1), width = kRowThreads * kHeld<WIDE>;
  const unsigned parts = op == RowOp::CombineGrad ? 1u : (unsigned)((pieces + width - 1) / width);
  const long long most = 64ll * sms;
  const dim3 grid((unsigned)(p.tokens < most ? p.tokens : most), parts);
  switch (op) {
    case RowOp::Dispatch: return launch_pdl(dispatch_kernel<T, WIDE, int32_t, false>, grid, kRowThreads, 0, st, p);
    case RowOp::DispatchSort32: return launch_pdl(dispatch_kernel<T, WIDE, int32_t, true>, grid, kRowThreads, 0, st, p);
    case RowOp::DispatchSort64: return launch_pdl(dispatch_kernel<T, WIDE, int64_t, true>, grid, kRowThreads, 0, st, p);
    case RowOp::Combine: return launch_pdl(combine_kernel<T, WIDE>, grid, kRowThreads, 0, st, p);
    default: return launch_pdl(combine_grad_kernel<T, WIDE>, grid, kRowThreads, 0, st, p);
  }
}
template <typename T>
int rows_of_type(RowOp op, const RowParams& p, bool wide, int sms, cudaStream_t st) {
  return status_of(wide ? launch_rows<T, true>(op, p, sms, st) : launch_rows<T, false>(op, p, sms, st));
}
int rows_launch(RowOp op, RowParams& p, int elem, cudaStream_t st) {
  if (elem < VOID_ELEM_F32 || elem > VOID_ELEM_BF16 || p.tokens < 0 || p.top < 1 || p.cols < 0) return VOID_ERR_BAD_ARG;
  if (p.tokens > 0x7fffffffll / p.top || p.cols > VOID_MOST_FEATURES) return VOID_ERR_TOO_LARGE;
  p.rows = p.tokens * p.top;
  const bool combine = op == RowOp::Combine, grad = op == RowOp::CombineGrad;
  // A matrix has a row per token, or (what lies in runs) one per choice.
  const long long rows_x = combine || grad ? p.rows : p.tokens, rows_out = combine ? p.tokens : p.rows;
  if ((rows_x > 1 && p.x != nullptr && p.ldx < p.cols) || (rows_out > 1 && p.out != nullptr && p.ldo < p.cols) ||
      (p.tokens > 1 && ((grad && p.ldg < p.cols) || (p.residual != nullptr && p.ldr < p.cols))))
    return VOID_ERR_SHAPE;
  if (p.tokens == 0 || (p.cols == 0 && p.dw == nullptr)) return VOID_OK;
  const int es = elem_size(elem);
  if (!lies_on(p.x, es) || !lies_on(p.g, es) || !lies_on(p.out, es) || !lies_on(p.residual, elem_size(p.residual_elem)) || !lies_on(p.weights, elem_size(p.weight_elem)) ||
      !lies_on(p.dw, elem_size(p.weight_elem)) || !lies_on(p.position, 4) || !lies_on(p.used, 4))
    return VOID_ERR_ALIGN;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  bool wide = p.cols % (16 / es) == 0 && (p.x == nullptr || in_pieces(p.x, p.ldx, es)) && (p.out == nullptr || in_pieces(p.out, p.ldo, es));
  if (grad) wide = wide && in_pieces(p.g, p.ldg, es);
  if (p.residual != nullptr) wide = wide && in_pieces(p.residual, p.ldr, elem_size(p.residual_elem));
  if (elem == VOID_ELEM_F32) return rows_of_type<float>(op, p, wide, dev.sms, st);
  return elem == VOID_ELEM_F16 ? rows_of_type<__half>(op, p, wide, dev.sms, st) : rows_of_type<__nv_bfloat16>(op, p, wide, dev.sms, st);
}

template <typename I, int STEPS>
int launch_sort_cluster(SortParams p, cudaStream_t st) {
  int blocks = 1;
  while ((long long)blocks * kSortThreads * STEPS < p.count) blocks *= 2;
  p.share = (long long)kSortThreads * STEPS;
  const int smem = 32 * p.pitch * 2;
  if (ensure_smem(reinterpret_cast<const void*>(sort_cluster_kernel<I, STEPS>), smem) != 0) return VOID_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)blocks;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return status_of(cudaLaunchKernelEx(&cfg, sort_cluster_kernel<I, STEPS>, p));
}
template <typename I>
int sort_of_index(SortParams p, void* ws, size_t ws_bytes, int sms, cudaStream_t st) {
  p.pitch = 2 * ((p.n_experts + 1) / 2 | 1);   // an odd number of words: a warp adds up a column without conflicts
  if (p.count <= kSortCluster * kSortThreads) return launch_sort_cluster<I, 1>(p, st);
  if (p.count <= kMostInCluster) return launch_sort_cluster<I, kSortSteps>(p, st);
  const int blocks = sort_blocks(p.count, sms < kMaxSortBlocks ? sms : kMaxSortBlocks), smem = 32 * p.pitch * 2 + 4 * p.n_experts;
  p.share = sort_share(p.count, blocks);
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 3u) != 0 || ws_bytes < (size_t)blocks * p.n_experts * 4) return VOID_ERR_WORKSPACE;
  p.table = reinterpret_cast<int32_t*>(ws);
  const cudaError_t rc = launch_pdl(sort_count_kernel<I>, blocks, kSortThreads, 0, st, p);
  if (rc != cudaSuccess) return VOID_ERR_CUDA;
  if (ensure_smem(reinterpret_cast<const void*>(sort_place_kernel<I>), smem) != 0) return VOID_ERR_CUDA;
  return status_of(launch_pdl(sort_place_kernel<I>, blocks, kSortThreads, smem, st, p));
}
int sort_launch(const SortParams& p, int index_bytes, void* ws, size_t ws_bytes, cudaStream_t st) {
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  return index_bytes == 4 ? sort_of_index<int32_t>(p, ws, ws_bytes, dev.sms, st) : sort_of_index<int64_t>(p, ws, ws_bytes, dev.sms, st);
}
// The arguments of a sort, or why not.
int check_sort(const void* experts, int32_t index_bytes, int64_t count, int32_t n_experts, const int32_t* offsets, const int32_t* position) {
  if (n_experts < 1 || count < 0 || (index_bytes != 4 && index_bytes != 8) || offsets == nullptr) return VOID_ERR_BAD_ARG;
  if (count > 0 && (experts == nullptr || position == nullptr)) return VOID_ERR_BAD_ARG;
  if (n_experts > kMaxSortExperts || count > 0x7fffffffll) return VOID_ERR_TOO_LARGE;
  if (!lies_on(experts, index_bytes) || !lies_on(offsets, 4) || !lies_on(position, 4)) return VOID_ERR_ALIGN;
  return VOID_OK;
}

}  // namespace

}  // namespace vb

extern "C" {

int void_route(const void* scores, int32_t elem, int64_t lds, int64_t rows, int32_t n_experts, int32_t top_k, int32_t normalize, int32_t* experts,
               float* weights, void_stream_t stream) {
  vb::RouteParams p = {};
  p.scores = scores; p.lds = lds; p.rows = rows; p.experts = n_experts; p.top = top_k; p.normalize = normalize; p.chosen = experts; p.weights = weights;
  return vb::route_launch<false>(p, elem, reinterpret_cast<cudaStream_t>(stream));
}
int void_route_grad(const void* scores, int32_t elem, int64_t lds, int64_t rows, int32_t n_experts, int32_t top_k, int32_t normalize,
                    const float* g, int64_t ldg, void* dscores, int64_t ldd, void_stream_t stream) {
  vb::RouteParams p = {};
  p.scores = scores; p.lds = lds; p.rows = rows; p.experts = n_experts; p.top = top_k; p.normalize = normalize; p.g = g; p.ldg = ldg; p.ds = dscores; p.ldd = ldd;
  return vb::route_launch<true>(p, elem, reinterpret_cast<cudaStream_t>(stream));
}

size_t void_sort_by_expert_ws_bytes(int64_t count, int32_t n_experts) {
  if (count < 0 || n_experts < 1) return 0;
  return count > vb::kMostInCluster ? (size_t)vb::sort_blocks(count, vb::kMaxSortBlocks) * n_experts * 4 : 0;
}
int void_sort_by_expert(const void* experts, int32_t index_bytes, int64_t count, int32_t n_experts, int32_t* offsets, int32_t* position, void* ws,
                        size_t ws_bytes, void_stream_t stream) {
  const int bad = vb::check_sort(experts, index_bytes, count, n_experts, offsets, position);
  if (bad != VOID_OK) return bad;
  vb::SortParams p = {};
  p.experts = experts; p.count = count; p.n_experts = n_experts; p.offsets = offsets; p.position = position;
  return vb::sort_launch(p, index_bytes, ws, ws_bytes, reinterpret_cast<cudaStream_t>(stream));
}

int void_dispatch(const void* x, int32_t elem, int64_t ldx, int64_t tokens, int32_t cols, const void* experts, int32_t index_bytes, int32_t top_k,
                  int32_t n_experts, int32_t* offsets, int32_t* position, void* out, int64_t ldo, int32_t zero_rest, void* ws, size_t ws_bytes,
                  void_stream_t stream) {
  if (tokens < 0 || top_k < 1 || cols < 0) return VOID_ERR_BAD_ARG;
  if (tokens > 0x7fffffffll / top_k) return VOID_ERR_TOO_LARGE;
  const int bad = vb::check_sort(experts, index_bytes, tokens * top_k, n_experts, offsets, position);
  if (bad != VOID_OK) return bad;
  if (tokens > 0 && cols > 0 && (x == nullptr || out == nullptr)) return VOID_ERR_BAD_ARG;
  const long long count = tokens * top_k;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  vb::RowParams p = {};
  p.x = x; p.ldx = ldx; p.tokens = tokens; p.cols = cols; p.top = top_k; p.out = out; p.ldo = ldo; p.zero_rest = zero_rest;
  p.position = position; p.used = offsets + n_experts;
  if (tokens > 0 && cols > 0 && vb::few_choices(count, n_experts)) {
    p.experts = experts; p.offsets = offsets; p.positions = position; p.n_experts = n_experts;
    return vb::rows_launch(index_bytes == 4 ? vb::RowOp::DispatchSort32 : vb::RowOp::DispatchSort64, p, elem, st);
  }
  const int sorted = void_sort_by_expert(experts, index_bytes, count, n_experts, offsets, position, ws, ws_bytes, stream);
  return sorted != VOID_OK ? sorted : vb::rows_launch(vb::RowOp::Dispatch, p, elem, st);
}

int void_combine(const void* rows, int32_t elem, int64_t ldx, int64_t tokens, int32_t cols, int32_t top_k, const int32_t* position, const void* weights,
                 int32_t weight_elem, const void* residual, int64_t ldr, int32_t residual_elem, void* out, int64_t ldo, void_stream_t stream) {
  if (tokens > 0 && cols > 0 && (rows == nullptr || position == nullptr || out == nullptr)) return VOID_ERR_BAD_ARG;
  if (weight_elem < VOID_ELEM_F32 || weight_elem > VOID_ELEM_BF16) return VOID_ERR_BAD_ARG;
  if (residual != nullptr && residual_elem != elem && residual_elem != VOID_ELEM_F32) return VOID_ERR_BAD_ARG;
  vb::RowParams p = {};
  p.x = rows; p.ldx = ldx; p.tokens = tokens; p.cols = cols; p.top = top_k; p.position = position; p.weights = weights; p.weight_elem = weight_elem;
  p.residual = residual; p.ldr = ldr; p.residual_elem = residual_elem; p.out = out; p.ldo = ldo;
  return vb::rows_launch(vb::RowOp::Combine, p, elem, reinterpret_cast<cudaStream_t>(stream));
}

int void_combine_grad(const void* g, int64_t ldg, const void* rows, int64_t ldx, int32_t elem, int64_t tokens, int32_t cols, int32_t top_k,
                      const int32_t* position, const int32_t* used_rows, const void* weights, int32_t weight_elem, void* drows, int64_t ldd,
                      void* dweights, void_stream_t stream) {
  if (weight_elem < VOID_ELEM_F32 || weight_elem > VOID_ELEM_BF16) return VOID_ERR_BAD_ARG;
  if (tokens > 0 && (position == nullptr || used_rows == nullptr || (cols > 0 && (g == nullptr || (dweights != nullptr && rows == nullptr)))))
    return VOID_ERR_BAD_ARG;
  if (drows == nullptr && dweights == nullptr) return VOID_OK;
  vb::RowParams p = {};
  p.x = rows; p.ldx = ldx; p.g = g; p.ldg = ldg; p.tokens = tokens; p.cols = cols; p.top = top_k; p.position = position; p.used = used_rows;
  p.weights = weights; p.weight_elem = weight_elem; p.out = drows; p.ldo = ldd; p.dw = dweights; p.zero_rest = 1;
  return vb::rows_launch(vb::RowOp::CombineGrad, p, elem, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
