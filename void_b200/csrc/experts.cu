// Linear layers of experts: tokens sorted by expert, each run of tokens multiplied with its own block-sparse weight,
//
//     out_t = act(x_t A_e^T + bias_e)          offsets[e] <= t < offsets[e + 1]
//
// The weights are one packed store, expert behind expert; the runs are cut into chunks of tokens on the device (the host does not
// know the offsets; by a kernel of one block, or for up to 32 experts by each warp for itself, RunTable), and a work item is (chunk, tile row).  The products themselves are those of rowacc.cuh (chunks of 32, 64 or 128
// tokens, B and C as they lie) and, for a handful of tokens per expert, of skinny.cu (chunks of 8).  A chunk never spans two experts: what
// a tile load brings beyond its end belongs to rows of the result that are not stored.
#include "experts.cuh"
#include "pipeline.cuh"

namespace vb {

namespace {

constexpr int kPlanThreads = 1024;

struct Max { __device__ __forceinline__ int operator()(int a, int b) const { return a > b ? a : b; } };
struct Sum { __device__ __forceinline__ int operator()(int a, int b) const { return a + b; } };
// Inclusive scan over the block; `s` has a word per warp.
template <class Op>
__device__ __forceinline__ int block_scan(int v, int* s, Op op) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = op(u, v);
  }
  __syncthreads();   // (the words may still be read by the scan before)
  if (lane == 31) s[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; ++w) v = op(s[w], v);
  return v;
}

// The experts' runs cut into chunks, by one block.  Offsets are not trusted: each is brought into [0, rows] and not below the one before,
// and the status word tells where one had to be.
template <typename O>
__global__ void __launch_bounds__(kPlanThreads) expert_plan_kernel(const O* offsets, int n_experts, int rows, int chunk, PlanView v, int32_t* status) {
  __shared__ int s[32];
  __shared__ int carry[2];   // last bound, chunks so far
  grid_dependency_wait();
  const int tid = threadIdx.x;
  auto bound = [&](int i) {
    const long long o = (long long)offsets[i];
    return o < 0 ? 0 : (o > rows ? rows : (int)o);
  };
  bool bad = false;
  if (tid == 0) {
    carry[0] = v.bounds[0] = bound(0);
    carry[1] = v.chunk_ptr[0] = 0;
    bad = (long long)offsets[0] != v.bounds[0];
  }
  __syncthreads();
  for (int base = 0; base < n_experts; base += blockDim.x) {
    const int e = base + tid, low = carry[0], first = carry[1];
    const int given = e < n_experts ? bound(e + 1) : 0;
    int end = block_scan(given, s, Max());
    if (end < low) end = low;
    // the bound before this one: the neighbour's
    int begin = __shfl_up_sync(0xffffffffu, end, 1);
    __shared__ int last_of_warp[32];
    if ((tid & 31) == 31) last_of_warp[tid >> 5] = end;
    __syncthreads();
    if ((tid & 31) == 0) begin = tid == 0 ? low : last_of_warp[(tid >> 5) - 1];
    const int mine = e < n_experts ? (end - begin + chunk - 1) / chunk : 0;
    const int upto = first + block_scan(mine, s, Sum());
    if (e < n_experts) {
      v.bounds[e + 1] = end;
      v.chunk_ptr[e + 1] = upto;
      bad = bad || (long long)offsets[e + 1] != end;
    }
    __syncthreads();
    if (tid == (int)blockDim.x - 1) {
      carry[0] = end;
      carry[1] = upto;
    }
    __syncthreads();
  }
  if (bad && status != nullptr) atomicCAS(status, 0, kStatusBadOffsets);
  const int total = carry[1];
  if (tid == 0) v.head[0] = total;
  for (int c = tid; c < total && c < v.capacity; c += blockDim.x) {
    int lo = 0, hi = n_experts;   // chunk_ptr[lo] <= c < chunk_ptr[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (v.chunk_ptr[mid] <= c) lo = mid;
      else hi = mid;
    }
    const int n0 = v.bounds[lo] + (c - v.chunk_ptr[lo]) * chunk, end = v.bounds[lo + 1];
    v.chunks[c] = make_int4(lo, n0, n0 + chunk < end ? n0 + chunk : end, 0);
  }
  grid_launch_dependents();
}

int experts_launch(const void_spmm_args* a, const void_epilogue* e, const void_experts* x, int kind, cudaStream_t st) {
  if (a == nullptr || x == nullptr) return VOID_ERR_BAD_ARG;
  if (kind != VOID_KIND_F16 && kind != VOID_KIND_BF16 && kind != VOID_KIND_TF32) return VOID_ERR_BAD_ARG;
  if (a->M < 0 || a->N < 0 || a->K < 0 || a->nbr < 0 || a->nnz < 0 || x->n_experts < 1) return VOID_ERR_BAD_ARG;
  if (x->chunk != 8 && x->chunk != 32 && x->chunk != 64 && x->chunk != kPanelN) return VOID_ERR_BAD_ARG;
  if (a->M == 0 || a->N == 0) return VOID_OK;
  if (a->out == nullptr || a->row_ptr == nullptr || x->plan == nullptr) return VOID_ERR_BAD_ARG;
  const bool given = x->offset_bytes != 0;   // offsets in the place of a plan: the kernels make it, warp by warp
  if (given && ((x->offset_bytes != 4 && x->offset_bytes != 8) || x->n_experts > 32)) return VOID_ERR_BAD_ARG;
  if (a->nnz > 0 && (a->tiles == nullptr || a->tile_cols == nullptr || a->b == nullptr)) return VOID_ERR_BAD_ARG;
  if (a->out_dtype < VOID_OUT_F32 || a->out_dtype > VOID_OUT_BF16 || a->act < VOID_ACT_NONE || a->act > VOID_ACT_SILU) return VOID_ERR_BAD_ARG;
  if (a->transposed != 1 || a->scale_mode != VOID_SCALE_ROW_MEAN || a->row_scale != nullptr || a->col_scale != nullptr || a->bias != nullptr ||
      a->segs != nullptr || a->acc_out != nullptr || a->worker_partials != nullptr || a->trace != nullptr || a->n_peers != 0 || a->tile_terms > 1)
    return VOID_ERR_BAD_ARG;
  if (e != nullptr && (e->residual != nullptr || (e->pre != nullptr && e->ldp < a->M) || e->bias_dtype < VOID_OUT_F32 ||
                       e->bias_dtype > VOID_OUT_BF16))
    return VOID_ERR_BAD_ARG;
  if ((long long)a->nbr * kTile < a->M || a->ldc < a->M) return VOID_ERR_SHAPE;
  const int es = kind == VOID_KIND_TF32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(a->tiles) & 1023u) != 0 || (reinterpret_cast<uintptr_t>(a->b) & 15u) != 0 || (a->ldb & 15) != 0 ||
      a->ldb < (long long)a->K * es || (reinterpret_cast<uintptr_t>(x->plan) & (given ? x->offset_bytes - 1u : 15u)) != 0)
    return VOID_ERR_ALIGN;
  const PlanView v = plan_of(*x, a->N);
  if ((long long)v.capacity * a->nbr > 0x7fffffffll) return VOID_ERR_TOO_LARGE;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  Tail tail = {};
  if (e != nullptr) {
    tail.pre = e->pre;
    tail.ldp = e->ldp;
    tail.bias_dtype = e->bias_dtype;
  }
  SpmmParams p = {};
  p.tiles = a->nnz > 0 ? reinterpret_cast<const uint8_t*>(a->tiles) : nullptr;
  p.tile_cols = a->tile_cols;
  p.row_ptr = a->row_ptr;
  p.nbr = a->nbr;
  p.nbc = a->nbc;
  p.nnz = a->nnz;
  p.N = a->N;
  p.M = a->M;
  p.b_scale = a->b_scale;
  p.row_bias = a->row_bias;
  p.out = a->out;
  p.ldc = a->ldc;
  p.out_dtype = a->out_dtype;
  p.act = a->act;
  p.status = a->status;
  p.wait_limit_ms = (a->test_hooks & 0xffff) ? (a->test_hooks & 0xffff) : kDefaultWaitLimitMs;
  p.drop_group = (a->test_hooks >> 16) & 1;
  const long long items = (long long)v.capacity * a->nbr;
  if (items > 0x3fffffff) return VOID_ERR_TOO_LARGE;
  const bool few = x->chunk == 8;   // another kernel: see skinny.cu
  CUtensorMap tmap;
  memset(&tmap, 0, sizeof(tmap));
  if (a->nnz > 0 && !panel_map_transposed(&tmap, a->b, a->ldb, a->K, a->N, es, x->chunk, !few)) return VOID_ERR_TENSOR_MAP;
  const int panel = x->chunk * kTile * es;
  const ExpertParams experts = {tail, v.head, v.bounds, v.chunks, given ? x->plan : nullptr, x->offset_bytes, x->chunk, x->row_order, x->n_experts, x->zero_rest, panel};
  if (few) return expert_stream_launch(p, experts, kind, tmap, items, dev, st);
  p.np = 1;
  p.terms = 1;
  // The ring takes the shared memory that three CTAs leave each other (as in spmm.cu), in stages of about 20 KB; panels of fewer tokens
  // leave room for more tiles.  The tensor cores read 128 rows behind the start of every panel, the last one's end with the slack.
  const int unit = panel + kTileBytes * es, slack = kPanelBytes * es - panel;
  const int room = dev.smem_per_sm / Mid::CTAS_PER_SM - 1024 - 640 - 1024 - slack;
  p.group = 2 * (kPanelBytes + kTileBytes) * 2 / unit;
  if (p.group > 8) p.group = 8;
  p.stages = room / (unit * p.group);
  if (p.stages > 8) p.stages = 8;
  if (p.stages < Mid::PW) return VOID_ERR_SHAPE;
  p.last_group = p.group;
  p.desc_hi_b = smem_desc_hi(128, 256 * es, kLayoutNone);
  p.desc_hi_a = smem_desc_hi(16, 256 * es, es == 4 ? kLayoutSw128 : kLayoutSw64);
  const uint32_t format = kind == VOID_KIND_TF32 ? 2u : (kind == VOID_KIND_BF16 ? 1u : 0u);
  p.idesc = instr_desc(1, format, format, 0, 0, 128, 32);
  int grid = dev.sms * Mid::CTAS_PER_SM;
  if (items < grid) grid = (int)items;
  const ExpertLaunch l = {grid, p.stages * p.group * unit + slack + 1024, !in_pieces(a->out, a->out_dtype, a->ldc), st, tmap, experts, p};
  return kind == VOID_KIND_TF32 ? launch_experts<VOID_KIND_TF32>(l) : launch_experts<VOID_KIND_F16>(l);
}

}  // namespace

}  // namespace vb

extern "C" {

int64_t void_expert_plan_words(int32_t n_experts, int32_t rows, int32_t chunk) {
  if (n_experts < 1 || rows < 0 || chunk < 1) return 0;
  return vb::plan_table(n_experts) + 4 * vb::plan_capacity(n_experts, rows, chunk);
}

int void_expert_plan(const void* offsets, int32_t offset_bytes, int32_t n_experts, int32_t rows, int32_t chunk, int32_t* plan, int32_t* status,
                     void_stream_t stream) {
  using namespace vb;
  if (offsets == nullptr || plan == nullptr || n_experts < 1 || rows < 0 || chunk < 1 || (offset_bytes != 4 && offset_bytes != 8))
    return VOID_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(plan) & 15u) != 0 || (reinterpret_cast<uintptr_t>(offsets) & (uintptr_t)(offset_bytes - 1)) != 0) return VOID_ERR_ALIGN;
  if (rows > 0x7fffffff - chunk) return VOID_ERR_TOO_LARGE;
  const DeviceInfo dev = device_info();
  if (!dev.ok) return VOID_ERR_CUDA;
  if (dev.cc_major != 10) return VOID_ERR_ARCH;
  void_experts x = {};
  x.plan = plan;
  x.n_experts = n_experts;
  x.chunk = chunk;
  const PlanView v = plan_of(x, rows);
  const int most = v.capacity > n_experts ? v.capacity : n_experts, threads = most >= kPlanThreads ? kPlanThreads : (most + 31) / 32 * 32;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return status_of(offset_bytes == 4 ? launch_pdl(expert_plan_kernel<int32_t>, 1, threads, 0, st, reinterpret_cast<const int32_t*>(offsets), n_experts, rows,
                                                  chunk, v, status)
                                     : launch_pdl(expert_plan_kernel<int64_t>, 1, threads, 0, st, reinterpret_cast<const int64_t*>(offsets), n_experts, rows,
                                                  chunk, v, status));
}

int void_expert_linear(const void_spmm_args* args, const void_epilogue* epilogue, const void_experts* experts, int32_t kind, void_stream_t stream) {
  return vb::experts_launch(args, epilogue, experts, kind, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
