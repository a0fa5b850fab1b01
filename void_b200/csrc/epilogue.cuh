// Epilogue of the tensor-memory product kernels: raw accumulators of one output column n and a few tile rows m to finished
// values of C (dequantise, bias, activation, conversion), stored directly, through a staging tile, or transposed.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/void_b200.h"
#include "ptx.cuh"

namespace vb {

constexpr int kTile = 32;
constexpr int kTileBytes = 1024;
constexpr int kPanelN = 128;
constexpr int kPanelBytes = kTile * kPanelN;  // 4096

// 1 / (1 + 2^w) with the hardware's exponential and reciprocal (a few ulp together; far inside the path's 1e-3 bar).
__device__ __forceinline__ float sigmoid_exp2(float w) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(w));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
constexpr double kLog2e = 1.4426950408889634074;
// GELU in the tanh form written with a sigmoid, void/fusion.py:38-43: x * 0.5 * (1 + (2 sigmoid(2u) - 1)) = x * sigmoid(2u),
// 2u = 1.5957691216 (x + 0.044715 x^3); the factor log2(e) of the exponential is in the constants.
constexpr float kGelu1 = (float)(-1.5957691216 * kLog2e), kGelu3 = (float)(-1.5957691216 * 0.044715 * kLog2e);
constexpr float kSilu = (float)-kLog2e;
// One value, for the kernels whose epilogue is no loop over registers.
__device__ __forceinline__ float activate(float x, int act) {
  if (act == VOID_ACT_NONE) return x;
  if (act == VOID_ACT_RELU) return fmaxf(x, 0.0f);
  return x * sigmoid_exp2(x * (act == VOID_ACT_GELU ? fmaf(x * x, kGelu3, kGelu1) : kSilu));
}
// The same for PAIRS pairs of values, the choice made once.
__device__ __forceinline__ f32x2 times_sigmoid(f32x2 x, f32x2 w) {
  float a, b;
  unpair(w, a, b);
  return mul2(x, pair(sigmoid_exp2(a), sigmoid_exp2(b)));
}
template <int PAIRS>
__device__ __forceinline__ void activate(f32x2 (&x)[PAIRS], int act) {
  if (act == VOID_ACT_NONE) return;
  if (act == VOID_ACT_GELU) {
#pragma unroll
    for (int k = 0; k < PAIRS; ++k)
      x[k] = times_sigmoid(x[k], mul2(x[k], fma2(mul2(x[k], x[k]), pair(kGelu3, kGelu3), pair(kGelu1, kGelu1))));
  } else if (act == VOID_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < PAIRS; ++k) {
      float a, b;
      unpair(x[k], a, b);
      x[k] = pair(fmaxf(a, 0.0f), fmaxf(b, 0.0f));
    }
  } else {
#pragma unroll
    for (int k = 0; k < PAIRS; ++k) x[k] = times_sigmoid(x[k], mul2(x[k], pair(kSilu, kSilu)));
  }
}
// What an epilogue thread needs to know about C, read from the kernel parameters once.
struct OutDesc {
  void* out;
  long long ldc;
  void* acc_out;
  const float* row_bias;  // [M] added per output row before the activation (linear-layer bias), or null
  int M, N, dtype, act;
};
// Raw accumulators of one output column, matrix rows r0 .. r0 + 2 PAIRS - 1, to finished values: dequantise (floating tiles have
// no row scale), bias, activation.
template <int KIND>
__device__ __forceinline__ f32x2 dequantise(uint32_t a, uint32_t b, f32x2 row_scale, f32x2 cs, f32x2 bias) {
  if (KIND == VOID_KIND_I8) return fma2(mul2(pair(__int2float_rn((int)a), __int2float_rn((int)b)), row_scale), cs, bias);
  const f32x2 x = pair(__uint_as_float(a), __uint_as_float(b));
  return fma2(KIND == VOID_KIND_F8E4M3 ? mul2(x, row_scale) : x, cs, bias);
}
// ACT: whether there may be a row bias or an activation.
template <int PAIRS>
__device__ __forceinline__ void row_bias_activation(const OutDesc& o, int r0, f32x2 (&x)[PAIRS]) {
  if (o.row_bias != nullptr) {
    const int rows = o.M - r0;  // rows left below r0
#pragma unroll
    for (int k = 0; k < PAIRS; ++k)
      x[k] = add2(x[k], pair(2 * k < rows ? o.row_bias[r0 + 2 * k] : 0.0f, 2 * k + 1 < rows ? o.row_bias[r0 + 2 * k + 1] : 0.0f));
  }
  activate<PAIRS>(x, o.act);
}
template <int KIND, int PAIRS, bool ACT>
__device__ __forceinline__ void finished(const OutDesc& o, int r0, const uint32_t* r, float row_scale, float cs, float bias,
                                         float (&v)[2 * PAIRS]) {
  const f32x2 rs2 = pair(row_scale, row_scale), cs2 = pair(cs, cs), bias2 = pair(bias, bias);
  f32x2 x[PAIRS];
#pragma unroll
  for (int k = 0; k < PAIRS; ++k) x[k] = dequantise<KIND>(r[2 * k], r[2 * k + 1], rs2, cs2, bias2);
  if (ACT) row_bias_activation<PAIRS>(o, r0, x);
#pragma unroll
  for (int k = 0; k < PAIRS; ++k) unpair(x[k], v[2 * k], v[2 * k + 1]);
}
// Store eight values of output column n, matrix rows row*32 + m0 .. + 7, after row bias and activation.
__device__ __forceinline__ void store8(const OutDesc& o, int row, int n, int m0, float (&v)[8]) {
  const int r0 = row * kTile + m0;
  const int rows = o.M - r0;
  f32x2 x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = pair(v[2 * k], v[2 * k + 1]);
  row_bias_activation<4>(o, r0, x);
#pragma unroll
  for (int k = 0; k < 4; ++k) unpair(x[k], v[2 * k], v[2 * k + 1]);
  if (o.dtype == VOID_OUT_F16) {
    __half* dst = reinterpret_cast<__half*>(o.out) + (size_t)r0 * o.ldc + n;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < rows) dst[(size_t)k * o.ldc] = __float2half_rn(v[k]);
  } else if (o.dtype == VOID_OUT_BF16) {
    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(o.out) + (size_t)r0 * o.ldc + n;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < rows) dst[(size_t)k * o.ldc] = __float2bfloat16_rn(v[k]);
  } else {
    float* dst = reinterpret_cast<float*>(o.out) + (size_t)r0 * o.ldc + n;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < rows) dst[(size_t)k * o.ldc] = v[k];
  }
}

// Epilogue of eight raw accumulators of one output column: dequantise, bias, activation, store.
template <int KIND>
__device__ __forceinline__ void finish8(const OutDesc& o, int row, int n, int m0, const uint32_t (&r)[8],
                                        float row_scale, float cs, float bias) {
  if (n >= o.N) return;
  if (o.acc_out != nullptr) {
    uint32_t* a = reinterpret_cast<uint32_t*>(o.acc_out) + ((size_t)row * kTile + m0) * o.N + n;
#pragma unroll
    for (int k = 0; k < 8; ++k) a[(size_t)k * o.N] = r[k];
  }
  const f32x2 rs2 = pair(row_scale, row_scale), cs2 = pair(cs, cs), bias2 = pair(bias, bias);
  float v[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) unpair(dequantise<KIND>(r[2 * k], r[2 * k + 1], rs2, cs2, bias2), v[2 * k], v[2 * k + 1]);
  store8(o, row, n, m0, v);
}

// Fast epilogue of sixteen raw accumulators of output column n (tile rows m0 .. m0 + 15) straight to C
// (no raw-accumulator dump, no split row), stores specialised per output type.
template <int KIND, bool ACT = true>
__device__ __forceinline__ void finish16(const OutDesc& o, int row, int n, int m0, const uint32_t* r,
                                         float row_scale, float cs, float bias) {
  if (n >= o.N) return;
  const int r0 = row * kTile + m0;
  const int rows = o.M - r0;
  float v[16];
  finished<KIND, 8, ACT>(o, r0, r, row_scale, cs, bias, v);
  const size_t first = (size_t)r0 * o.ldc + n;
  if (o.dtype == VOID_OUT_F16) {
    __half* dst = reinterpret_cast<__half*>(o.out) + first;
#pragma unroll
    for (int k = 0; k < 16; ++k, dst += o.ldc)
      if (k < rows) *dst = __float2half_rn(v[k]);
  } else if (o.dtype == VOID_OUT_BF16) {
    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(o.out) + first;
#pragma unroll
    for (int k = 0; k < 16; ++k, dst += o.ldc)
      if (k < rows) *dst = __float2bfloat16_rn(v[k]);
  } else {
    float* dst = reinterpret_cast<float*>(o.out) + first;
#pragma unroll
    for (int k = 0; k < 16; ++k, dst += o.ldc)
      if (k < rows) *dst = v[k];
  }
}

// A warp's 32 columns of a tile row of raw accumulators, as fragments (tmem_ld_fragments: lanes are columns), to finished
// 16-bit values in a part of shared memory, rows of 64 bytes whose 16-byte pieces lie as the copy engine's 64-byte swizzle
// has them (piece ^ row / 2 % 4; a part starts on 512 bytes).  cs and bias: those of the lane's own column.
// What bounds an epilogue is the number of its instructions, the sixteen epilogue warps of an SM being in theirs together; a
// thread that owns a column puts 32 halves into shared memory one by one; pairs of rows and matrix stores take a third of it.
// Instructions of a launch and its time, before and now: INT8 16384^2 power-law rows, N = 256, GELU 7.0 M 17.8 us, 5.4 M 14.2;
// bf16 4096 -> 16384, 2048 columns, GELU 57 M 95 us, 41 M 75; INT8 4096^2, 90 %, N = 512 2.67 M, 2.40 M.
template <bool F16>
__device__ __forceinline__ uint32_t half2_bits(f32x2 x) {
  float a, b;
  uint32_t d;
  unpair(x, a, b);
  if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}
template <int KIND, bool ACT>
__device__ __forceinline__ void finish_fragments(const OutDesc& o, int r0, const uint32_t (&lo)[16], const uint32_t (&hi)[16],
                                                 float row_scale, float cs, float bias, bool biased, uint32_t part, int lane) {
  const f32x2 rs2 = pair(row_scale, row_scale);
  f32x2 x[16];   // [group of rows][columns t / 4 + 8 q]
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float c = __shfl_sync(0xffffffffu, cs, 8 * q + (lane >> 2));
    const float b = biased ? __shfl_sync(0xffffffffu, bias, 8 * q + (lane >> 2)) : 0.0f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int k = 4 * g + 2 * (q & 1);
      x[4 * g + q] = dequantise<KIND>(q < 2 ? lo[k] : hi[k], q < 2 ? lo[k + 1] : hi[k + 1], rs2, pair(c, c), pair(b, b));
    }
  }
  if (ACT && o.row_bias != nullptr) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r = r0 + 8 * g + 2 * (lane & 3);
      const f32x2 rb = pair(r < o.M ? o.row_bias[r] : 0.0f, r + 1 < o.M ? o.row_bias[r + 1] : 0.0f);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[4 * g + q] = add2(x[4 * g + q], rb);
    }
  }
  if (ACT) activate<16>(x, o.act);
  const uint32_t at = part + (uint32_t)(lane & 7) * 64u + (uint32_t)(((lane >> 3) ^ ((lane >> 1) & 3)) << 4);
  if (o.dtype == VOID_OUT_F16) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      stmatrix_x4_trans(at + (uint32_t)g * 512u, half2_bits<true>(x[4 * g]), half2_bits<true>(x[4 * g + 1]), half2_bits<true>(x[4 * g + 2]),
                        half2_bits<true>(x[4 * g + 3]));
  } else {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      stmatrix_x4_trans(at + (uint32_t)g * 512u, half2_bits<false>(x[4 * g]), half2_bits<false>(x[4 * g + 1]),
                        half2_bits<false>(x[4 * g + 2]), half2_bits<false>(x[4 * g + 3]));
  }
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, int dtype) {
  if (dtype == VOID_OUT_F16) {
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
// Sixteen consecutive elements of a row-major matrix from `first` on, `cols` of them inside, in whole 32-byte sectors or 16-byte pieces
// where they lie so.  (A sector in two stores goes to L2 twice: bf16 4096^2, 90 %, 4096 tokens, plain 44.2 us and 39.4 in whole sectors,
// with a residual 58.0 and 48.0, keeping the value before the activation too 83 and 66.)
__device__ __forceinline__ void store16_row(void* out, int dtype, size_t first, int cols, const float (&v)[16]) {
  if (dtype == VOID_OUT_F32) {
    float* dst = reinterpret_cast<float*>(out) + first;
    if (cols >= 16 && (reinterpret_cast<uintptr_t>(dst) & 31u) == 0) {
#pragma unroll
      for (int k = 0; k < 16; k += 8) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[k + i]);
        st_global_v8(dst + k, w);
      }
    } else if (cols >= 16 && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
#pragma unroll
      for (int k = 0; k < 16; k += 4) *reinterpret_cast<float4*>(dst + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k < cols) dst[k] = v[k];
    }
  } else {
    uint32_t h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = pack16(v[2 * k], v[2 * k + 1], dtype);
    uint16_t* dst = reinterpret_cast<uint16_t*>(out) + first;
    if (cols >= 16 && (reinterpret_cast<uintptr_t>(dst) & 31u) == 0) {
      st_global_v8(dst, h);
    } else if (cols >= 16 && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(dst + 8) = make_uint4(h[4], h[5], h[6], h[7]);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k < cols) dst[k] = (uint16_t)(h[k >> 1] >> ((k & 1) * 16));
    }
  }
}

// Rows that do not lie in whole 16-byte pieces (a pitch of an odd number of elements): written by the lane that owns it, every element
// of 32 rows would be a store of 32 sectors.  Instead eight lanes exchange words first - w[i] of lane j becomes w[j] of lane i - and then
// write eight words of a row together, four rows at a time.  The kernels that can (kLoose) are others, for the code and the registers
// of it: bf16 4096^2, 90 %, 4096 tokens with a residual takes 46 us, with the code for both 70.
__device__ __forceinline__ void turn8(uint32_t (&w)[8]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 4; s > 0; s >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((i & s) == 0) {
        const bool high = (lane & s) != 0;
        const uint32_t got = __shfl_xor_sync(0xffffffffu, high ? w[i] : w[i + s], s);
        if (high) w[i] = got;
        else w[i + s] = got;
      }
}
__host__ __device__ __forceinline__ bool in_pieces(const void* base, int dtype, long long ld, int bytes = 16) {
  return ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)(ld * (dtype == VOID_OUT_F32 ? 4 : 2))) & (uintptr_t)(bytes - 1)) == 0;
}
// Eight words of each of the warp's rows (lane n's row is n) of an [N, M] matrix, from column c0 on: eight fp32 or sixteen 16-bit values.
// For whole warps.
struct Words8 { uint32_t w[8]; };
__device__ __forceinline__ void store_loose(void* out, int dtype, long long ld, int n, int N, int c0, int M, Words8 x) {
  const int j = threadIdx.x & 7, first = n - j;
  turn8(x.w);
  if (dtype == VOID_OUT_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (first + i < N && c0 + j < M) reinterpret_cast<uint32_t*>(out)[(size_t)(first + i) * (size_t)ld + c0 + j] = x.w[i];
    return;
  }
  const int c = c0 + 2 * j;
  const bool words = in_pieces(out, dtype, ld, 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint16_t* dst = reinterpret_cast<uint16_t*>(out) + (size_t)(first + i) * (size_t)ld + c;
    if (first + i >= N) continue;
    if (words && c + 1 < M) {
      *reinterpret_cast<uint32_t*>(dst) = x.w[i];
    } else {
      if (c < M) dst[0] = (uint16_t)x.w[i];
      if (c + 1 < M) dst[1] = (uint16_t)(x.w[i] >> 16);
    }
  }
}
// (to be turned: the loads can be on their way while something else is done)
__device__ __forceinline__ Words8 load_loose(const void* from, int dtype, long long ld, int n, int N, int c0, int M) {
  const int j = threadIdx.x & 7, first = n - j;
  Words8 x;
  if (dtype == VOID_OUT_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x.w[i] = first + i < N && c0 + j < M ? reinterpret_cast<const uint32_t*>(from)[(size_t)(first + i) * (size_t)ld + c0 + j] : 0u;
  } else {
    const int c = c0 + 2 * j;
    const bool words = in_pieces(from, dtype, ld, 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t* src = reinterpret_cast<const uint16_t*>(from) + (size_t)(first + i) * (size_t)ld + c;
      x.w[i] = 0u;
      if (first + i >= N) continue;
      if (words && c + 1 < M) {
        x.w[i] = *reinterpret_cast<const uint32_t*>(src);
      } else {
        if (c < M) x.w[i] = src[0];
        if (c + 1 < M) x.w[i] |= (uint32_t)src[1] << 16;
      }
    }
  }
  return x;
}
// Sixteen columns from c0 on of the lane's row n of an [N, M] matrix; LOOSE: of the warp's rows, which may lie anyhow.
template <bool LOOSE>
__device__ __forceinline__ void store16_rows(void* out, int dtype, long long ld, int n, int N, int c0, int M, const float (&v)[16]) {
  if constexpr (!LOOSE) {
    if (n < N) store16_row(out, dtype, (size_t)n * (size_t)ld + c0, M - c0, v);
  } else if (dtype == VOID_OUT_F32) {
#pragma unroll
    for (int half = 0; half < 16; half += 8) {
      Words8 x;
#pragma unroll
      for (int i = 0; i < 8; ++i) x.w[i] = __float_as_uint(v[half + i]);
      store_loose(out, dtype, ld, n, N, c0 + half, M, x);
    }
  } else {
    Words8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.w[i] = pack16(v[2 * i], v[2 * i + 1], dtype);
    store_loose(out, dtype, ld, n, N, c0, M, x);
  }
}

// Transposed output (C stored as [N, M], m contiguous): the thread owns output row n and sixteen consecutive
// columns m0 .. m0 + 15 of it, so the values leave in 16-byte stores (LOOSE: for whole warps, C may lie anyhow).  bias_n is the bias of this n, the
// per-m bias (o.row_bias) is the same for every thread of the warp.
template <int KIND, bool ACT = true, bool LOOSE = false>
__device__ __forceinline__ void finish16_tr(const OutDesc& o, int row, int n, int m0, const uint32_t* r,
                                            float row_scale, float cs, float bias_n) {
  const int c0 = row * kTile + m0;   // first output column (a row index of A)
  if (c0 >= o.M || (!LOOSE && n >= o.N)) return;
  float v[16];
  finished<KIND, 8, ACT>(o, c0, r, row_scale, cs, bias_n, v);
  store16_rows<LOOSE>(o.out, o.dtype, o.ldc, n, o.N, c0, o.M, v);
}

// What a linear layer's epilogue may do besides: keep the value before the activation, add a residual behind it.
struct Tail {
  const void* residual;   // [N, M], or null
  void* pre;              // [N, M] of the output's type, or null
  long long ldr, ldp;
  int residual_dtype;
  int bias_dtype;         // type of OutDesc::row_bias: of a layer in training it may be 16 bits
};
__device__ __forceinline__ float f16_value(uint32_t bits, bool f16) {
  return f16 ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16);
}
// A product whose weight is one of several experts', each multiplied with its own run of tokens (B and C transposed): a work item is one
// chunk of an expert's tokens and some of its tile rows, chunks as laid out by expert_plan_kernel (experts.cu).
struct ExpertParams {
  Tail tail;
  const int32_t* head;        // number of chunks
  const int32_t* bounds;      // [experts + 1]: where the experts' runs of tokens begin, and the end of the last
  const int4* chunks;         // expert, first token, token behind the last
  const void* offsets;        // or, for these three: the runs' offsets themselves, of up to 32 experts (RunTable)
  int offset_bytes, chunk;    // of one of them; tokens of a chunk
  const int32_t* row_order;   // [experts][tile rows]: tile row of the k-th row taken, or null for k
  int n_experts, zero_rest;   // zero_rest: tokens outside all runs get zeros
  int panel_bytes;            // of a panel in shared memory (row kernel): as many tokens as a chunk has
};
struct Nothing {};
template <class X>
constexpr bool kExpertsOf = std::is_same<X, ExpertParams>::value;

// The plan of up to 32 experts as a warp makes it for itself, expert e's run and first chunk in lane e, as expert_plan_kernel would: a few
// steps of shuffles for a launch of two or three microseconds.  For whole warps, behind the wait on the kernel before.
struct RunTable {
  int begin, end, first, total;   // tokens; chunks before the run's, chunks in all
  bool bad;                       // the offsets are not as given
  __device__ __forceinline__ RunTable(const ExpertParams& x, int rows) {
    const int lane = threadIdx.x & 31, e = lane < x.n_experts ? lane : x.n_experts - 1;
    auto offset = [&](int i) {
      return x.offset_bytes == 8 ? reinterpret_cast<const long long*>(x.offsets)[i] : (long long)reinterpret_cast<const int32_t*>(x.offsets)[i];
    };
    auto inside = [&](long long o) { return o < 0 ? 0 : (o > rows ? rows : (int)o); };
    const long long from = offset(0), to = offset(e + 1);
    const int low = inside(from);
    end = inside(to);
    if (end < low) end = low;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o && u > end) end = u;
    }
    begin = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) begin = low;
    const int shift = __ffs(x.chunk) - 1, mine = (end - begin + x.chunk - 1) >> shift;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    first = upto - mine;
    total = __shfl_sync(0xffffffffu, upto, 31);
    bad = from != low || to != end;
  }
  // chunk c < total of each lane, as x.chunks has it: the last expert whose first chunk is not behind it
  __device__ __forceinline__ int4 chunk(const ExpertParams& x, int c) const {
    int e = 0;
#pragma unroll 4
    for (int k = 1; k < 32; ++k) {
      const int f = __shfl_sync(0xffffffffu, first, k);
      if (k < x.n_experts && f <= c) e = k;
    }
    const int n0 = __shfl_sync(0xffffffffu, begin, e) + (c - __shfl_sync(0xffffffffu, first, e)) * x.chunk, stop = __shfl_sync(0xffffffffu, end, e);
    return make_int4(e, n0, n0 + x.chunk < stop ? n0 + x.chunk : stop, 0);
  }
};
// Zeros for the tokens in no expert's run, dealt out over the CTAs.  For whole warps.
__device__ __forceinline__ void zero_rest_rows(const OutDesc& o, const ExpertParams& x, int tid, int threads) {
  int before, behind;
  if (x.offsets != nullptr) {
    const RunTable runs(x, o.N);
    before = __shfl_sync(0xffffffffu, runs.begin, 0);
    behind = __shfl_sync(0xffffffffu, runs.end, 31);
  } else {
    before = x.bounds[0];
    behind = x.bounds[x.n_experts];
  }
  const int rest = before + o.N - behind;
  for (int i = blockIdx.x; i < rest; i += gridDim.x) {
    const size_t first = (size_t)(i < before ? i : i - before + behind) * (size_t)o.ldc;
    if (o.dtype == VOID_OUT_F32)
      for (int c = tid; c < o.M; c += threads) reinterpret_cast<float*>(o.out)[first + c] = 0.0f;
    else
      for (int c = tid; c < o.M; c += threads) reinterpret_cast<uint16_t*>(o.out)[first + c] = 0;
  }
}
// Expert e's biases of M each.
__device__ __forceinline__ const float* bias_of_expert(const float* bias, int dtype, int e, int M) {
  return reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(bias) + (size_t)e * (size_t)M * (dtype == VOID_OUT_F32 ? 4u : 2u));
}
// Sixteen consecutive elements of a row, `cols` of them inside, added in fp32.
__device__ __forceinline__ void add16(const void* from, int dtype, size_t first, int cols, float (&v)[16]) {
  if (dtype == VOID_OUT_F32) {
    const float* src = reinterpret_cast<const float*>(from) + first;
    if (cols >= 16 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        const float4 r = *reinterpret_cast<const float4*>(src + k);
        v[k] += r.x; v[k + 1] += r.y; v[k + 2] += r.z; v[k + 3] += r.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k < cols) v[k] += src[k];
    }
  } else {
    const bool f16 = dtype == VOID_OUT_F16;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(from) + first;
    if (cols >= 16 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
      uint32_t w[8];
      if ((reinterpret_cast<uintptr_t>(src) & 31u) == 0) {
        ld_global_v8(src, w);
      } else {
        const uint4 r0 = *reinterpret_cast<const uint4*>(src), r1 = *reinterpret_cast<const uint4*>(src + 8);
        w[0] = r0.x; w[1] = r0.y; w[2] = r0.z; w[3] = r0.w; w[4] = r1.x; w[5] = r1.y; w[6] = r1.z; w[7] = r1.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[2 * k] += f16_value(w[k] & 0xffffu, f16);
        v[2 * k + 1] += f16_value(w[k] >> 16, f16);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k < cols) v[k] += f16_value(src[k], f16);
    }
  }
}
// The same of the lane's row n of an [N, M] matrix; LOOSE: of the warp's rows, which may lie anyhow.
template <bool LOOSE>
__device__ __forceinline__ void add16_rows(const void* from, int dtype, long long ld, int n, int N, int c0, int M, float (&v)[16]) {
  if constexpr (!LOOSE) {
    if (n < N) add16(from, dtype, (size_t)n * (size_t)ld + c0, M - c0, v);
  } else if (dtype == VOID_OUT_F32) {
#pragma unroll
    for (int half = 0; half < 16; half += 8) {
      Words8 x = load_loose(from, dtype, ld, n, N, c0 + half, M);
      turn8(x.w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[half + i] += __uint_as_float(x.w[i]);
    }
  } else {
    const bool f16 = dtype == VOID_OUT_F16;
    Words8 x = load_loose(from, dtype, ld, n, N, c0, M);
    turn8(x.w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[2 * i] += f16_value(x.w[i] & 0xffffu, f16);
      v[2 * i + 1] += f16_value(x.w[i] >> 16, f16);
    }
  }
}
// The residual of COLS columns of a tile row from m0 on, asked for before the accumulators are there: 16-bit ones that lie in whole
// sectors, or (LOOSE) anyhow.
template <int COLS, bool LOOSE = false>
struct Ahead {
  uint32_t w[COLS / 2];
  bool valid;
  __device__ __forceinline__ void load(const OutDesc& o, const Tail& t, int row, int n, int m0 = 0) {
    if constexpr (LOOSE) {
      valid = t.residual != nullptr && t.residual_dtype != VOID_OUT_F32;
      if (!valid) return;
#pragma unroll
      for (int k = 0; k < COLS / 2; k += 8) {
        const Words8 x = load_loose(t.residual, t.residual_dtype, t.ldr, n, o.N, row * kTile + m0 + 2 * k, o.M);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[k + i] = x.w[i];
      }
      return;
    }
    const uint16_t* src = reinterpret_cast<const uint16_t*>(t.residual) + (size_t)n * t.ldr + row * kTile + m0;
    valid = t.residual != nullptr && t.residual_dtype != VOID_OUT_F32 && n < o.N && row * kTile + kTile <= o.M && (reinterpret_cast<uintptr_t>(src) & 31u) == 0;
    if (valid)
#pragma unroll
      for (int k = 0; k < COLS / 2; k += 8) ld_global_v8(src + 2 * k, *reinterpret_cast<uint32_t(*)[8]>(w + k));
  }
};
// The bias of the lane's row of a tile row, asked for before the accumulators are there: behind them, every row would wait for it, and
// while weights are on their way that is a microsecond or two.  bias: the first of the layer's (or the expert's).
__device__ __forceinline__ float bias_of_lane(const float* bias, int dtype, int row, int M) {
  const int m = row * kTile + (int)(threadIdx.x & 31);
  if (bias == nullptr || m >= M) return 0.0f;
  if (dtype == VOID_OUT_F32) return bias[m];
  return f16_value(reinterpret_cast<const uint16_t*>(bias)[m], dtype == VOID_OUT_F16);
}
// Of a z that is kept, ReLU's slope asks the sign.  What fp16 would round to zero keeps it as fp16's smallest number.  A sum that its bias takes to
// nothing becomes -0, which has no slope either, until relu_border_kernel has computed it again.
constexpr float kRoundsToZero = 2.9802322e-8f, kLeast = 5.9604645e-8f;   // 2^-25 (a tie, to even) and 2^-24
__device__ __forceinline__ bool loses_sign(float z) { return z != 0.0f && fabsf(z) <= kRoundsToZero; }
__device__ __forceinline__ float keep_sign(float z, int act, int dtype) {
  return act == VOID_ACT_RELU && dtype == VOID_OUT_F16 && loses_sign(z) ? copysignf(kLeast, z) : z;
}
// (behind a row's store, over what it wrote: replaced before it, the values that the result is made of would take registers of their own, and every
// activation 5 us of 63, bf16 4096^2, 90 %, 4096 tokens)
__device__ __forceinline__ void store16_signs(void* out, size_t first, int cols, const float (&z)[16]) {
#pragma unroll
  for (int k = 0; k < 16; ++k)
    if (k < cols && loses_sign(z[k])) reinterpret_cast<uint16_t*>(out)[first + k] = z[k] > 0.0f ? 0x0001u : 0x8001u;
}
__device__ __forceinline__ float with_bias(float sum, float bias, bool signs) {
  const float z = sum + bias;
  return signs && z == 0.0f && sum != 0.0f ? -0.0f : z;
}
// finish16_tr with the rest of a linear layer: z = dequantised accumulator + bias, kept where asked; act(z) + residual.  For whole
// warps: of_lane is bias_of_lane.  ahead: the residual where it is there already.
template <int KIND, bool LOOSE = false>
__device__ __forceinline__ void finish16_tail(const OutDesc& o, const Tail& t, int row, int n, int m0, const uint32_t* r, float row_scale,
                                              float cs, float bias_n, float of_lane, const uint32_t* ahead = nullptr) {
  const int c0 = row * kTile + m0;
  if (c0 >= o.M) return;
  float v[16];
  finished<KIND, 8, false>(o, c0, r, row_scale, cs, bias_n, v);
  if (o.row_bias != nullptr) {
    if (t.pre != nullptr && o.act == VOID_ACT_RELU) {
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = with_bias(v[k], __shfl_sync(0xffffffffu, of_lane, m0 + k), true);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] += __shfl_sync(0xffffffffu, of_lane, m0 + k);
    }
  }
  if (!LOOSE && n >= o.N) return;
  if (t.pre != nullptr) {
    store16_rows<false>(t.pre, o.dtype, t.ldp, n, o.N, c0, o.M, v);
    if (o.act == VOID_ACT_RELU && o.dtype == VOID_OUT_F16 && n < o.N) store16_signs(t.pre, (size_t)n * (size_t)t.ldp + c0, o.M - c0, v);
  }
  if (o.act != VOID_ACT_NONE) {
    f32x2 x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = pair(v[2 * k], v[2 * k + 1]);
    activate<8>(x, o.act);
#pragma unroll
    for (int k = 0; k < 8; ++k) unpair(x[k], v[2 * k], v[2 * k + 1]);
  }
  if (ahead != nullptr) {
    const bool f16 = t.residual_dtype == VOID_OUT_F16;
    Words8 x;
#pragma unroll
    for (int k = 0; k < 8; ++k) x.w[k] = ahead[k];
    if constexpr (LOOSE) turn8(x.w);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[2 * k] += f16_value(x.w[k] & 0xffffu, f16);
      v[2 * k + 1] += f16_value(x.w[k] >> 16, f16);
    }
  } else if (t.residual != nullptr) {
    add16_rows<LOOSE>(t.residual, t.residual_dtype, t.ldr, n, o.N, c0, o.M, v);
  }
  store16_rows<LOOSE>(o.out, o.dtype, o.ldc, n, o.N, c0, o.M, v);
}

}  // namespace vb
