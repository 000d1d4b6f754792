// Shared pieces of the 8-bit block-scaled kernels.
//
// An e4m3 group is 128 numbers of a row (activations) or a block of 128 x 128 (weights) and a float32 scale s: the value is
// q s.  The quantisers here take the smallest power of two s with max|x| <= 448 s.  A power of two costs a floating format
// no precision (but for the last octave of its subnormals), makes x / s and q s exact, and so leaves one rounding, the
// one to e4m3, whose result does not depend on how the division is carried out.  The products take any float32 scale.
#pragma once

#include "gq_common.hpp"
#include "gq_internal.hpp"

namespace gq {

constexpr int kFp8Block = 128;

typedef int int4_t __attribute__((ext_vector_type(4)));
typedef int int8_vt __attribute__((ext_vector_type(8)));

// max|x| over the finite numbers of a group -> the bits of its scale: 448 = 1.75 2^8, so a top of 1.f 2^e takes
// 2^(e-8) while 1.f <= 1.75 and 2^(e-7) beyond.  Not below 2^-126, and 1 for a group of zeros.
__device__ __forceinline__ uint32_t fp8_scale_bits(float top) {
  const uint32_t u = __builtin_bit_cast(uint32_t, top);
  const int e = static_cast<int>(u >> 23) - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return top > 0.f ? static_cast<uint32_t>(e < 1 ? 1 : e) << 23 : 0x3f800000u;
}
// 1 / s of such a scale, exact (s lies in 2^-126 .. 2^120)
__device__ __forceinline__ float fp8_inverse(uint32_t scale_bits) {
  return __builtin_bit_cast(float, (254u << 23) - scale_bits);
}
// |x| where it is finite, 0 for an infinity or NaN: those become NaN in e4m3, and the scale is that of the others
__device__ __forceinline__ float fp8_magnitude(float x) {
  const float a = __builtin_fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
// two numbers, already divided by their scale, to e4m3 (nearest, ties to even) in the low half; not finite -> NaN
__device__ __forceinline__ uint32_t fp8_pair(float a, float b) {
  const float nan = __builtin_bit_cast(float, 0x7fc00000u);
  a = __builtin_fabsf(a) <= 448.f ? a : nan;
  b = __builtin_fabsf(b) <= 448.f ? b : nan;
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false)) & 0xffffu;
}
__device__ __forceinline__ uint32_t fp8_quad(float a, float b, float c, float d) {
  return fp8_pair(a, b) | fp8_pair(c, d) << 16;
}

__device__ __forceinline__ float silu_mul_f32(float gate, float up) { return gate / (1.0f + expf(-gate)) * up; }

// the largest of the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ float row_max16(float v) {
  v = fmaxf(v, dpp_f<0xB1>(v));   // quad_perm [1,0,3,2]
  v = fmaxf(v, dpp_f<0x4E>(v));   // quad_perm [2,3,0,1]
  v = fmaxf(v, dpp_f<0x141>(v));  // row_half_mirror
  return fmaxf(v, dpp_f<0x140>(v));  // row_mirror
}

// eight neighbouring numbers of DT (MODEL_F16, MODEL_F32, MODEL_BF16) at a 16-byte boundary as float32
template <int DT>
__device__ __forceinline__ void fp8_load8(const void* p, int64_t i, float (&f)[8]) {
  if constexpr (DT == MODEL_F32) {
    const float4_t* q = reinterpret_cast<const float4_t*>(static_cast<const float*>(p) + i);
    const float4_t a = q[0], b = q[1];
#pragma unroll
    for (int v = 0; v < 4; ++v) f[v] = a[v], f[v + 4] = b[v];
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      f[2 * v] = DT == MODEL_BF16 ? bf2f(u[v] & 0xffffu) : h2f(u[v] & 0xffffu);
      f[2 * v + 1] = DT == MODEL_BF16 ? bf2f(u[v] >> 16) : h2f(u[v] >> 16);
    }
  }
}
// eight numbers of each of 16 neighbouring lanes, a group: its e4m3 numbers of this lane and the bits of its scale
__device__ __forceinline__ uint2 fp8_group(const float (&f)[8], uint32_t* bits) {
  float top = 0.f;
#pragma unroll
  for (int v = 0; v < 8; ++v) top = fmaxf(top, fp8_magnitude(f[v]));
  *bits = fp8_scale_bits(row_max16(top));
  const float inv = fp8_inverse(*bits);
  uint2 q;
  q.x = fp8_quad(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
  q.y = fp8_quad(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
  return q;
}

// Arguments of an e4m3 product y[r, n] = sum over blocks g of xs[g, r] ws[n / 128, g] sum_k xq[r, k] wq[n, k].
struct Fp8Args {
  const uint8_t* x = nullptr;   // [x_rows, K], rows x_pitch bytes apart
  const float* xs = nullptr;    // [ceil(K / 128), x_rows]
  const uint8_t* w = nullptr;   // [experts, N, K], rows w_pitch bytes apart
  const float* ws = nullptr;    // [experts, ceil(N / 128), ceil(K / 128)]
  const void* bias = nullptr;      // [N] in model_dtype, or null
  const void* residual = nullptr;  // [rows, N] in model_dtype, or null
  void* y = nullptr;            // [rows, N] in out_dtype
  const int32_t* indptr = nullptr;       // [experts + 1]: rows indptr[e] .. of expert e; null: one segment of all rows
  const int32_t* x_row_index = nullptr;  // row r reads row x_row_index[r] of x; null: row r
  int64_t rows = 0, x_rows = 0, N = 0, K = 0, x_pitch = 0, w_pitch = 0, experts = 1;
  int model_dtype = 0, out_dtype = 0;
  bool precise = false;  // blocks summed in float32, whatever the output type
  uint8_t* q_out = nullptr;  // see launch_fp8_tile
  float* scale_out = nullptr;
  void* workspace = nullptr;
  int64_t workspace_bytes = 0;
};

// ... of few rows a segment, with what the kernel for them takes besides
constexpr int kXFp8 = 3;  // kind of x: MODEL_F16, MODEL_F32 or MODEL_BF16 (dense [x_rows, K], quantised by the kernel), or e4m3 with its scales
struct Fp8RowsArgs {
  const void* x = nullptr;
  const float* xs = nullptr;
  int64_t x_pitch = 0, x_rows = 0;
  int x_kind = kXFp8;
  const uint8_t* w = nullptr;
  const float* ws = nullptr;
  int64_t w_pitch = 0, N = 0, K = 0, experts = 1;
  const void* bias = nullptr;
  const void* residual = nullptr;
  void* y = nullptr;  // [rows, N]
  int64_t rows = 0;
  const int32_t* indptr = nullptr;       // (launch_fp8_rows) segments as in Fp8Args
  const int32_t* x_row_index = nullptr;
  const int32_t* ids = nullptr;          // (launch_fp8_gemv) [rows] the expert of each row, which reads row r / x_div of x
  int x_div = 1;
  int silu = 0;                          // (launch_fp8_gemv with ids) y [rows, N / 2] = silu(first half) * second half
  int model_dtype = 0, out_dtype = 0;
  int y_aligned = 0;  // y starts at 16 bytes
  uint8_t* q_out = nullptr;  // (launch_fp8_rows on quantised x) silu(first half) * second half quantised, [rows, N / 2] and its scales
  float* scale_out = nullptr;  // [N / 256, rows], instead of y; N / 2 a multiple of 128
};
// What the products take that quantise silu(first half) * second half in their epilogue (q_out), few rows and tiles: whole groups of the
// activation, offsets into W in 32 bits.
inline bool fp8_silu_takes(int64_t N, int64_t w_pitch) {
  return N % (2 * kFp8Block) == 0 && static_cast<uint64_t>(N) * w_pitch < 0xffffffffull;
}
// Sixteen rows of a segment at a time; hipErrorNotSupported where the kernel does not apply.
hipError_t launch_fp8_rows(const Fp8RowsArgs& a, hipStream_t s);
// What the kernels of one row take: a row of K in registers, offsets into W in 32 bits.
inline bool fp8_gemv_takes(int64_t N, int64_t K, int64_t w_pitch) {
  return K % 16 == 0 && K <= 8192 && static_cast<uint64_t>(N) * w_pitch < 0xffffffffull;
}
// One row, or (ids) one row of each expert; hipErrorNotSupported as above.  _sum: the rows' products with their experts' W, weighted
// and added up, y [1, N]; x float32 [top_k, K].
hipError_t launch_fp8_gemv(const Fp8RowsArgs& a, hipStream_t s);
hipError_t launch_fp8_gemv_sum(const Fp8RowsArgs& a, const float* weights, int top_k, hipStream_t s);

// Tiles, on the 8-bit matrix instruction or (precise) in float32 sums; K split over workgroups where the scratch for it is there.
// silu: x [rows, K] times gate and up rows of w (N = 2 I), silu(gate) * up quantised into q_out [rows, I] and its scales
// scale_out [I / 128, rows]; I a multiple of 128.
hipError_t launch_fp8_tile(const Fp8Args& a, hipStream_t s);
int64_t fp8_tile_workspace_bytes(int64_t rows, int64_t N, int64_t K);

// CNT (4 or 8) neighbouring results from column n of row r: bias, residual, one rounding, store.  a: Fp8Args or Fp8RowsArgs.
// vec: y and residual start at 16 bytes and N is a multiple of CNT.
template <int CNT, class Args>
__device__ __forceinline__ void fp8_store(const Args& a, int64_t r, int n, int N, bool vec, float (&o)[CNT]) {
  const int64_t at = r * N + n;
  const int count = N - n < CNT ? N - n : CNT;
  auto add = [&](const void* q, int64_t from) {
#pragma unroll
    for (int v = 0; v < CNT; ++v)
      if (v < count)
        o[v] += a.model_dtype == MODEL_F32    ? static_cast<const float*>(q)[from + v]
                : a.model_dtype == MODEL_BF16 ? bf2f(static_cast<const uint16_t*>(q)[from + v])
                                              : h2f(static_cast<const uint16_t*>(q)[from + v]);
  };
  if (a.bias) add(a.bias, n);
  if (a.residual) add(a.residual, at);
  if (a.out_dtype == MODEL_F32) {
    float* y = static_cast<float*>(a.y) + at;
    if (vec) {
#pragma unroll
      for (int v = 0; v < CNT; v += 4) *reinterpret_cast<float4_t*>(y + v) = float4_t{o[v], o[v + 1], o[v + 2], o[v + 3]};
    } else {
#pragma unroll
      for (int v = 0; v < CNT; ++v)
        if (v < count) y[v] = o[v];
    }
  } else {
    uint32_t h[CNT];
#pragma unroll
    for (int v = 0; v < CNT; ++v) h[v] = a.out_dtype == MODEL_BF16 ? f2bf(o[v]) : f2h(o[v]);
    uint16_t* y = static_cast<uint16_t*>(a.y) + at;
    if (vec) {
      uint32_t u[CNT / 2];
#pragma unroll
      for (int v = 0; v < CNT / 2; ++v) u[v] = h[2 * v] | h[2 * v + 1] << 16;
      if constexpr (CNT == 8) *reinterpret_cast<uint4*>(y) = uint4{u[0], u[1], u[2], u[3]};
      else *reinterpret_cast<uint2*>(y) = uint2{u[0], u[1]};
    } else {
#pragma unroll
      for (int v = 0; v < CNT; ++v)
        if (v < count) y[v] = static_cast<uint16_t>(h[v]);
    }
  }
}

// one result, likewise
template <class Args>
__device__ __forceinline__ void fp8_store_one(const Args& a, int64_t r, int n, int N, float o) {
  const int64_t at = r * N + n;
  auto load = [&](const void* q, int64_t i) {
    return a.model_dtype == MODEL_F32    ? static_cast<const float*>(q)[i]
           : a.model_dtype == MODEL_BF16 ? bf2f(static_cast<const uint16_t*>(q)[i])
                                         : h2f(static_cast<const uint16_t*>(q)[i]);
  };
  if (a.bias) o += load(a.bias, n);
  if (a.residual) o += load(a.residual, at);
  if (a.out_dtype == MODEL_F32) static_cast<float*>(a.y)[at] = o;
  else static_cast<uint16_t*>(a.y)[at] = a.out_dtype == MODEL_BF16 ? f2bf(o) : f2h(o);
}

// eight e4m3 numbers as an operand of the bfloat16 matrix instruction (a bfloat16 holds them exactly)
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8_t fp8_widen(uint32_t lo, uint32_t hi) {
  const bf16x2_dot_t a = __builtin_bit_cast(bf16x2_dot_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
  const bf16x2_dot_t b = __builtin_bit_cast(bf16x2_dot_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
  const bf16x2_dot_t c = __builtin_bit_cast(bf16x2_dot_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
  const bf16x2_dot_t d = __builtin_bit_cast(bf16x2_dot_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// rows of x [rows, cols] (silu_mul: of x [rows, 2 cols], silu(first half) * second half) to e4m3 groups; the q bytes between
// cols and the next multiple of 8 are written as zeros, nothing behind them
hipError_t launch_fp8_quantize(const void* x, int64_t rows, int64_t cols, int model_dtype, bool silu_mul, uint8_t* q,
                               int64_t q_pitch, float* scale, hipStream_t s);
hipError_t launch_fp8_quantize_weight(const void* w, int64_t mats, int64_t N, int64_t K, int model_dtype, uint8_t* q,
                                      int64_t q_pitch, float* scale, hipStream_t s);
hipError_t launch_fp8_dequantize(const uint8_t* q, int64_t q_pitch, const float* scale, int64_t mats, int64_t rows,
                                 int64_t cols, bool row_groups, int out_dtype, void* out, hipStream_t s);

// router logits [T, E] -> weights, ids [T, k]; see mi355gq_moe_gating
struct GatingArgs {
  const void* logits;
  const float* bias;
  int64_t T;
  int E, k, sigmoid, groups, top_groups, renormalize, model_dtype;
  float scale;
  float* weights;
  int32_t* ids;
};
hipError_t launch_moe_gating(const GatingArgs& a, hipStream_t s);
// ids [slots] -> the slots in order of their expert, stable: row_token [slots] (slot / k), slot_row [slots] (-1 for an id
// outside the experts), indptr [E + 1]
hipError_t launch_moe_plan(const int32_t* ids, int64_t slots, int k, int E, int32_t* row_token, int32_t* slot_row,
                           int32_t* indptr, hipStream_t s);
// ... and in the same launch rows of x [rows, cols] (float16 or bfloat16, 16-byte aligned, cols a multiple of 16) to e4m3 groups
hipError_t launch_moe_plan_quantize(const int32_t* ids, int64_t slots, int k, int E, int32_t* row_token, int32_t* slot_row,
                                    int32_t* indptr, const void* x, int64_t rows, int64_t cols, int model_dtype, uint8_t* q, float* scale,
                                    hipStream_t s);
// out[t] = sum over j of weights[t, j] y[slot_row[t k + j]] in float32 (a negative row: nothing); out in model_dtype, float16 or
// bfloat16, H % 8 == 0
hipError_t launch_moe_weighted_sum(const float* y, const int32_t* slot_row, const float* weights, int64_t T, int k, int64_t H, int model_dtype,
                                   void* out, hipStream_t s);

}  // namespace gq
