// Shared pieces of the operators on 16-bit weights (float16 or bfloat16, x, W, bias and residual alike): the epilogue that every
// kernel of them ends in, and the matrix instruction by type.
#pragma once

#include "gq_common.hpp"
#include "gq_internal.hpp"

namespace gq {

typedef int int4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// values of the public enum MI355GQ_ACT_*
constexpr int ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4;

// y = act(x W^T + bias) + residual, or (gated, W = gate rows then up rows) y = act(gate + bias) * (up + bias).
struct DenseArgs {
  const uint16_t* x = nullptr;  // [rows, K]
  const uint16_t* w = nullptr;  // [N, K]
  const uint16_t* bias = nullptr;      // [N] or null
  const uint16_t* residual = nullptr;  // [rows, N] or null (not gated)
  void* y = nullptr;            // [rows, N], gated [rows, N / 2]
  int64_t rows = 0, N = 0, K = 0;
  int act = 0, gated = 0, bf16 = 0, out_f32 = 0;
  int vec = 0;      // columns of y a multiple of 8 and y, bias and residual at 16 bytes: whole runs of columns are loaded and stored
  void* workspace = nullptr;
  int64_t workspace_bytes = 0;
};

// x and w at 16 bytes and K a multiple of 8, for the kernels that load eight numbers at a time.
inline bool dense_aligned(const DenseArgs& a) {
  return a.K % 8 == 0 && ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w)) & 15u) == 0;
}

// Up to 16 rows of aligned operands; hipErrorNotSupported beyond.
hipError_t launch_dense_rows(const DenseArgs& a, hipStream_t s);

// Any number of aligned rows; K split over workgroups where the scratch for it is there.
hipError_t launch_dense_tile(const DenseArgs& a, hipStream_t s);
int64_t dense_tile_workspace_bytes(int64_t rows, int64_t N, int64_t K);

// One expert layer on up to kMoeTokens tokens, see mi355gq_dense_moe.
constexpr int kMoeTokens = 64;
struct DenseMoeArgs {
  const uint16_t* x = nullptr;    // [T, hidden]
  const uint16_t* w13 = nullptr;  // [experts, 2 inter, hidden]
  const uint16_t* w2 = nullptr;   // [experts, hidden, inter]
  uint16_t* out = nullptr;        // [T, hidden]
  const void* logits = nullptr;   // [T, experts] in logits_dtype
  const float* score_bias = nullptr;
  int T = 0, experts = 0, k = 0, hidden = 0, inter = 0, act = 0, bf16 = 0;
  int sigmoid = 0, groups = 1, top_groups = 1, renormalize = 1, logits_dtype = 0;
  float scale = 1.f;
  void* workspace = nullptr;
};
int64_t dense_moe_workspace_bytes(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t k);
hipError_t launch_dense_moe(const DenseMoeArgs& a, hipStream_t s);

// Any sizes and alignments; the kernel of the calls that the others do not take.
hipError_t launch_dense_simple(const DenseArgs& a, hipStream_t s);

// a 16 x 16 tile of float32 sums, W as operand A and x as operand B: lane l holds row l % 16 of x and rows 4 (l / 16) .. + 3 of W
template <bool BF>
__device__ __forceinline__ float4_t dense_mfma(int4_t w, int4_t x, float4_t acc) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), __builtin_bit_cast(bf16x8_t, x), acc, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, w), __builtin_bit_cast(half8_t, x), acc, 0, 0, 0);
}

// 1 / (1 + exp(-v)) by the hardware's exp2 and reciprocal, 1 ulp each: 16-bit results round 2^12 times coarser, float32 ones are
// the sums of products of 16-bit numbers
__device__ __forceinline__ float dense_sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896341f));
}

// v Phi(v).  Phi(-a) = exp(-a^2 / 2) t P(t), t = 1 / (1 + 0.3 a), for a >= 0: the factor behind the exponential is smooth in t, and P is the
// Chebyshev interpolation of degree 7 of it over 0 <= a <= 14, beyond which Phi(-a) is 0 in float32.  t P(t) is good to 4.5e-7 of its value.  The exponential has its
// argument in float32, which adds up to 2^-24 a^2 on the negative side: 1.5e-6 of Phi(-5) in all, 8e-6 of Phi(-12).  (The C library's erfc takes three times the instructions; the epilogue of 2048 x 14336 results of
// a large product is otherwise idle time of its matrix cores.)
__device__ __forceinline__ float dense_gelu(float v) {
  const float a = __builtin_fabsf(v), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, a, 1.0f));
  float p = 0.03622337058186531f;
  p = __builtin_fmaf(p, t, -0.1593545526266098f);
  p = __builtin_fmaf(p, t, 0.20981964468955994f);
  p = __builtin_fmaf(p, t, -0.05664501339197159f);
  p = __builtin_fmaf(p, t, 0.13000500202178955f);
  p = __builtin_fmaf(p, t, 0.09951350837945938f);
  p = __builtin_fmaf(p, t, 0.12081217765808105f);
  p = __builtin_fmaf(p, t, 0.11962586641311646f);
  const float tail = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f) * (t * p);
  return v * (v > 0.f ? 1.0f - tail : tail);
}

__device__ __forceinline__ float dense_gelu_tanh(float v) {
  // v / 2 (1 + tanh(u)) = v / (1 + exp(-2 u)), u = sqrt(2 / pi) (v + 0.044715 v^3)
  return v * dense_sigmoid(1.5957691216057308f * v * __builtin_fmaf(0.044715f * v, v, 1.0f));
}
__device__ __forceinline__ float dense_relu(float v) { return v > 0.f ? v : v != v ? v : 0.f; }
// (one switch for all: `act` is the same for the whole launch)
template <int CNT>
__device__ __forceinline__ void dense_act(float (&o)[CNT], int act) {
  auto all = [&](auto f) {
#pragma unroll
    for (int v = 0; v < CNT; ++v) o[v] = f(o[v]);
  };
  switch (act) {
    case ACT_RELU: return all(dense_relu);
    case ACT_SILU: return all([](float v) { return v * dense_sigmoid(v); });
    case ACT_GELU: return all(dense_gelu);
    case ACT_GELU_TANH: return all(dense_gelu_tanh);
    default: return;
  }
}

// one 16-bit number as float32, and two rounded ones side by side
template <bool BF>
__device__ __forceinline__ float dense_widen(uint32_t h) {
  return BF ? bf2f(static_cast<uint16_t>(h)) : h2f(static_cast<uint16_t>(h));
}
template <bool BF>
__device__ __forceinline__ uint32_t dense_pair(float a, float b) {
  typedef float float2_v __attribute__((ext_vector_type(2)));
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_v{a, b}), bf16x2_dot_t));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_v{a, b}), half2_t));
}

// CNT (4 or 8) neighbouring 16-bit numbers, at 8 (16) bytes, as float32
template <bool BF, int CNT>
__device__ __forceinline__ void dense_load_run(const uint16_t* p, float (&f)[CNT]) {
  uint32_t u[CNT / 2];
  if constexpr (CNT == 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    u[0] = q.x, u[1] = q.y, u[2] = q.z, u[3] = q.w;
  } else {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    u[0] = q.x, u[1] = q.y;
  }
#pragma unroll
  for (int i = 0; i < CNT / 2; ++i) {
    f[2 * i] = dense_widen<BF>(u[i] & 0xffffu);
    f[2 * i + 1] = dense_widen<BF>(u[i] >> 16);
  }
}

// CNT numbers from `from` on, `count` of them there
template <bool BF, int CNT>
__device__ __forceinline__ void dense_add_run(const DenseArgs& a, const uint16_t* from, int count, float (&to)[CNT]) {
  if (a.vec) {
    float f[CNT];
    dense_load_run<BF, CNT>(from, f);
#pragma unroll
    for (int v = 0; v < CNT; ++v) to[v] += f[v];
  } else {
#pragma unroll
    for (int v = 0; v < CNT; ++v)
      if (v < count) to[v] += dense_widen<BF>(from[v]);
  }
}

// The epilogue behind the bias, in float32 with one rounding at its end: CNT (4 or 8) numbers o of row r from column n on; gated: u are the up
// numbers of the same columns.
template <bool BF, int CNT, bool GATED>
__device__ __forceinline__ void dense_finish(const DenseArgs& a, int64_t r, int n, float (&o)[CNT], float (&u)[CNT]) {
  const int cols = static_cast<int>(GATED ? a.N / 2 : a.N), count = cols - n < CNT ? cols - n : CNT;
  const int64_t at = r * cols + n;
  dense_act<CNT>(o, a.act);
  if constexpr (GATED) {
#pragma unroll
    for (int v = 0; v < CNT; ++v) o[v] *= u[v];
  } else if (a.residual) {
    dense_add_run<BF, CNT>(a, a.residual + at, count, o);
  }
  if (a.out_f32) {
    float* y = static_cast<float*>(a.y) + at;
    if (a.vec) {
#pragma unroll
      for (int v = 0; v < CNT; v += 4) *reinterpret_cast<float4_t*>(y + v) = float4_t{o[v], o[v + 1], o[v + 2], o[v + 3]};
    } else {
#pragma unroll
      for (int v = 0; v < CNT; ++v)
        if (v < count) y[v] = o[v];
    }
  } else {
    uint32_t q[CNT / 2];
#pragma unroll
    for (int v = 0; v < CNT / 2; ++v) q[v] = dense_pair<BF>(o[2 * v], o[2 * v + 1]);
    uint16_t* y = static_cast<uint16_t*>(a.y) + at;
    if (a.vec) {
      if constexpr (CNT == 8) *reinterpret_cast<uint4*>(y) = uint4{q[0], q[1], q[2], q[3]};
      else *reinterpret_cast<uint2*>(y) = uint2{q[0], q[1]};
    } else {
#pragma unroll
      for (int v = 0; v < CNT; ++v)
        if (v < count) y[v] = static_cast<uint16_t>(v % 2 ? q[v / 2] >> 16 : q[v / 2]);
    }
  }
}

// ... of sums, with the bias
template <bool BF, int CNT, bool GATED>
__device__ __forceinline__ void dense_store(const DenseArgs& a, int64_t r, int n, float (&o)[CNT], float (&u)[CNT]) {
  if (a.bias) {
    const int cols = static_cast<int>(GATED ? a.N / 2 : a.N), count = cols - n < CNT ? cols - n : CNT;
    dense_add_run<BF, CNT>(a, a.bias + n, count, o);
    if constexpr (GATED) dense_add_run<BF, CNT>(a, a.bias + cols + n, count, u);
  }
  dense_finish<BF, CNT, GATED>(a, r, n, o, u);
}

}  // namespace gq
