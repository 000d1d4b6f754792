// e4m3 block-scaled products of a single row, dense or of one token's experts: bound by HBM, and by the latency of one call.
//
//   y[n] = sum over blocks g of 128 of  xs[g] ws[n / 128, g] sum_{k in g} xq[k] wq[n, k]
//
// A wave takes whole rows of W, a load instruction 1 KiB of one: lane l holds chunk l (16 numbers) of each 1024 of K, so a block is
// eight lanes.  x stays in registers in the same places, as bfloat16 pairs (which hold e4m3 numbers exactly) with a scale per
// chunk; it is quantised there by every wave, the group's maximum three DPP steps away, so that nothing but the row's sum ever
// leaves a lane: no LDS, no barrier.  Rows go through v_dot2_f32_bf16 (float32 sums), each chunk is scaled, and the lanes add up.
// x is asked for before W: loads come back in order, and x has to be converted while W is on its way.
//
// Measured: 4096 x 4096 6.1 us a call among others (16.8 MB, of which 3.2 us at a large copy's rate; an empty launch takes 1.9),
// 28672 x 4096 25.2 us = 4.7 TB/s.  The few-row kernel, which brings x through LDS and shares K between waves, took 8.7 us for the first.
// Longer K than 8192 stays with it: 16 chunks of x a lane leave too few registers for W (4096 x 14336 18.2 us there).
// One token of six experts of 2048 x 1408: 19 us, in two launches here and the router's (52 MB; 10 us at the copy's rate).
#include "gq_fp8_common.hpp"

namespace gq {

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;

constexpr int kGemvWaves = 4;

// chunk i of a lane: numbers 1024 i + 16 lane ..
template <int X>
struct Raw {
  uint4 v[X == MODEL_F32 ? 4 : X == kXFp8 ? 1 : 2];
  float scale;
};
template <int X>
__device__ __forceinline__ Raw<X> load_raw(const Fp8RowsArgs& p, int64_t row, int k, int K, int groups) {
  Raw<X> r;
  const int at = k < K ? k : 0;  // (K is a multiple of 16)
  if constexpr (X == kXFp8) {
    r.v[0] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.x) + row * p.x_pitch + at);
    r.scale = p.xs[static_cast<int64_t>(at / kFp8Block) * p.x_rows + row];
  } else {
    constexpr int kSize = X == MODEL_F32 ? 4 : 2;
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const char*>(p.x) + (row * K + at) * kSize);
#pragma unroll
    for (int v = 0; v < kSize; ++v) r.v[v] = q[v];
  }
  return r;
}

// sixteen numbers as eight bfloat16 pairs and their scale; zeros past K
struct Chunk {
  uint32_t v[8];
  float scale;
};
__device__ __forceinline__ void widen_chunk(const uint32_t (&q)[4], uint32_t (&out)[8]) {
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    out[2 * v] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[v], 1.0f, false));
    out[2 * v + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[v], 1.0f, true));
  }
}
template <int X>
__device__ __forceinline__ Chunk quantize_chunk(const Raw<X>& r, bool in) {
  Chunk c;
  uint32_t q[4];
  if constexpr (X == kXFp8) {
    q[0] = in ? r.v[0].x : 0u, q[1] = in ? r.v[0].y : 0u, q[2] = in ? r.v[0].z : 0u, q[3] = in ? r.v[0].w : 0u;
    c.scale = r.scale;
  } else {
    float f[16];
#pragma unroll
    for (int h = 0; h < (X == MODEL_F32 ? 4 : 2); ++h) {
      const uint32_t u[4] = {r.v[h].x, r.v[h].y, r.v[h].z, r.v[h].w};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        if constexpr (X == MODEL_F32) {
          f[4 * h + v] = in ? __builtin_bit_cast(float, u[v]) : 0.f;
        } else {
          f[8 * h + 2 * v] = !in ? 0.f : X == MODEL_BF16 ? bf2f(u[v] & 0xffffu) : h2f(u[v] & 0xffffu);
          f[8 * h + 2 * v + 1] = !in ? 0.f : X == MODEL_BF16 ? bf2f(u[v] >> 16) : h2f(u[v] >> 16);
        }
      }
    }
    float top = 0.f;
#pragma unroll
    for (int v = 0; v < 16; ++v) top = fmaxf(top, fp8_magnitude(f[v]));
    top = fmaxf(top, dpp_f<0xB1>(top));   // quad_perm [1,0,3,2]
    top = fmaxf(top, dpp_f<0x4E>(top));   // quad_perm [2,3,0,1]
    top = fmaxf(top, dpp_f<0x141>(top));  // row_half_mirror: the eight lanes of a block
    const uint32_t bits = fp8_scale_bits(top);
    const float inv = fp8_inverse(bits);
#pragma unroll
    for (int v = 0; v < 4; ++v) q[v] = fp8_quad(f[4 * v] * inv, f[4 * v + 1] * inv, f[4 * v + 2] * inv, f[4 * v + 3] * inv);
    c.scale = __builtin_bit_cast(float, bits);
  }
  widen_chunk(q, c.v);
  return c;
}

constexpr uint32_t kNowhere = 0xffffffffu;  // past any buffer's end: reads as zeros, and asks the memory for nothing

// one row's share of this lane
template <int NI>
__device__ __forceinline__ float row_dot(const int4_t (&w)[NI], const Chunk (&x)[NI], const float (&scale)[NI]) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const uint32_t q[4] = {static_cast<uint32_t>(w[i][0]), static_cast<uint32_t>(w[i][1]), static_cast<uint32_t>(w[i][2]), static_cast<uint32_t>(w[i][3])};
    uint32_t b[8];
    widen_chunk(q, b);
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      lo = dot2_bf16(b[v], x[i].v[v], lo);
      hi = dot2_bf16(b[v + 4], x[i].v[v + 4], hi);
    }
    sum = __builtin_fmaf(lo + hi, scale[i], sum);
  }
  return sum;
}

}  // namespace

// R rows of W a set (SILU: R / 2 gate rows and their up rows), the next set in flight while one is computed.
template <int NI, int R, int X, bool SILU>
__global__ __launch_bounds__(64 * kGemvWaves, 2) void fp8_gemv_kernel(Fp8RowsArgs p, int sets) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int K = static_cast<int>(p.K), N = static_cast<int>(p.N), half = N >> 1;
  const int groups = (K + kFp8Block - 1) / kFp8Block, n_blocks = (N + kFp8Block - 1) / kFp8Block;
  const int slot = blockIdx.y;
  Raw<X> raw[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) raw[i] = load_raw<X>(p, p.ids != nullptr ? slot / p.x_div : 0, 1024 * i + 16 * lane, K, groups);
  int e = 0;
  if (p.ids != nullptr) {
    e = p.ids[slot];
    if (e < 0 || e >= p.experts) return;
    e = __builtin_amdgcn_readfirstlane(e);
  }
  const rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w + static_cast<int64_t>(e) * N * p.w_pitch), 0,
                                                          static_cast<int>((N - 1) * static_cast<uint32_t>(p.w_pitch) + K), 0x00027000);
  const rsrc_t s_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p.ws + static_cast<int64_t>(e) * n_blocks * groups), 0,
                                                          n_blocks * groups * 4, 0x00027000);
  constexpr int P = SILU ? 2 : 1;
  const int stride = gridDim.x * kGemvWaves, rows_of = SILU ? half : N;
  int4_t w[R][NI];
  float ws[P][NI];
  // row r of set s; a set's rows (SILU: of each kind) share a block of W
  auto row_of = [&](int s, int r) { return SILU ? s * (R / 2) + (r >> 1) + (r & 1) * half : s * R + r; };
  auto load = [&](int s) {
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int k = 1024 * i + 16 * lane;
        ws[q][i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
            s_rsrc, s < sets && k < K ? static_cast<uint32_t>(row_of(s, q) / kFp8Block * groups + k / kFp8Block) * 4 : kNowhere, 0, 0));
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int n = row_of(s, r);
      const bool there = s < sets && (SILU ? s * (R / 2) + (r >> 1) < half : n < N);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int k = 1024 * i + 16 * lane;
        w[r][i] = __builtin_bit_cast(int4_t, __builtin_amdgcn_raw_buffer_load_b128(
            w_rsrc, there && k < K ? static_cast<uint32_t>(n) * static_cast<uint32_t>(p.w_pitch) + k : kNowhere, 0, 0));
      }
    }
  };
  int s = blockIdx.x * kGemvWaves + wave;
  load(s);
  Chunk x[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) x[i] = quantize_chunk<X>(raw[i], 1024 * i + 16 * lane < K);
  for (; s < sets; s += stride) {
    float sum[R];
#pragma unroll
    for (int q = 0; q < P; ++q) {
      float scale[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i) scale[i] = ws[q][i] * x[i].scale;
#pragma unroll
      for (int r = q; r < R; r += P) sum[r] = row_dot<NI>(w[r], x, scale);
    }
    load(s + stride);
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r] = wave_sum_last(sum[r]);
    if (lane == 63) {
#pragma unroll
      for (int r = 0; r < R / P; ++r) {
        const int n = s * (R / P) + r;
        float o[4] = {SILU ? silu_mul_f32(sum[P * r], sum[P * r + P - 1]) : sum[r], 0.f, 0.f, 0.f};
        if (n < rows_of) fp8_store_one(p, slot, n, rows_of, o[0]);
      }
    }
  }
}

// One token's second expert product and the weighted sum over its experts: a wave an expert, R rows of every W, out [N] in
// out_dtype.
template <int NI, int R>
__global__ __launch_bounds__(512) void fp8_gemv_sum_kernel(Fp8RowsArgs p, const float* __restrict__ weights, int top_k) {
  __shared__ float part[32][R];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int K = static_cast<int>(p.K), N = static_cast<int>(p.N), n0 = blockIdx.x * R;
  const int groups = (K + kFp8Block - 1) / kFp8Block, n_blocks = (N + kFp8Block - 1) / kFp8Block;
  for (int j = wave; j < top_k; j += waves) {
    Raw<MODEL_F32> raw[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) raw[i] = load_raw<MODEL_F32>(p, j, 1024 * i + 16 * lane, K, groups);
    const int e = __builtin_amdgcn_readfirstlane(p.ids[j]);
    const bool known = e >= 0 && e < p.experts;
    const float weight = known ? weights[j] : 0.f;
    const int64_t at = known ? e : 0;
    const rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w + at * N * p.w_pitch), 0,
                                                            static_cast<int>((N - 1) * static_cast<uint32_t>(p.w_pitch) + K), 0x00027000);
    const float* const ws = p.ws + (at * n_blocks + n0 / kFp8Block) * groups;
    int4_t w[R][NI];
    float scale[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int k = 1024 * i + 16 * lane;
      scale[i] = ws[k < K ? k / kFp8Block : 0];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int k = 1024 * i + 16 * lane;
        w[r][i] = __builtin_bit_cast(int4_t, __builtin_amdgcn_raw_buffer_load_b128(
            w_rsrc, n0 + r < N && k < K ? static_cast<uint32_t>(n0 + r) * static_cast<uint32_t>(p.w_pitch) + k : kNowhere, 0, 0));
      }
    Chunk x[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      x[i] = quantize_chunk<MODEL_F32>(raw[i], 1024 * i + 16 * lane < K);
      scale[i] *= x[i].scale;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float sum = wave_sum_last(row_dot<NI>(w[r], x, scale));
      if (lane == 63) part[j][r] = known ? weight * sum : 0.f;
    }
  }
  __syncthreads();
  if (threadIdx.x < R && n0 + static_cast<int>(threadIdx.x) < N) {
    float sum = 0.f;
    for (int j = 0; j < top_k; ++j) sum += part[j][threadIdx.x];
    fp8_store_one(p, 0, n0 + threadIdx.x, N, sum);
  }
}

namespace {

template <int NI, int R, int X, bool SILU>
hipError_t launch_gemv_one(const Fp8RowsArgs& a, hipStream_t s) {
  const int rows_of = static_cast<int>(SILU ? a.N / 2 : a.N), per = SILU ? R / 2 : R, sets = (rows_of + per - 1) / per;
  const int slots = a.ids ? static_cast<int>(a.rows) : 1;
  const int most = 2048 / slots < 1 ? 1 : 2048 / slots, want = (sets + kGemvWaves - 1) / kGemvWaves;
  const int rounds = (want + most - 1) / most;
  note_kernel("fp8_gemv %d KiB, %d rows", NI, R);
  hipLaunchKernelGGL((fp8_gemv_kernel<NI, R, X, SILU>), dim3((want + rounds - 1) / rounds, slots), dim3(64 * kGemvWaves), 0, s, a, sets);
  return hipGetLastError();
}
template <int X, bool SILU>
hipError_t launch_gemv_by_k(const Fp8RowsArgs& a, hipStream_t s) {
  if (a.K <= 1024) return launch_gemv_one<1, 4, X, SILU>(a, s);
  if (a.K <= 2048) return launch_gemv_one<2, 2, X, SILU>(a, s);
  if (a.K <= 4096) return launch_gemv_one<4, 2, X, SILU>(a, s);
  return launch_gemv_one<8, SILU ? 2 : 1, X, SILU>(a, s);
}

}  // namespace

hipError_t launch_fp8_gemv(const Fp8RowsArgs& a, hipStream_t s) {
  if (!fp8_gemv_takes(a.N, a.K, a.w_pitch) || (a.silu && a.N % 4 != 0)) return hipErrorNotSupported;
  if (a.silu) {
    if (a.x_kind == MODEL_BF16) return launch_gemv_by_k<MODEL_BF16, true>(a, s);
    return a.x_kind == MODEL_F16 ? launch_gemv_by_k<MODEL_F16, true>(a, s) : hipErrorNotSupported;
  }
  if (a.x_kind == kXFp8) return launch_gemv_by_k<kXFp8, false>(a, s);
  if (a.x_kind == MODEL_BF16) return launch_gemv_by_k<MODEL_BF16, false>(a, s);
  if (a.x_kind == MODEL_F16) return launch_gemv_by_k<MODEL_F16, false>(a, s);
  return launch_gemv_by_k<MODEL_F32, false>(a, s);
}

hipError_t launch_fp8_gemv_sum(const Fp8RowsArgs& a, const float* weights, int top_k, hipStream_t s) {
  if (!fp8_gemv_takes(a.N, a.K, a.w_pitch) || top_k > 32) return hipErrorNotSupported;
  const int waves = top_k < 8 ? top_k : 8;
  auto go = [&](auto ni, auto r) {
    constexpr int R = decltype(r)::value;
    hipLaunchKernelGGL((fp8_gemv_sum_kernel<decltype(ni)::value, R>), dim3(static_cast<unsigned>((a.N + R - 1) / R)), dim3(64 * waves), 0, s, a,
                       weights, top_k);
    return hipGetLastError();
  };
  note_kernel("fp8_gemv_sum %d experts", top_k);
  if (a.K <= 1024) return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
  if (a.K <= 2048) return go(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
  if (a.K <= 4096) return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
  return go(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
}

}  // namespace gq
