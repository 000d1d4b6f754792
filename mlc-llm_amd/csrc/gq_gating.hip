// Routing of expert layers: scores, selection in groups of experts, weights; the stable order of the
// slots by expert; the weighted sum over a token's experts.  Small integer and float32 work, bound by latency.
#include "gq_gating.hpp"

namespace gq {

template <int NC, int DT>
__global__ __launch_bounds__(64) void gating_kernel(const void* __restrict__ logits, const float* __restrict__ bias,
                                                    int64_t T, int E, int k, int sigmoid, int groups, int top_groups,
                                                    int group_inv, int renormalize, float scale, int vec,
                                                    float* __restrict__ weights, int32_t* __restrict__ ids) {
  const GateRule rule{bias, E, k, sigmoid, groups, top_groups, group_inv, renormalize, scale};
  __shared__ __attribute__((aligned(16))) GateScratch<NC> lds;
  const int r = threadIdx.x & 31, token = threadIdx.x >> 5;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 2 + token;
  const bool there = at < T;
  const int64_t t = there ? at : T - 1;  // (a token past the end computes the last one's and writes nothing)
  float score[NC];
  gate_load<NC, DT>(logits, t, E, r, vec, score);
  int id;
  const float w = gate_pair<NC>(lds, score, rule, &id);
  if (r < k && there) {
    weights[t * k + r] = w;
    ids[t * k + r] = id;
  }
}

hipError_t launch_moe_gating(const GatingArgs& a, hipStream_t s) {
  const int vec = a.E % 8 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15u) == 0;
  constexpr int64_t kTokensALaunch = int64_t(1) << 26;  // (32 work items each; 2^32 of them would wrap, without an error)
  auto go = [&](auto nc, auto dt) {
    for (int64_t t0 = 0; t0 < a.T; t0 += kTokensALaunch) {
      const int64_t here = a.T - t0 < kTokensALaunch ? a.T - t0 : kTokensALaunch;
      hipLaunchKernelGGL((gating_kernel<decltype(nc)::value, decltype(dt)::value>), dim3(static_cast<unsigned>((here + 1) / 2)), dim3(64), 0, s,
                         static_cast<const char*>(a.logits) + t0 * a.E * (a.model_dtype == MODEL_F32 ? 4 : 2), a.bias, here, a.E, a.k, a.sigmoid,
                         a.groups, a.top_groups, gate_group_inv(a.E, a.groups), a.renormalize, a.scale, vec, a.weights + t0 * a.k, a.ids + t0 * a.k);
    }
  };
  auto by_type = [&](auto nc) {
    if (a.model_dtype == MODEL_F32) go(nc, std::integral_constant<int, MODEL_F32>{});
    else if (a.model_dtype == MODEL_BF16) go(nc, std::integral_constant<int, MODEL_BF16>{});
    else go(nc, std::integral_constant<int, MODEL_F16>{});
  };
  if (a.E <= 64) by_type(std::integral_constant<int, 2>{});
  else if (a.E <= 128) by_type(std::integral_constant<int, 4>{});
  else if (a.E <= 256) by_type(std::integral_constant<int, 8>{});
  else by_type(std::integral_constant<int, 16>{});
  return hipGetLastError();
}

// The slots in the order of their expert, and in slot order within one: a workgroup an expert, each of which reads all ids
// (a few hundred KiB at most, from the L2) and counts those before its own, so no table of counts goes through memory and
// one launch does it.  A wave takes a run of slots, 64 at a time; its offsets come from the waves before it through LDS.
//
// DT: with E workgroups for this, further ones quantise rows of x, which the expert layer needs at the same point; a wave four
// groups of a row at a time.  kPlanOnly: none.
constexpr int kPlanOnly = -1;
template <int DT>
__global__ __launch_bounds__(1024) void moe_plan_kernel(const int32_t* __restrict__ ids, int slots, int k, int E, int per_wave,
                                                        int32_t* __restrict__ row_token, int32_t* __restrict__ slot_row,
                                                        int32_t* __restrict__ indptr, const void* __restrict__ x, int64_t rows, int cols,
                                                        uint8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ int counts[2][16];
  if constexpr (DT != kPlanOnly) {
    if (static_cast<int>(blockIdx.x) >= E) {
      const int runs = (cols + 511) / 512;
      const int64_t at = static_cast<int64_t>(blockIdx.x - E) * (blockDim.x >> 6) + (threadIdx.x >> 6), row = at / runs;
      const int col = static_cast<int>(at - row * runs) * 512 + (threadIdx.x & 63) * 8;
      if (row >= rows) return;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (col < cols) fp8_load8<DT == kPlanOnly ? MODEL_F16 : DT>(x, row * cols + col, f);
      uint32_t bits;
      const uint2 out = fp8_group(f, &bits);
      if (col < cols) *reinterpret_cast<uint2*>(q + row * cols + col) = out;
      if ((threadIdx.x & 15) == 0 && col < cols) scale[static_cast<int64_t>(col / kFp8Block) * rows + row] = __builtin_bit_cast(float, bits);
      return;
    }
  }
  const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int begin = wave * per_wave, end = begin + per_wave < slots ? begin + per_wave : slots;
  int own = 0, before = 0;
  int held[4];  // (asked for together, and kept for the second pass)
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int s0 = begin + 64 * c + lane;
    held[c] = s0 < end ? ids[s0] : -1;
  }
  auto id_of = [&](int c) {
    const int s0 = begin + 64 * c + lane;
    return s0 < end ? ids[s0] : -1;
  };
  auto count = [&](int id) {
    own += __popcll(__ballot(id == e));
    before += __popcll(__ballot(id >= 0 && id < e));
  };
#pragma unroll
  for (int c = 0; c < 4; ++c) count(held[c]);
  for (int c = 4; begin + 64 * c < end; ++c) count(id_of(c));
  if (lane == 0) {
    counts[0][wave] = own;
    counts[1][wave] = before;
  }
  __syncthreads();
  int base = 0, total = 0, first = 0;
  for (int w = 0; w < waves; ++w) {
    base += counts[1][w];
    total += counts[0][w];
    if (w < wave) first += counts[0][w];
  }
  if (threadIdx.x == 0) {
    indptr[e] = base;
    if (e == E - 1) indptr[E] = base + total;
  }
  int at = base + first;
  auto place = [&](int c, int id) {
    const int s = begin + 64 * c + lane;
    const unsigned long long m = __ballot(id == e);
    if (id == e) {
      const int row = at + __popcll(m & ((1ull << lane) - 1ull));
      row_token[row] = s / k;
      slot_row[s] = row;
    } else if (e == 0 && s < end && (id < 0 || id >= E)) {
      slot_row[s] = -1;
    }
    at += __popcll(m);
  };
#pragma unroll
  for (int c = 0; c < 4; ++c) place(c, held[c]);
  for (int c = 4; begin + 64 * c < end; ++c) place(c, id_of(c));
}

template <int DT>
static hipError_t launch_plan(const int32_t* ids, int64_t slots, int k, int E, int32_t* row_token, int32_t* slot_row, int32_t* indptr,
                              const void* x, int64_t rows, int64_t cols, uint8_t* q, float* scale, hipStream_t s) {
  const int n = static_cast<int>(slots);
  const int waves = n >= 4096 ? 16 : n >= 1024 ? 8 : 4;
  const int per_wave = ((n + waves - 1) / waves + 63) / 64 * 64;
  const int64_t more = DT == kPlanOnly ? 0 : (rows * ((cols + 511) / 512) + waves - 1) / waves;
  hipLaunchKernelGGL(moe_plan_kernel<DT>, dim3(static_cast<unsigned>(E + more)), dim3(64 * waves), 0, s, ids, n, k, E, per_wave, row_token,
                     slot_row, indptr, x, rows, static_cast<int>(cols), q, scale);
  return hipGetLastError();
}

hipError_t launch_moe_plan(const int32_t* ids, int64_t slots, int k, int E, int32_t* row_token, int32_t* slot_row,
                           int32_t* indptr, hipStream_t s) {
  return launch_plan<kPlanOnly>(ids, slots, k, E, row_token, slot_row, indptr, nullptr, 0, 0, nullptr, nullptr, s);
}

hipError_t launch_moe_plan_quantize(const int32_t* ids, int64_t slots, int k, int E, int32_t* row_token, int32_t* slot_row,
                                    int32_t* indptr, const void* x, int64_t rows, int64_t cols, int model_dtype, uint8_t* q, float* scale,
                                    hipStream_t s) {
  return model_dtype == MODEL_BF16 ? launch_plan<MODEL_BF16>(ids, slots, k, E, row_token, slot_row, indptr, x, rows, cols, q, scale, s)
                                   : launch_plan<MODEL_F16>(ids, slots, k, E, row_token, slot_row, indptr, x, rows, cols, q, scale, s);
}

// One thread eight neighbouring columns of a token; y and the sum in float32, one rounding at the end.  Four experts at a time, rows and then
// values asked for together: one after the other, 16 tokens of 8 experts and 2048 columns took 6.2 us.  A slot without an expert reads row 0 and
// adds nothing.
template <int DT>
__global__ __launch_bounds__(256) void moe_weighted_sum_kernel(const float* __restrict__ y, const int32_t* __restrict__ slot_row,
                                                               const float* __restrict__ weights, int64_t T, int k, int64_t H,
                                                               void* __restrict__ out) {
  const int64_t per_row = H / 8, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= T * per_row) return;
  const int64_t t = i / per_row, h = (i - t * per_row) * 8;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  constexpr int kAtATime = 4;
  for (int j0 = 0; j0 < k; j0 += kAtATime) {
    int at[kAtATime];
    float w[kAtATime], f[kAtATime][8];
#pragma unroll
    for (int u = 0; u < kAtATime; ++u) {
      const int j = j0 + u < k ? j0 + u : k - 1;
      at[u] = slot_row[t * k + j];
      w[u] = weights[t * k + j];
      if (j0 + u >= k) at[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < kAtATime; ++u) fp8_load8<MODEL_F32>(y, (at[u] < 0 ? 0 : at[u]) * H + h, f[u]);
#pragma unroll
    for (int u = 0; u < kAtATime; ++u)
#pragma unroll
      for (int v = 0; v < 8; ++v) acc[v] = at[u] < 0 ? acc[v] : __builtin_fmaf(w[u], f[u][v], acc[v]);
  }
#pragma unroll
  for (int v = 0; v < 8; ++v) Elem<DT>::store(out, t * H + h + v, acc[v]);
}

hipError_t launch_moe_weighted_sum(const float* y, const int32_t* slot_row, const float* weights, int64_t T, int k, int64_t H, int model_dtype,
                                   void* out, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((T * (H / 8) + 255) / 256));
  if (model_dtype == MODEL_BF16)
    hipLaunchKernelGGL(moe_weighted_sum_kernel<MODEL_BF16>, grid, dim3(256), 0, s, y, slot_row, weights, T, k, H, out);
  else
    hipLaunchKernelGGL(moe_weighted_sum_kernel<MODEL_F16>, grid, dim3(256), 0, s, y, slot_row, weights, T, k, H, out);
  return hipGetLastError();
}

}  // namespace gq
