// Routing of 8-bit block-scaled expert layers: scores, selection in groups of experts, weights; the stable order of the
// slots by expert; the weighted sum over a token's experts.  Small integer and float32 work, bound by latency.
#include "gq_fp8_common.hpp"
#include "gq_topk.hpp"

namespace gq {

namespace {

__device__ __forceinline__ float wave_max(float v) {
  v = row_max16(v);
  float m = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 0));
#pragma unroll
  for (int r = 1; r < 4; ++r)
    m = fmaxf(m, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 16 * r)));
  return m;
}

}  // namespace

// One wave a token; lane l holds experts l, l + 64, ...  With logits x:
//   score = softmax(x) or 1 / (1 + exp(-x)) in float32, with the division and the exponential of the C library;
//   key   = score + bias.
// With groups, a group's standing is its best key, or the sum of its best two where there is a bias, and only the experts
// of the top_groups best are looked at.  Then k rounds pick the largest key left.  Equal keys and equal groups go to the
// lower index: chunk by chunk, a ballot of the lanes that hold the round's maximum, whose first bit is the lowest expert.
// A NaN logit has score 0 and stands behind every other expert (as one of a NaN key does); +inf counts as the largest finite number, and a
// softmax over nothing but -inf has scores 0.  Weights whose sum is 0 stay 0.
template <int NCH, int DT>
__global__ __launch_bounds__(256) void gating_kernel(const void* __restrict__ logits, const float* __restrict__ bias,
                                                     int64_t T, int E, int k, int sigmoid, int groups, int top_groups,
                                                     int group_inv, int renormalize, float scale,
                                                     float* __restrict__ weights, int32_t* __restrict__ ids) {
  __shared__ float lds[4][NCH * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  if (t >= T) return;  // whole waves; no barrier below
  constexpr float kBig = 3.402823466e38f;
  const float inf = __builtin_inff();
  float score[NCH], key[NCH];
  unsigned alive = 0;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int e = lane + 64 * c;
    float x = -inf;
    if (e < E) {
      x = Elem<DT>::load(logits, t * E + e);
      alive |= 1u << c;
    }
    score[c] = fminf(x, kBig);       // (a NaN becomes kBig here: set apart below)
    key[c] = x == x ? 0.f : -inf;    // added to the key at the end
    if (!(x == x)) score[c] = -inf;
  }
  if (sigmoid) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) score[c] = 1.0f / (1.0f + expf(-score[c]));
  } else {
    float m = score[0];
#pragma unroll
    for (int c = 1; c < NCH; ++c) m = fmaxf(m, score[c]);
    m = wave_max(m);
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      score[c] = score[c] == -inf ? 0.f : expf(score[c] - m);
      sum += score[c];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int c = 0; c < NCH; ++c) score[c] = sum > 0.f ? score[c] / sum : 0.f;
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int e = lane + 64 * c;
    float v = score[c];
    if (bias != nullptr && e < E) v += bias[e];
    v += key[c];
    key[c] = v == v ? v : -inf;
  }
  if (groups > 1) {  // uniform
    float* mine = lds[wave];
    const int size = E / groups;
#pragma unroll
    for (int c = 0; c < NCH; ++c) mine[lane + 64 * c] = key[c];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float standing = -inf;
    if (lane < groups) {
      float best = -inf, next = -inf;
      for (int j = 0; j < size; ++j) {
        const float v = mine[lane * size + j];
        next = fmaxf(next, fminf(best, v));
        best = fmaxf(best, v);
      }
      standing = best;
      if (bias != nullptr && size > 1) {
        standing = best + next;
        standing = standing == standing ? standing : -inf;
      }
    }
    int ahead = 0;
    for (int g = 0; g < groups; ++g) {
      const float o = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, standing), g));
      ahead += (o > standing || (o == standing && g < lane)) ? 1 : 0;
    }
    const unsigned long long kept = __ballot(lane < groups && ahead < top_groups);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int g = ((lane + 64 * c) * group_inv) >> 20;  // (lane + 64 c) / size
      if (!((kept >> (g & 63)) & 1ull)) alive &= ~(1u << c);
    }
  }
  float my_score = 0.f, sum = 0.f;
  int my_id = 0;
  for (int i = 0; i < k; ++i) {
    float m = -inf;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      if ((alive >> c) & 1u) m = fmaxf(m, key[c]);
    m = wave_max(m);
    bool found = false;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const unsigned long long at = __ballot(((alive >> c) & 1u) && key[c] == m);
      if (!found && at != 0ull) {  // uniform
        found = true;
        const int src = __builtin_ctzll(at);
        const float s =
            __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, score[c]), src));
        if (lane == src) alive &= ~(1u << c);
        if (lane == i) {
          my_id = src + 64 * c;
          my_score = s;
        }
        sum += s;
      }
    }
  }
  if (lane < k) {
    if (renormalize) my_score = sum > 0.f ? my_score / sum : 0.f;
    weights[t * k + lane] = my_score * scale;
    ids[t * k + lane] = my_id;
  }
}

hipError_t launch_moe_gating(const GatingArgs& a, hipStream_t s) {
  const int nch = (a.E + 63) / 64, size = a.E / a.groups;
  const dim3 grid(static_cast<unsigned>((a.T + 3) / 4));
  auto go = [&](auto ch, auto dt) {
    hipLaunchKernelGGL((gating_kernel<decltype(ch)::value, decltype(dt)::value>), grid, dim3(256), 0, s, a.logits, a.bias,
                       a.T, a.E, a.k, a.sigmoid, a.groups, a.top_groups, ((1 << 20) + size - 1) / size, a.renormalize,
                       a.scale, a.weights, a.ids);
  };
  auto by_type = [&](auto ch) {
    if (a.model_dtype == MODEL_F32) go(ch, std::integral_constant<int, MODEL_F32>{});
    else if (a.model_dtype == MODEL_BF16) go(ch, std::integral_constant<int, MODEL_BF16>{});
    else go(ch, std::integral_constant<int, MODEL_F16>{});
  };
  if (nch <= 1) by_type(std::integral_constant<int, 1>{});
  else if (nch <= 2) by_type(std::integral_constant<int, 2>{});
  else if (nch <= 4) by_type(std::integral_constant<int, 4>{});
  else by_type(std::integral_constant<int, 8>{});
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
  for (int s0 = begin; s0 < end; s0 += 64) {
    const int id = s0 + lane < end ? ids[s0 + lane] : -1;
    own += __popcll(__ballot(id == e));
    before += __popcll(__ballot(id >= 0 && id < e));
  }
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
  for (int s0 = begin; s0 < end; s0 += 64) {
    const int s = s0 + lane, id = s < end ? ids[s] : -1;
    const unsigned long long m = __ballot(id == e);
    if (id == e) {
      const int row = at + __popcll(m & ((1ull << lane) - 1ull));
      row_token[row] = s / k;
      slot_row[s] = row;
    } else if (e == 0 && s < end && (id < 0 || id >= E)) {
      slot_row[s] = -1;
    }
    at += __popcll(m);
  }
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

// One thread eight neighbouring columns of a token (H % 8 == 0) or one (any H); float32 throughout, one rounding at the end.
template <int DT, int VEC>
__global__ __launch_bounds__(256) void moe_weighted_sum_kernel(const void* __restrict__ y, const int32_t* __restrict__ slot_row,
                                                               const int32_t* __restrict__ ids, int E, const float* __restrict__ weights, int64_t T, int k, int64_t H,
                                                               void* __restrict__ out) {
  const int64_t per_row = H / VEC, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= T * per_row) return;
  const int64_t t = i / per_row, h = (i - t * per_row) * VEC;
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
  for (int j = 0; j < k; ++j) {
    const int at = slot_row ? slot_row[t * k + j] : ids[t * k + j];
    if (at < 0 || (!slot_row && at >= E)) continue;
    const int64_t row = slot_row ? at : t * k + j;
    const float w = weights[t * k + j];
    if constexpr (VEC == 8) {
      float f[8];
      if constexpr (DT == MODEL_F32) {
        const float4_t* p = reinterpret_cast<const float4_t*>(static_cast<const float*>(y) + row * H + h);
        const float4_t a = p[0], b = p[1];
#pragma unroll
        for (int v = 0; v < 4; ++v) f[v] = a[v], f[v + 4] = b[v];
      } else {
        const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(y) + row * H + h);
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          f[2 * v] = DT == MODEL_BF16 ? bf2f(u[v] & 0xffffu) : h2f(u[v] & 0xffffu);
          f[2 * v + 1] = DT == MODEL_BF16 ? bf2f(u[v] >> 16) : h2f(u[v] >> 16);
        }
      }
#pragma unroll
      for (int v = 0; v < 8; ++v) acc[v] = __builtin_fmaf(w, f[v], acc[v]);
    } else {
      acc[0] = __builtin_fmaf(w, Elem<DT>::load(y, row * H + h), acc[0]);
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) Elem<DT>::store(out, t * H + h + v, acc[v]);
}

hipError_t launch_moe_weighted_sum(const void* y, const int32_t* slot_row, const int32_t* ids, int E, const float* weights, int64_t T,
                                   int k, int64_t H, int model_dtype, void* out, hipStream_t s) {
  auto go = [&](auto dt, auto vec) {
    const int64_t n = T * (H / decltype(vec)::value);
    hipLaunchKernelGGL((moe_weighted_sum_kernel<decltype(dt)::value, decltype(vec)::value>),
                       dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, s, y, slot_row, ids, E, weights, T, k, H, out);
  };
  auto by_type = [&](auto vec) {
    if (model_dtype == MODEL_F32) go(std::integral_constant<int, MODEL_F32>{}, vec);
    else if (model_dtype == MODEL_BF16) go(std::integral_constant<int, MODEL_BF16>{}, vec);
    else go(std::integral_constant<int, MODEL_F16>{}, vec);
  };
  if (H % 8 == 0) by_type(std::integral_constant<int, 8>{});
  else by_type(std::integral_constant<int, 1>{});
  return hipGetLastError();
}

}  // namespace gq
