// The routing of two tokens by one wave, for the kernels that route.
#pragma once

#include "gq_fp8_common.hpp"
#include "gq_topk.hpp"

namespace gq {

namespace {

// over the 32 lanes of a token, two rows of 16: rotations within a row, then each row with its neighbour
template <class Op>
__device__ __forceinline__ uint32_t reduce32(uint32_t v, Op op) {
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x128, 0xf, 0xf, false)));  // row_ror:8
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x124, 0xf, 0xf, false)));
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x122, 0xf, 0xf, false)));
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x121, 0xf, 0xf, false)));
  const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return op(both[0], both[1]);
}
template <class Op>
__device__ __forceinline__ float reduce32_f(float v, Op op) {
  return __builtin_bit_cast(float, reduce32(__builtin_bit_cast(uint32_t, v), [op](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, op(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
  }));
}
// bits in the order of the numbers; 0 stands behind all of them
__device__ __forceinline__ uint32_t in_order(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  return b ^ ((b >> 31) != 0u ? 0xffffffffu : 0x80000000u);
}

}  // namespace

// LDS of one wave's two tokens
template <int NC>
struct GateScratch {
  float scores[2][NC * 32];
  float keys[2][NC * 32];
  float standings[2][64];
};

// what the routing of a token goes by, as in GatingArgs; group_inv: gate_group_inv
struct GateRule {
  const float* bias;
  int E, k, sigmoid, groups, top_groups, group_inv, renormalize;
  float scale;
};
inline int gate_group_inv(int E, int groups) { return ((1 << 20) + E / groups - 1) / (E / groups); }

// The logits of row t that lane r of a token's 32 holds, experts NC r to NC r + NC - 1 (-infinity past the last one).  vec: E % 8 == 0
// and aligned.
template <int NC, int DT>
__device__ __forceinline__ void gate_load(const void* logits, int64_t t, int E, int r, int vec, float (&score)[NC]) {
  const int e0 = r * NC;
  const float inf = __builtin_inff();
  if (NC >= 8 && vec) {  // uniform
#pragma unroll
    for (int c = 0; c < NC; c += 8) {
      float f[8] = {-inf, -inf, -inf, -inf, -inf, -inf, -inf, -inf};
      if (e0 + c < E) fp8_load8<DT>(logits, t * E + e0 + c, f);
#pragma unroll
      for (int v = 0; v < 8; ++v)
        if (c + v < NC) score[c + v] = f[v];
    }
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c) score[c] = e0 + c < E ? Elem<DT>::load(logits, t * E + e0 + c) : -inf;
  }
}

// Two tokens a wave: lane r of a token's 32 holds experts NC r to NC r + NC - 1.  With logits x:
//   score = softmax(x) or 1 / (1 + exp(-x)) in float32, with the division and the exponential of the C library;
//   key   = score + bias.
// With groups, a group's standing is its best key, or the sum of its best two where there is a bias, and only the experts
// of the top_groups best are looked at.  Then k rounds pick the largest key left, and of equal ones (as of equal groups) the one of the
// lowest index: the largest of a lane's keys, then of the 32 lanes', then the lowest expert that has it.
// A NaN logit has score 0 and stands behind every other expert (as one of a NaN key does); +inf counts as the largest finite number, and a
// softmax over nothing but -inf has scores 0.  Weights whose sum is 0 stay 0.
//
// Bound by the length of one wave's chain of instructions: a round is about 5 NC + 20 of them.  4096
// tokens of 256 experts in 8 groups 7.1 to 7.3 us in a graph of them, 1.9 of it the launch, and 6.6 a call among others (a token a wave, and ballots
// for the choice: 9.2 in a graph; four tokens a wave: 8.4); one token of 64 experts 2.6.
//
// score: the logits.  Lane r < k of a token's 32 ends up with the r-th choice: its expert in *id and its weight in the result.
template <int NC>
__device__ __forceinline__ float gate_pair(GateScratch<NC>& lds, float (&score)[NC], const GateRule& rule, int* id) {
  const int r = threadIdx.x & 31, token = (threadIdx.x >> 5) & 1, e0 = r * NC;
  const int E = rule.E, k = rule.k, groups = rule.groups;
  const float* const bias = rule.bias;
  constexpr float kBig = 3.402823466e38f;
  const float inf = __builtin_inff();
  float key[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float x = score[c];
    key[c] = x == x ? 0.f : -inf;  // added to the key at the end
    score[c] = x == x ? fminf(x, kBig) : -inf;
  }
  if (rule.sigmoid) {
#pragma unroll
    for (int c = 0; c < NC; ++c) score[c] = 1.0f / (1.0f + expf(-score[c]));
  } else {
    float m = score[0];
#pragma unroll
    for (int c = 1; c < NC; ++c) m = fmaxf(m, score[c]);
    m = reduce32_f(m, [](float a, float b) { return fmaxf(a, b); });
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      score[c] = score[c] == -inf ? 0.f : expf(score[c] - m);
      sum += score[c];
    }
    sum = reduce32_f(sum, [](float a, float b) { return a + b; });
#pragma unroll
    for (int c = 0; c < NC; ++c) score[c] = sum > 0.f ? score[c] / sum : 0.f;
  }
  uint32_t order[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float v = score[c];
    if (bias != nullptr && e0 + c < E) v += bias[e0 + c];
    v += key[c];
    key[c] = v == v ? v : -inf;
    order[c] = e0 + c < E ? in_order(key[c]) : 0u;
    lds.scores[token][e0 + c] = score[c];
  }
  // (what a wave wrote to LDS it may read behind a fence)
  auto written = [] {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  if (groups > 1) {  // uniform
    const int size = E / groups;
    auto join = [&](float& best, float& next, float other, float other_next) {
      next = fmaxf(fmaxf(next, other_next), fminf(best, other));
      best = fmaxf(best, other);
    };
    auto standing_of = [&](float best, float next) {
      if (bias == nullptr || size == 1) return best;
      const float both = best + next;
      return both == both ? both : -inf;
    };
    auto groups_ahead = [&](int g, float mine) {
      int ahead = 0;
#pragma unroll 4
      for (int o = 0; o < groups; ++o) {
        const float v = lds.standings[token][o];
        ahead += (v > mine || (v == mine && o < g)) ? 1 : 0;
      }
      return ahead;
    };
    const int lanes = size / NC;  // of a group
    if (lanes * NC == size && (lanes & (lanes - 1)) == 0) {  // a lane's experts are of one group: no way through LDS
      float best = -inf, next = -inf;
#pragma unroll
      for (int c = 0; c < NC; ++c) join(best, next, key[c], -inf);
      for (int d = 1; d < lanes; d *= 2) {
        const float other = __shfl_xor(best, d), other_next = __shfl_xor(next, d);
        join(best, next, other, other_next);
      }
      const int g = r / lanes;
      const float mine = standing_of(best, next);
      lds.standings[token][g] = mine;  // (from each of the group's lanes; past the last group: unread)
      written();
      const bool kept = groups_ahead(g, mine) < rule.top_groups;
#pragma unroll
      for (int c = 0; c < NC; ++c) order[c] = kept ? order[c] : 0u;
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) lds.keys[token][e0 + c] = key[c];
      written();
      for (int g = r; g < groups; g += 32) {
        float best = -inf, next = -inf;
#pragma unroll 4
        for (int j = 0; j < size; ++j) join(best, next, lds.keys[token][g * size + j], -inf);
        lds.standings[token][g] = standing_of(best, next);
      }
      written();
      uint64_t kept = 0;  // groups of this lane's, then of all lanes'
      for (int g = r; g < groups; g += 32)
        if (groups_ahead(g, lds.standings[token][g]) < rule.top_groups) kept |= 1ull << g;
      auto either = [](uint32_t a, uint32_t b) { return a | b; };
      kept = reduce32(static_cast<uint32_t>(kept), either) |
             static_cast<uint64_t>(reduce32(static_cast<uint32_t>(kept >> 32), either)) << 32;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int g = ((e0 + c) * rule.group_inv) >> 20;  // (e0 + c) / size
        if (!((kept >> (g & 63)) & 1ull)) order[c] = 0u;
      }
    }
  }
  written();
  float sum = 0.f;
  int my_id = 0;
  for (int i = 0; i < k; ++i) {
    uint32_t m = order[0];
#pragma unroll
    for (int c = 1; c < NC; ++c) m = m > order[c] ? m : order[c];
    m = reduce32(m, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    uint32_t first = 0x7fffffffu;
#pragma unroll
    for (int c = NC - 1; c >= 0; --c) first = order[c] == m ? static_cast<uint32_t>(e0 + c) : first;
    first = reduce32(first, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
#pragma unroll
    for (int c = 0; c < NC; ++c) order[c] = static_cast<uint32_t>(e0 + c) == first ? 0u : order[c];
    if (r == i) my_id = static_cast<int>(first);
    sum += lds.scores[token][first];
  }
  *id = my_id;
  float v = lds.scores[token][my_id];
  if (rule.renormalize) v = sum > 0.f ? v / sum : 0.f;
  return v * rule.scale;
}

}  // namespace gq
