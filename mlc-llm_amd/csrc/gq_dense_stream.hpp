// The core of the products of few rows: weights stream from memory into registers and through the matrix instruction once.
//
// An operand of v_mfma_f32_16x16x32 is 16 rows by 32 numbers of K, 8 of them a lane.  A wave takes 16 rows of W (operand A) times 16
// rows of x (operand B) in blocks of 64 of K: two loads of 16 rows x 64 bytes, which are the two halves of the same 128-byte lines.  x comes
// from the caches in the same form.  D blocks are in flight while one is computed, also from one tile to the next: bound by HBM.
#pragma once

#include "gq_dense_common.hpp"

namespace gq {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr uint32_t kNowhere = 0xffffffffu;  // past any buffer's end: reads as zeros, and asks the memory for nothing
constexpr int kStreamBlock = 64;            // numbers of K in a block

__device__ __forceinline__ rsrc_t dense_buffer(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes > 0xfffffff0ll ? 0xfffffff0u : static_cast<uint32_t>(bytes)),
                                           0x00027000);
}
__device__ __forceinline__ int4_t dense_chunk(rsrc_t r, uint32_t at) {
  return __builtin_bit_cast(int4_t, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
}

// What a wave works on: NR times 16 rows of W, each from the start of its buffer (which ends behind the last row that is there: the
// others read as zeros), and TT times 16 rows of x.  end: K, or 0 for nothing.
template <int NR, int TT>
struct StreamPlace {
  rsrc_t w[NR];
  uint32_t x_at[TT];  // byte offset of this lane's row of x
  int end;
};

// `rounds` places one after the other.  This wave takes every KW-th block of K from block kw on, nb blocks of each place (a multiple of D; past
// K they are zeros).  place_of(round) gives a place, done(round, sums) takes its sums: the lane holds row lane % 16 of x, rows
// 4 (lane / 16) .. + 3 of W.
template <bool BF, int NR, int TT, int D, class PlaceOf, class Done>
__device__ __forceinline__ void dense_stream(int K, int kw, int KW, int nb, int rounds, rsrc_t x, PlaceOf place_of, Done done) {
  const int lane = threadIdx.x & 63, quad = lane >> 4;
  const uint32_t w_at = static_cast<uint32_t>(lane & 15) * static_cast<uint32_t>(K) * 2u;
  int4_t wq[D][NR][2], xq[D][TT][2];
  auto load = [&](const StreamPlace<NR, TT>& p, int j, int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = (j * KW + kw) * kStreamBlock + 32 * h + 8 * quad;  // a chunk of 8; K is a multiple of 8
      const bool in = k < p.end;
#pragma unroll
      for (int i = 0; i < NR; ++i) wq[s][i][h] = dense_chunk(p.w[i], in ? w_at + 2u * k : kNowhere);
#pragma unroll
      for (int t = 0; t < TT; ++t) xq[s][t][h] = dense_chunk(x, in ? p.x_at[t] + 2u * k : kNowhere);
    }
  };
  StreamPlace<NR, TT> here = place_of(0);
#pragma unroll
  for (int s = 0; s < D; ++s) load(here, s, s);
  for (int round = 0; round < rounds; ++round) {
    float4_t acc[NR][TT];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[i][t] = float4_t{};
    auto compute = [&](int s) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int t = 0; t < TT; ++t) acc[i][t] = dense_mfma<BF>(wq[s][i][h], xq[s][t][h], acc[i][t]);
    };
    for (int j = D; j < nb; j += D) {
#pragma unroll
      for (int s = 0; s < D; ++s) {
        compute(s);
        load(here, j + s, s);
        __builtin_amdgcn_sched_barrier(0);  // a block after the other: operands of all would not fit the registers twice
      }
    }
    here = place_of(round + 1);
#pragma unroll
    for (int s = 0; s < D; ++s) {
      compute(s);
      load(here, s, s);
      __builtin_amdgcn_sched_barrier(0);
    }
    done(round, acc);
  }
}

// How a launch shares work: KW of a workgroup's eight waves take a share of K each, the fewest that keep the memory busy.
struct StreamPlan {
  int kw_log2, nb;
};
inline StreamPlan stream_plan(double items, int64_t K, int D, double target) {
  const int64_t blocks = (K + kStreamBlock - 1) / kStreamBlock;
  int log2 = 0;
  while (log2 < 3 && items * (1 << log2) < target && (blocks >> (log2 + 1)) * 2 > D) ++log2;
  const int64_t each = (blocks + (1 << log2) - 1) >> log2;
  return {log2, static_cast<int>((each + D - 1) / D * D)};
}

}  // namespace gq
