// The core of the products of few rows: weights stream from memory through LDS and the matrix instruction once, bound by HBM.
//
// A block is 16 rows of W by 64 numbers of K, 128 bytes of a row, and the same part of 8 XG rows of x.  Loads go past the registers into
// the wave's own ring in LDS, eight rows of whole 128-byte lines an instruction, D blocks ahead of their use, without a barrier: the wave waits
// for its own loads alone.  From there v_mfma_f32_16x16x32 takes W as operand A and x as operand B.
// Measured on the way here, 128256 x 4096 of 5 rows: operands loaded straight into registers, 64 bytes of 16 rows an instruction, 175 us; the same
// with `nt` loads (of lines that are read once), which then come for every half of a line, 196; whole lines through LDS 170, with `nt` 156, and x
// on the same way 153 = 6.85 TB/s, what a large copy's reads reach.  16 rows of 4096 x 14336 in these forms: 31, 36, 27, 26 and 23.6 us.
#pragma once

#include "gq_dense_common.hpp"

namespace gq {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr uint32_t kNowhere = 0xc0000000u;  // past the end of any buffer here, also with an offset into a row behind it: reads as zeros
constexpr int64_t kReach = 0xc0000000ll;    // bytes of a buffer, below
constexpr int kStreamBlock = 64;            // numbers of K in a block
constexpr int kStreamWaves = 8;             // of a workgroup
constexpr int kStreamUnits = 256;           // workgroups that run at a time, where their rings take most of a unit's LDS

__device__ __forceinline__ rsrc_t dense_buffer(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes < kReach ? static_cast<uint32_t>(bytes) : kNowhere), 0x00027000);
}
// 16 bytes a lane into LDS at lds + 16 * lane.  ONCE: weights, which no other load will ask for (`nt`).
template <bool ONCE>
__device__ __forceinline__ void dense_to_lds(rsrc_t r, uint32_t at, uint8_t* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, at, 0, 0, ONCE ? 2 : 0);
}

// What a wave works on: twice eight rows of W, each from the start of its buffer (which ends behind the last row that is there: the
// others read as zeros), and XG times eight rows of x.
template <int XG>
struct StreamPlace {
  rsrc_t w[2];
  rsrc_t x;
  uint32_t x_at[XG];  // byte offset of this lane's row of x, row lane / 8 of eight
  int k, end;         // this wave's first number of K and the end of K in a row (0: nothing to do)
};

template <int XG>
constexpr int stream_stage() { return 2048 + XG * 1024; }
template <int XG, int D>
constexpr int stream_ring() { return D * stream_stage<XG>(); }

// One block from number k of the rows on, into a stage.  Chunk c of 16 bytes of a row lies at place c ^ (row & 7), so that the 16 lanes that LDS
// serves at a time meet all its banks.
template <int XG>
__device__ __forceinline__ void stream_load(const StreamPlace<XG>& p, int k, uint32_t w_pitch, uint8_t* stage) {
  const int lane = threadIdx.x & 63, kc = k + 8 * ((lane & 7) ^ (lane >> 3));  // a chunk of 8; K is a multiple of 8
  const bool in = kc < p.end;
  const uint32_t w_at = in ? static_cast<uint32_t>(lane >> 3) * w_pitch + 2u * kc : kNowhere;
#pragma unroll
  for (int i = 0; i < 2; ++i) dense_to_lds<true>(p.w[i], w_at, stage + 1024 * i);
#pragma unroll
  for (int g = 0; g < XG; ++g) dense_to_lds<false>(p.x, in ? p.x_at[g] + 2u * kc : kNowhere, stage + 2048 + g * 1024);
  asm volatile("" ::: "memory");  // (before the next block's, by which the wait counts)
}
// Waits until all but the newest D - 1 blocks have landed.
template <int XG, int D>
__device__ __forceinline__ void stream_wait() {
  static_assert((D - 1) * (2 + XG) < 64, "the counter of loads");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * (2 + XG)) : "memory");
}
// sums += the block in a stage; the lane holds row 16 t + lane % 16 of x and rows 4 (lane / 16) .. + 3 of W.
template <bool BF, int XG>
__device__ __forceinline__ void stream_block(const uint8_t* stage, float4_t (&acc)[(XG + 1) / 2]) {
  constexpr int TT = (XG + 1) / 2;
  const int lane = threadIdx.x & 63, quad = lane >> 4, row = lane & 15;
  const int c0 = (quad ^ (row & 7)) << 4, c1 = ((quad + 4) ^ (row & 7)) << 4;
  const int4_t w0 = *reinterpret_cast<const int4_t*>(stage + row * 128 + c0), w1 = *reinterpret_cast<const int4_t*>(stage + row * 128 + c1);
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    // (eight rows of x: rows 8 to 15 of the operand are those again, and their sums nobody's)
    const uint8_t* const x = stage + 2048 + (XG == 1 ? row & 7 : 16 * t + row) * 128;
    acc[t] = dense_mfma<BF>(w0, *reinterpret_cast<const int4_t*>(x + c0), acc[t]);
    acc[t] = dense_mfma<BF>(w1, *reinterpret_cast<const int4_t*>(x + c1), acc[t]);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (read, before the stage is loaded again)
}

// `rounds` places one after the other, of each nb blocks, `step` numbers of K apart; past K they are zeros.  place_of(round) gives a place,
// done(round, sums) takes its sums.  nb a multiple of D goes around the ring without a branch (128 x 2048 of one row 3.7 us, and 4.2 the other way);
// with ANY it may be anything, and a place's last stage is followed by the next one's first (2 x 9728 x 2560, five blocks a wave, 12.1 us, and 13.8
// padded to eight).
template <bool BF, int XG, int D, bool ANY, class PlaceOf, class Done>
__device__ __forceinline__ void dense_stream(uint8_t* ring, uint32_t w_pitch, int step, int nb, int rounds, PlaceOf place_of, Done done) {
  constexpr int TT = (XG + 1) / 2, kStage = stream_stage<XG>();
  StreamPlace<XG> here = place_of(0);
  float4_t acc[TT];
  auto clear = [&] {
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = float4_t{};
  };
  if constexpr (!ANY) {
#pragma unroll
    for (int s = 0; s < D; ++s) stream_load(here, here.k + s * step, w_pitch, ring + s * kStage);
    for (int round = 0; round < rounds; ++round) {
      clear();
      for (int j = D; j < nb; j += D) {
#pragma unroll
        for (int s = 0; s < D; ++s) {
          stream_wait<XG, D>();
          stream_block<BF, XG>(ring + s * kStage, acc);
          stream_load(here, here.k + (j + s) * step, w_pitch, ring + s * kStage);
        }
      }
      here = place_of(round + 1);
#pragma unroll
      for (int s = 0; s < D; ++s) {
        stream_wait<XG, D>();
        stream_block<BF, XG>(ring + s * kStage, acc);
        stream_load(here, here.k + s * step, w_pitch, ring + s * kStage);
      }
      done(round, acc);
    }
  } else {
    int at = 0, block = 0;  // place and number there of the next block to load
    auto load = [&](uint8_t* stage) {
      stream_load(here, here.k + block * step, w_pitch, stage);
      if (++block == nb) {
        block = 0;
        here = place_of(++at);
      }
    };
#pragma unroll 1
    for (int s = 0; s < D; ++s) load(ring + s * kStage);
    uint8_t* stage = ring;
    for (int round = 0; round < rounds; ++round) {
      clear();
#pragma unroll 1
      for (int j = 0; j < nb; ++j) {
        stream_wait<XG, D>();
        stream_block<BF, XG>(stage, acc);
        load(stage);
        stage = stage == ring + (D - 1) * kStage ? ring : stage + kStage;
      }
      done(round, acc);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (loads of nothing may still land in the ring)
}

// The same with this wave's part of x in registers, loaded where the item's rows of x change: NB blocks of an item, those of K that the wave takes.
// x of a segment comes once a workgroup and not with every item, and the ring holds weights alone.
template <int NB, int TT>
struct StreamKept {
  int4_t v[NB][2][TT];
};
struct StreamRows {
  rsrc_t w[2];
  int end;  // K, or 0: nothing to do
};
constexpr int kKeptStage = 2048;
// at[t]: byte offset of row 16 t + lane % 16 of x; k: this wave's first number of K, its blocks `step` apart.
template <int NB, int TT>
__device__ __forceinline__ void kept_x(StreamKept<NB, TT>& to, rsrc_t x, const uint32_t (&at)[TT], int k, int step, int K) {
  const int kc = k + 8 * ((threadIdx.x & 63) >> 4);
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const int at_k = kc + j * step + 32 * i;
        to.v[j][i][t] = __builtin_bit_cast(int4_t, __builtin_amdgcn_raw_buffer_load_b128(x, at_k < K ? at[t] + 2u * at_k : kNowhere, 0, 0));
      }
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < TT; ++t) asm volatile("" : "+v"(to.v[j][i][t]));  // (waited for here, not behind the loads of weights that follow)
}
__device__ __forceinline__ void kept_load(const StreamRows& p, int k, uint32_t w_pitch, uint8_t* stage) {
  const int lane = threadIdx.x & 63, kc = k + 8 * ((lane & 7) ^ (lane >> 3));
  const uint32_t at = kc < p.end ? static_cast<uint32_t>(lane >> 3) * w_pitch + 2u * kc : kNowhere;
#pragma unroll
  for (int i = 0; i < 2; ++i) dense_to_lds<true>(p.w[i], at, stage + 1024 * i);
  asm volatile("" ::: "memory");  // (before the next block's, by which the wait counts)
}
// keep(round, kept) brings x where it changes, rows_of(round) gives the rows of W.  k: this wave's first number of K.
template <bool BF, int TT, int NB, int D, class RowsOf, class Keep, class Done>
__device__ __forceinline__ void dense_stream_kept(uint8_t* ring, uint32_t w_pitch, int k, int step, int rounds, RowsOf rows_of, Keep keep, Done done) {
  static_assert(NB % D == 0, "the stages of a block in every item");
  const int lane = threadIdx.x & 63, quad = lane >> 4, row = lane & 15;
  const int c0 = (quad ^ (row & 7)) << 4, c1 = ((quad + 4) ^ (row & 7)) << 4;
  StreamRows here = rows_of(0);
#pragma unroll
  for (int s = 0; s < D; ++s) kept_load(here, k + s * step, w_pitch, ring + s * kKeptStage);
  StreamKept<NB, TT> x;
  for (int round = 0; round < rounds; ++round) {
    keep(round, x);
    float4_t acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = float4_t{};
    const StreamRows next = rows_of(round + 1);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      uint8_t* const stage = ring + j % D * kKeptStage;
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * (D - 1)) : "memory");
      const int4_t w0 = *reinterpret_cast<const int4_t*>(stage + row * 128 + c0), w1 = *reinterpret_cast<const int4_t*>(stage + row * 128 + c1);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        acc[t] = dense_mfma<BF>(w0, x.v[j][0][t], acc[t]);
        acc[t] = dense_mfma<BF>(w1, x.v[j][1][t], acc[t]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (read, before the stage is loaded again)
      kept_load(j + D < NB ? here : next, k + (j + D) % NB * step, w_pitch, stage);
    }
    here = next;
    done(round, acc);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// The sums of the KW waves that share an item, in the first one's acc; buf: kStreamWaves TT KiB, no use of it may be left.
template <int TT>
__device__ __forceinline__ void stream_join(float4_t* buf, int wave, int KW, float4_t (&acc)[TT]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int t = 0; t < TT; ++t) buf[(wave * TT + t) * 64 + lane] = acc[t];
  // (no __syncthreads, which waits for the loads ahead as well)
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if ((wave & (KW - 1)) != 0) return;
  for (int w = 1; w < KW; ++w)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] += buf[((wave + w) * TT + t) * 64 + lane];
}

// Gated: rows 0 to 7 of a block are gates and rows 8 to 15 their up rows, two quarters of the wave apart.
__device__ __forceinline__ float4_t stream_up(float4_t v) {
  float4_t u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = __shfl_down(v[i], 32);
  return u;
}

// KW of a workgroup's eight waves share the K of an item.  More of them read longer runs of a row, fewer leave more blocks a wave between two
// items: the KW of the fewest blocks that a wave takes one after the other, padding and the ends of up to six rounds (0.65 of a block each) counted,
// a twelfth more for a KW of four or two and a third for one.  One row, by KW 8, 4, 2 and 1, us: 28672 x 4096 38.4, 36.2, 45.4, 40.4 (the rule: 8);
// 8192 x 8192 27.0, 29.7, 28.0, 52.2 (8); 6144 x 4096 11.1, 12.3, 15.3, 24.2 (8); 5120 x 5120, of whose 10 blocks a wave of eight has two empty
// ones, 13.4, 12.1, 18.1, 30.7 (4); 152064 x 3584 162.6, 151.8, 153.4, 155.2 (2).
// any: nb may be no multiple of D where it is more, at a seventh more for a block.
struct StreamPlan {
  int kw_log2, nb, rounds;
};
inline StreamPlan stream_plan(double items, int64_t K, int D, bool any) {
  const int64_t blocks = (K + kStreamBlock - 1) / kStreamBlock;
  StreamPlan best{0, 0, 0};
  double best_cost = 0;
  for (int log2 = 3; log2 >= 0; --log2) {
    const int64_t each = (blocks + (1 << log2) - 1) >> log2, whole = (each + D - 1) / D * D, nb = any && each > D ? each : whole;
    const double rounds = __builtin_ceil(items / ((kStreamWaves >> log2) * kStreamUnits));
    const double ends = 0.65 * (rounds < 6 ? rounds : 6);
    const double cost = (rounds * static_cast<double>(nb) + ends) * (log2 == 0 ? 1.3 : log2 < 3 ? 1.08 : 1.0) * (nb < whole ? 1.15 : 1.0);
    if (best.nb == 0 || cost < best_cost) {
      best_cost = cost;
      best = {log2, static_cast<int>(nb), static_cast<int>(rounds)};
    }
  }
  return best;
}

}  // namespace gq
