// A mixture-of-experts layer with 16-bit weights on a few tokens, in two kernels.
//
//   y_t = sum over j of w_tj  W2[e_tj] h_tj,  h_tj = act(Wg[e_tj] x_t) * (Wu[e_tj] x_t),  (w, e)_t the routing of token t
//
// The first routes (every workgroup all tokens for itself: 2.7 us, where a launch of its own takes as long before its results' way through
// memory) and streams the gate and up rows of the experts that some token chose past these experts' tokens.  A row of w h, the
// weighted activation of one token and expert, goes to the workspace in float32.
// The second streams the down rows past the same rows of w h, which go through the matrix instruction as two or three 16-bit planes (down_planes); what
// comes out of an expert joins the sums of its tokens, which lie in LDS.  An expert meets the tokens that chose it alone, whatever W or the other tokens hold.
// Bound by HBM.  Both kernels, us (of their bytes at 6.85 TB/s): one token, 6 of 64 experts of 2048 x 1408, 27.8 (15.2); 2 of 8 experts of 4096 x 14336,
// 4 tokens 296 (283), 16 tokens 431 (411), 32 tokens 454 (411), 64 tokens 533 (411), where the way of x from the L2 counts beside W's; 16 tokens, 8
// of 128 experts of 2048 x 768, 130 (118).  In memory that a process has given back and taken again all of these take 10 to 20 % more.
#include "gq_dense_stream.hpp"
#include "gq_gating.hpp"

namespace gq {

namespace {

constexpr int kWaves = kStreamWaves, kThreads = 64 * kWaves;

// Up to 8 XG rows of one expert, a matrix instruction's columns in both products.
struct MoeSegment {
  int e, row0, rows;
};
// The workspace: what the first kernel leaves for the second.  Offsets; at 0 the number of segments, at kSegsAt these.
constexpr int64_t kSegsAt = 256;
struct MoeLayout {
  int64_t row_token, tickets, shares, h, bytes;  // h: float32 [T k][inter]
};
inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
inline int moe_shares(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t k);
inline MoeLayout moe_layout(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t k) {
  const int64_t slots = T * k, tiles = (hidden + 31) / 32 * 2;
  MoeLayout l;
  l.row_token = kSegsAt + up256(slots * static_cast<int64_t>(sizeof(MoeSegment)));
  l.tickets = l.row_token + up256(slots * 4);
  l.shares = l.tickets + up256(tiles * 4);
  const int shares = moe_shares(T, hidden, inter, experts, k);
  l.h = l.shares + (shares > 1 ? up256(static_cast<int64_t>(shares) * tiles * T * 64) : 0);
  l.bytes = l.h + up256(slots * inter * 4);
  return l;
}
// experts that some token chooses, where all are alike
inline double experts_chosen(int64_t T, int64_t experts, int64_t k) {
  double none = 1;
  for (int64_t t = 0; t < T; ++t) none *= 1 - static_cast<double>(k) / static_cast<double>(experts);
  return static_cast<double>(experts) * (1 - none);
}
// Eights of rows of a segment: sixteen rows but for one token, whose experts have one each.  The second kernel takes 16 columns a workgroup then, and 32 with
// sixteen rows, where x, which comes half as often, goes straight into registers.  Its us with eights / sixteens: one token, 6 of 64 experts of 2048 x 1408, 10.5 /
// 11.8, 2 of 8 of 4096 x 14336 37.9 / 40.7; 2 tokens, 8 of 64 of 3584 x 2560, 49.5 / 48.3; 4 tokens, 2 of 8 of 4096 x 14336, 105 / 102, 32 tokens 240 / 169; 16
// tokens, 8 of 128 of 2048 x 768, 50 / 46, 64 tokens 93 / 73.
inline int moe_eights(int64_t T) { return T > 1 ? 2 : 1; }
// Workgroups that share the K (all chosen experts' inter) of the columns of one in the second kernel: about one a unit.  The second kernel's us with 1, 2,
// 4 and 8 shares: one token of 64 experts of 2048 x 1408, 128 tiles, 13.4, 10.3, 11.8 and 16.3 (the rule: 2); 16 tokens of 128 of 2048 x 768, 64 tiles, 123, 67, 46
// and 51 (4); 32 tokens of 16 of 7168 x 2048, 224 tiles, 87, 95, 98 and 106 (1).
inline int moe_shares(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t k) {
  if (options().gemm_split_k > 0) return options().gemm_split_k < 8 ? options().gemm_split_k : 8;
  const int64_t tiles = moe_eights(T) == 2 ? (hidden + 31) / 32 : (hidden + 15) / 16;
  const double blocks = experts_chosen(T, experts, k) * static_cast<double>((inter + kStreamBlock - 1) / kStreamBlock);
  int s = 1;
  while (s < 8 && tiles * s < 200 && blocks / (2 * s) >= 4 * kWaves) s *= 2;
  return s;
}

// blocks of K of the first product a wave where all waves of a workgroup share them
inline int moe_blocks(int64_t hidden) { return static_cast<int>((hidden + kWaves * kStreamBlock - 1) / (kWaves * kStreamBlock)); }
// Whether the first kernel keeps x in registers, in segments of 32 rows, rather than load it beside W, in segments of 8 or 16.  It does where that
// fits (4 blocks a wave, or 7 and 8) and a segment is long enough for the wait that each change of x is.  The first kernel's us, with W / kept
// in the same memory:
// 8 experts of 4096 x 14336, 2 a token, 4 tokens 194 / 193, 8 tokens 262 / 262, 16 285 / 280, 32 299 / 285, 48 324 / 290, 64 476 / 300; 64 of 64 experts of 2048 x
// 1408, 6 a token, 127 / 127; 128 experts of 2048 x 768, 8 a token, 16 tokens 85 / 92, 64 tokens 137 / 138.
inline bool moe_keeps(const DenseMoeArgs& a) {
  const int blocks = moe_blocks(a.hidden);
  return (blocks == 4 || blocks == 7 || blocks == 8) && a.T * a.k >= 2 * a.experts && a.inter >= 1024;
}

// Rows of a segment of the second kernel: 32 where the first one keeps x and experts have more than twelve on average (64 tokens, 2 of 8 experts of 4096
// x 14336, 269 -> 235 us; 48 tokens would take 213 and take 191).
inline int moe_down_rows(const DenseMoeArgs& a) {
  return moe_keeps(a) && a.T * a.k > 12 * a.experts ? 32 : 8 * moe_eights(a.T);
}

struct MoeTables {  // in LDS, in front of the rest
  uint64_t* mask;      // [experts] tokens of each
  MoeSegment* segs;    // [T k at most]
  int* expert_row;     // [experts] the first row of each
  int* slot_id;        // [T k]
  float* slot_w;       // [T k]
  int* row_token;      // [T k] in the order of the experts
  float* row_w;        // [T k]
  uint64_t* totals;    // [waves]
};
inline size_t moe_tables_bytes(int experts, int slots) {
  return (64 + static_cast<size_t>(experts) * 12 + static_cast<size_t>(slots) * (16 + sizeof(MoeSegment)) + 15) / 16 * 16;
}

}  // namespace

// NC: experts a lane in the routing.  XG: eights of rows of a segment.  NB: blocks of K a wave whose x it keeps in registers; 0: x comes with every
// item.  down_rows: rows of a segment of the second kernel, 8 XG where NB is 0.
template <bool BF, int NC, int XG, int D, int NB>
__global__ __launch_bounds__(kThreads, D == 2 ? 4 : 2) void dense_moe_up_kernel(
    const void* __restrict__ logits, int T, int E, int top_k, int logits_dtype, int logits_vec, int tables_bytes, int group_inv, int kw_log2, int nb,
    int down_rows, DenseMoeArgs a, MoeLayout layout) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int TT = (XG + 1) / 2, kSegRows = 8 * XG;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slots = T * top_k, K = a.hidden, I = a.inter;
  MoeTables tab;
  tab.totals = reinterpret_cast<uint64_t*>(smem);
  tab.mask = tab.totals + 8;
  tab.expert_row = reinterpret_cast<int*>(tab.mask + E);
  tab.slot_id = tab.expert_row + E;
  tab.slot_w = reinterpret_cast<float*>(tab.slot_id + slots);
  tab.row_token = reinterpret_cast<int*>(tab.slot_w + slots);
  tab.row_w = reinterpret_cast<float*>(tab.row_token + slots);
  tab.segs = reinterpret_cast<MoeSegment*>(tab.row_w + slots);
  uint8_t* const rest = smem + tables_bytes;
  GateScratch<NC>& gate = reinterpret_cast<GateScratch<NC>*>(rest)[wave];

  // ---- routing ----
  if (tid < E) tab.mask[tid] = 0;
  __syncthreads();
  const GateRule rule{a.score_bias, E, top_k, a.sigmoid, a.groups, a.top_groups, group_inv, a.renormalize, a.scale};
  for (int t0 = 2 * wave; t0 < T; t0 += 2 * kWaves) {
    const int t = t0 + (lane >> 5), r = lane & 31;
    const int from = t < T ? t : T - 1;
    float score[NC];
    if (logits_dtype == MODEL_F32) gate_load<NC, MODEL_F32>(logits, from, E, r, logits_vec, score);
    else if (logits_dtype == MODEL_BF16) gate_load<NC, MODEL_BF16>(logits, from, E, r, logits_vec, score);
    else gate_load<NC, MODEL_F16>(logits, from, E, r, logits_vec, score);
    int id;
    const float w = gate_pair<NC>(gate, score, rule, &id);
    if (r < top_k && t < T) {
      tab.slot_id[t * top_k + r] = id;
      tab.slot_w[t * top_k + r] = w;
      atomicOr(reinterpret_cast<unsigned long long*>(tab.mask) + id, 1ull << t);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // Rows and segments in front of each expert: the sums in one number.
  const uint64_t mine = tid < E ? tab.mask[tid] : 0;
  const int n_rows = __popcll(mine), n_segs = (n_rows + kSegRows - 1) / kSegRows;
  typedef std::conditional_t<(NB > 0), uint64_t, uint32_t> Sums;  // the second kernel's segments are others where x is kept: a third sum
  const Sums own = static_cast<Sums>(n_rows) | static_cast<Sums>(n_segs) << 16 |
                   (NB > 0 ? static_cast<uint64_t>((n_rows + down_rows - 1) / down_rows) << 32 : 0);
  Sums upto = own;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const Sums other = __shfl_up(upto, d);
    if (lane >= d) upto += other;
  }
  if (lane == 63) tab.totals[wave] = upto;
  __syncthreads();
  Sums before = upto - own, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const Sums v = static_cast<Sums>(tab.totals[w]);
    if (w < wave) before += v;
    all += v;
  }
  const int row0 = before & 0xffff, segs_all = __builtin_amdgcn_readfirstlane(static_cast<int>(all >> 16 & 0xffff));
  for (int s = 0; s < n_segs; ++s) {
    const int left = n_rows - kSegRows * s;
    tab.segs[(before >> 16 & 0xffff) + s] = MoeSegment{tid, row0 + kSegRows * s, left < kSegRows ? left : kSegRows};
  }
  if (tid < E) tab.expert_row[tid] = row0;
  __syncthreads();
  // a slot's row: behind its expert's tokens of lower numbers
  for (int i = tid; i < slots; i += kThreads) {
    const int e = tab.slot_id[i], t = i / a.k;
    const int row = tab.expert_row[e] + __popcll(tab.mask[e] & ((1ull << t) - 1));
    tab.row_token[row] = t;
    tab.row_w[row] = tab.slot_w[i];
  }
  __syncthreads();
  char* const ws = static_cast<char*>(a.workspace);
  if (blockIdx.x == 0) {
    MoeSegment* const segs = reinterpret_cast<MoeSegment*>(ws + kSegsAt);
    if constexpr (NB > 0) {
      for (int s = 0; s * down_rows < n_rows; ++s) {
        const int left = n_rows - s * down_rows;
        segs[(before >> 32) + s] = MoeSegment{tid, row0 + s * down_rows, left < down_rows ? left : down_rows};
      }
    } else {
      for (int i = tid; i < segs_all; i += kThreads) segs[i] = tab.segs[i];
    }
    for (int i = tid; i < slots; i += kThreads) reinterpret_cast<int*>(ws + layout.row_token)[i] = tab.row_token[i];
    for (int i = tid; i < (K + 15) / 16; i += kThreads) reinterpret_cast<int*>(ws + layout.tickets)[i] = 0;
    if (tid == 0) *reinterpret_cast<int*>(ws) = NB > 0 ? static_cast<int>(static_cast<uint64_t>(all) >> 32) : segs_all;
  }

  // ---- the product: items of 8 gate rows and their up rows of one segment ----
  const int n_tiles = (I + 7) / 8, items = segs_all * n_tiles;
  // all waves share an item and a workgroup has a run of items, or KW share one and they go around
  const int KW = NB > 0 ? kWaves : 1 << kw_log2, kw = wave & (KW - 1), nw = NB > 0 ? 0 : wave >> kw_log2;
  const int stride = NB > 0 ? 1 : gridDim.x * (kWaves >> kw_log2);
  const int first = NB > 0 ? static_cast<int>(static_cast<int64_t>(items) * blockIdx.x / gridDim.x) : blockIdx.x * (kWaves >> kw_log2) + nw;
  const int rounds = NB > 0 ? static_cast<int>(static_cast<int64_t>(items) * (blockIdx.x + 1) / gridDim.x) - first : (items + stride - 1) / stride;
  const int64_t pitch = static_cast<int64_t>(K) * 2;
  struct Item {
    int e, n0, row0, rows;
    bool there;
  };
  auto item_of = [&](int round) {
    const int i = round * stride + first;
    Item it;
    it.there = round < rounds && i < items;
    const int s = it.there ? i / n_tiles : 0;
    const MoeSegment seg = tab.segs[s];
    it.e = __builtin_amdgcn_readfirstlane(seg.e);
    it.row0 = __builtin_amdgcn_readfirstlane(seg.row0);
    it.rows = __builtin_amdgcn_readfirstlane(seg.rows);
    it.n0 = it.there ? (i - s * n_tiles) * 8 : 0;
    return it;
  };
  const rsrc_t x = dense_buffer(a.x, a.T * pitch);
  auto place_of = [&](int round) {
    const Item it = item_of(round);
    StreamPlace<XG> p;
    p.k = kw * kStreamBlock;
    p.end = it.there ? K : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)  // (inter is a multiple of 8)
      p.w[i] = dense_buffer(reinterpret_cast<const char*>(a.w13) + ((static_cast<int64_t>(it.e) * 2 + i) * I + it.n0) * pitch, 8 * pitch);
    p.x = x;
#pragma unroll
    for (int g = 0; g < XG; ++g) {
      const int c = 8 * g + (lane >> 3);
      p.x_at[g] = c < it.rows ? static_cast<uint32_t>(tab.row_token[it.row0 + c]) * static_cast<uint32_t>(pitch) : kNowhere;
    }
    return p;
  };
  auto done = [&](int round, float4_t (&acc)[TT]) {
    if (KW > 1) {  // (two buffers in turn: one barrier a round)
      stream_join(reinterpret_cast<float4_t*>(rest + kWaves * (NB > 0 ? D * kKeptStage : stream_ring<XG, D>())) + (round & 1) * kWaves * TT * 64, wave, KW, acc);
      if (kw != 0) return;
    }
    const Item it = item_of(round);
    const int n = it.n0 + 4 * (lane >> 4);
    float* const h = reinterpret_cast<float*>(ws + layout.h);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int c = 16 * t + (lane & 15);
      const float4_t g = acc[t], up = stream_up(g);
      if (!it.there || c >= it.rows || lane >= 32) continue;
      const int row = it.row0 + c;
      const float w = tab.row_w[row];
      float f[4] = {g[0], g[1], g[2], g[3]};
      dense_act<4>(f, a.act);
      *reinterpret_cast<float4_t*>(h + static_cast<int64_t>(row) * I + n) =
          float4_t{w * (f[0] * up[0]), w * (f[1] * up[1]), w * (f[2] * up[2]), w * (f[3] * up[3])};
    }
  };
  __syncthreads();  // (the routing's part of LDS is the rings' now)
  if constexpr (NB == 0) {
    dense_stream<BF, XG, D, false>(rest + wave * stream_ring<XG, D>(), static_cast<uint32_t>(pitch), KW * kStreamBlock, nb, rounds, place_of, done);
  } else {
    auto rows_of = [&](int round) {
      const Item it = item_of(round);
      StreamRows p;
      p.end = it.there ? K : 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        p.w[i] = dense_buffer(reinterpret_cast<const char*>(a.w13) + ((static_cast<int64_t>(it.e) * 2 + i) * I + it.n0) * pitch, 8 * pitch);
      return p;
    };
    int kept = -1;  // first row of the segment
    auto keep = [&](int round, StreamKept<NB, TT>& of) {
      const Item it = item_of(round);
      if (it.row0 == kept) return;
      kept = it.row0;
      uint32_t at[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const int c = 16 * t + (lane & 15);
        at[t] = c < it.rows ? static_cast<uint32_t>(tab.row_token[it.row0 + c]) * static_cast<uint32_t>(pitch) : kNowhere;
      }
      kept_x(of, x, at, wave * kStreamBlock, kWaves * kStreamBlock, K);
    };
    dense_stream_kept<BF, TT, NB, D>(rest + wave * D * kKeptStage, static_cast<uint32_t>(pitch), wave * kStreamBlock, kWaves * kStreamBlock, rounds,
                                     rows_of, keep, done);
  }
}

template <bool BF>
__device__ __forceinline__ void moe_store(uint16_t* to, const float4_t& v) {
  *reinterpret_cast<uint2*>(to) = uint2{dense_pair<BF>(v[0], v[1]), dense_pair<BF>(v[2], v[3])};
}

// Eight float32 numbers as 16-bit planes for the matrix instruction.
// bfloat16: three planes, the upper 16 bits of what is left each time, which is all 24 bits of the number.
// float16: two planes of v = scale f, a power of two times the number: v rounded, and what that left rounded.  Together they are off by at most 2^-23 of v, or
// 2^-25 where that is more; a row's largest v is between 4 and 2^15, so that this is 2^-27 of it.  (float32, of which they take the place, has 2^-24 of v.)
template <bool BF>
struct DownPlanes {
  int4_t v[BF ? 3 : 2];
};
template <bool BF>
__device__ __forceinline__ DownPlanes<BF> down_planes(const float* f, float scale) {
  DownPlanes<BF> p;
  float minus = -1.f;
  asm("" : "+s"(minus));  // (not folded into a subtraction, which would widen its float16 operand first)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = f[2 * i], b = f[2 * i + 1];
    if constexpr (BF) {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const uint32_t ua = __builtin_bit_cast(uint32_t, a), ub = __builtin_bit_cast(uint32_t, b);
        p.v[j][i] = static_cast<int>(__builtin_amdgcn_perm(ub, ua, 0x07060302u));
        if (j < 2) {
          a -= __builtin_bit_cast(float, ua & 0xffff0000u);
          b -= __builtin_bit_cast(float, ub & 0xffff0000u);
        }
      }
    } else {
      a *= scale;
      b *= scale;
      const uint32_t h = dense_pair<false>(a, b);
      p.v[0][i] = static_cast<int>(h);
      p.v[1][i] = static_cast<int>(dense_pair<false>(__builtin_fmaf(dense_widen<false>(h & 0xffffu), minus, a), __builtin_fmaf(dense_widen<false>(h >> 16), minus, b)));
    }
  }
  return p;
}
// the largest over the four lanes of a row
__device__ __forceinline__ float down_row_max(float v) {
  auto larger = [](uint32_t x, uint32_t y) { return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y))); };
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto sixteens = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = larger(sixteens[0], sixteens[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, larger(halves[0], halves[1]));
}

template <int XG, int C>
constexpr int down_stage() { return C == 1 ? 2048 + 2048 * XG : 2048 * C; }

// 16 C columns of the output for all tokens a workgroup; gridDim.y workgroups share the K, which is all segments' inter.  The activations come through
// LDS beside W, or, with C 2, straight into registers; as float32, of which the wave that multiplies makes 16-bit planes.
template <bool BF, int XG, int D, int C>
__global__ __launch_bounds__(kThreads, XG == 1 && C == 1 && D == 2 ? 4 : 2) void dense_moe_down_kernel(
    const void* __restrict__ from, const int* __restrict__ tokens, const uint16_t* __restrict__ w2, int T, int slots, int H, int I, DenseMoeArgs a,
    MoeLayout layout) {
  static_assert(C == 2 || XG == 1, "eight rows a stage");
  constexpr int TT = (XG + 1) / 2, kStage = down_stage<XG, C>();
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
  char* const ws = static_cast<char*>(a.workspace);
  uint8_t* const ring = smem + wave * D * kStage;
  float4_t* const sums = reinterpret_cast<float4_t*>(smem + kWaves * D * kStage);  // [waves][T][4 C]
  int* const row_token = reinterpret_cast<int*>(sums + kWaves * T * 4 * C);      // [T k]
  MoeSegment* const segs = reinterpret_cast<MoeSegment*>(row_token + slots);     // [T k at most]
  const int n_segs = __builtin_amdgcn_readfirstlane(*static_cast<const int*>(from));
  for (int i = tid; i < slots; i += kThreads) {  // (all that may be there, without a wait for their number)
    row_token[i] = tokens[i];
    segs[i] = reinterpret_cast<const MoeSegment*>(static_cast<const char*>(from) + kSegsAt)[i];
  }
  for (int i = tid; i < kWaves * T * 4 * C; i += kThreads) sums[i] = float4_t{};
  __syncthreads();
  const int n0 = blockIdx.x * 16 * C, per = (I + kStreamBlock - 1) / kStreamBlock;  // blocks a segment
  const int blocks = n_segs * per;
  const int begin = static_cast<int>(static_cast<int64_t>(blocks) * blockIdx.y / gridDim.y);
  const int end = static_cast<int>(static_cast<int64_t>(blocks) * (blockIdx.y + 1) / gridDim.y);
  const uint32_t pitch = static_cast<uint32_t>(I) * 2u, h_pitch = 2u * pitch;  // (below 2^25)
  const uint64_t expert = static_cast<uint64_t>(static_cast<uint32_t>(H)) * pitch;
  const char* const w_first = reinterpret_cast<const char*>(w2) + static_cast<uint64_t>(static_cast<uint32_t>(n0)) * pitch;

  // this wave's blocks: every kWaves-th; (segment, block of it) of the next one to load, and of the one to compute
  struct At {
    int b, i, kb;
  };
  auto next = [&](At& at) {
    at.b += kWaves;
    at.kb += kWaves;
    while (at.kb >= per) {
      at.kb -= per;
      ++at.i;
    }
  };
  At ahead{begin + wave, (begin + wave) / per, (begin + wave) % per}, now = ahead;
  int4_t x_of[C == 2 ? D : 1][TT][2][2];  // [stage][16 rows][half of a block][four numbers]
  MoeSegment coming = segs[ahead.b < end ? ahead.i : 0];  // of the next block to load, read ahead
  auto load = [&](int s) {
    const bool there = ahead.b < end;
    const uint32_t e = __builtin_amdgcn_readfirstlane(coming.e), row0 = __builtin_amdgcn_readfirstlane(coming.row0);
    const int rows = __builtin_amdgcn_readfirstlane(coming.rows);
    rsrc_t w[2 * C];
#pragma unroll
    for (int i = 0; i < 2 * C; ++i)  // (hidden is a multiple of 8)
      w[i] = dense_buffer(w_first + e * expert + static_cast<uint64_t>(8 * i) * pitch, H - n0 > 8 * i ? static_cast<int64_t>(8 * pitch) : 0);
    const rsrc_t h = dense_buffer(ws + layout.h + static_cast<uint64_t>(row0) * h_pitch, static_cast<int64_t>(static_cast<uint32_t>(rows) * h_pitch));
    const int k = ahead.kb * kStreamBlock, last = there ? I : 0;
    const int kc = k + 8 * ((lane & 7) ^ (lane >> 3));
    const uint32_t w_at = kc < last ? static_cast<uint32_t>(lane >> 3) * pitch + 2u * kc : kNowhere;
#pragma unroll
    for (int i = 0; i < 2 * C; ++i) dense_to_lds<true>(w[i], w_at, ring + s * kStage + 1024 * i);
    asm volatile("" ::: "memory");  // (in this order)
    if constexpr (C == 1) {
      // four rows of 256 bytes an instruction, chunk c of four numbers of a row at place c ^ (row & 7)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 4 * i + quad, at_k = k + 4 * ((lane & 15) ^ row);
        const uint32_t at = row < rows && at_k < last ? static_cast<uint32_t>(row) * h_pitch + 4u * at_k : kNowhere;
        dense_to_lds<false>(h, at, ring + s * kStage + 2048 + 1024 * i);
      }
    } else {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const int c = 16 * t + (lane & 15);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at_k = k + 32 * i + 8 * quad;
          const uint32_t at = c < rows && at_k < last ? static_cast<uint32_t>(c) * h_pitch + 4u * at_k : kNowhere;
#pragma unroll
          for (int j = 0; j < 2; ++j) x_of[s][t][i][j] = __builtin_bit_cast(int4_t, __builtin_amdgcn_raw_buffer_load_b128(h, at + 16u * j, 0, 0));
        }
      }
    }
    asm volatile("" ::: "memory");
    next(ahead);
    coming = segs[ahead.b < end ? ahead.i : 0];
  };
  // Sums of the first planes, and of the others: where the first ones' are infinite or NaN, they are the result, and the others', in which an infinity meets
  // zeros and numbers of the other sign, are nothing.
  // C 1: eight rows of x are columns 0 to 7 of the operand with the first half of a block's K and columns 8 to 15 with the second.  The sums of W's first
  // half have the results in columns 0 to 7, those of W's second half in columns 8 to 15, and half the numbers go through down_planes.
  constexpr int NF = C == 1 ? 8 : 16;  // numbers of a lane in a block
  float4_t acc[2][TT], left[2][TT];    // C 1: halves of K, C 2: of the columns
  // float16: the scale of this lane's row of each 16, 2^scale_log2; it starts where it may well stay
  constexpr int kScaleStart = 12, kScaleMost = 126;
  constexpr float kSmallest = 4.f, kLargest = 0x1p15f;
  int scale_log2[TT];
  float scale[TT], small[TT];  // small: kSmallest, or 0 once the lane has met a number other than 0
  auto clear = [&] {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      scale_log2[t] = kScaleStart;
      scale[t] = static_cast<float>(1 << kScaleStart);
      small[t] = kSmallest;
#pragma unroll
      for (int u = 0; u < 2; ++u) acc[u][t] = left[u][t] = float4_t{};
    }
  };
  clear();
  // Moves the scale of the rows, and their sums with it, where a block has numbers that it would bring past kLargest, or none above kSmallest in the first block
  // that is not all zeros.
  auto fit = [&](int t, const float (&f)[NF]) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < NF; ++i) most = fmaxf(most, __builtin_fabsf(f[i]));
    const float v = most * scale[t], was = small[t];
    small[t] = most > 0.f ? 0.f : was;
    if (__any(v >= kLargest || (v < was && most > 0.f)) == 0) return;
    asm volatile("");  // (a branch: few blocks come here)
    if (__any(most == __builtin_inff())) {  // the largest finite one
      most = 0.f;
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        const float v = __builtin_fabsf(f[i]);
        most = v < __builtin_inff() ? fmaxf(most, v) : most;
      }
    }
    most = down_row_max(most);
    const bool first = down_row_max(was == 0.f ? 1.f : 0.f) == 0.f;
    const bool move = most * scale[t] >= kLargest || (first && most > 0.f && most * scale[t] < kSmallest);
    const int fitting = 13 - __builtin_amdgcn_frexp_expf(most);  // to 2^12 to 2^13: there is room above
    const int to = !move ? scale_log2[t] : fitting < kScaleMost ? fitting : kScaleMost, by = to - scale_log2[t];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        acc[u][t][v] = __builtin_amdgcn_ldexpf(acc[u][t][v], by);
        left[u][t][v] = __builtin_amdgcn_ldexpf(left[u][t][v], by);
      }
    scale_log2[t] = to;
    scale[t] = __builtin_amdgcn_ldexpf(1.f, to);
  };
  int token[TT];  // of this lane's row of the segment in hand, -1: none
  auto take = [&](int i) {
    const MoeSegment seg = segs[i];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int c = 16 * t + (lane & 15);
      token[t] = c < seg.rows ? row_token[seg.row0 + c] : -1;
    }
  };
  auto join = [&] {  // the segment's sums go to its tokens'
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float4_t v[C];
#pragma unroll
      for (int u = 0; u < C; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool second = C == 1 && (lane & 8) != 0;  // this lane's half of K
          const float first = second ? acc[1][t][j] : acc[u][t][j], others = second ? left[1][t][j] : left[u][t][j];
          float sum = __builtin_fabsf(first) < __builtin_inff() ? first + others : first;
          if constexpr (!BF) sum = __builtin_amdgcn_ldexpf(sum, -scale_log2[t]);
          if constexpr (C == 1) {
            const int bits = __builtin_bit_cast(int, sum);
            sum += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, bits, 0x128, 0xf, 0xf, false));  // row_ror:8
          }
          v[u][j] = sum;
        }
      if (token[t] >= 0)
#pragma unroll
        for (int u = 0; u < C; ++u) sums[(wave * T + token[t]) * 4 * C + 4 * u + quad] += v[u];
    }
    clear();
  };
#pragma unroll
  for (int s = 0; s < D; ++s) load(s);
  int current = now.i;
  if (now.b < end) take(current);
  while (now.b < end) {
#pragma unroll
    for (int s = 0; s < D; ++s) {
      const int segment = now.b < end ? now.i : current;  // (past the end: zeros)
      constexpr int kLoads = C == 1 ? 4 : 2 * C + 4 * TT;
      static_assert((D - 1) * kLoads < 64, "the counter of loads");
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * kLoads) : "memory");
      const uint8_t* const stage = ring + s * kStage;
      const int row = lane & 15;
      int4_t w[C][2];
#pragma unroll
      for (int u = 0; u < C; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) w[u][i] = *reinterpret_cast<const int4_t*>(stage + 2048 * u + row * 128 + (((quad + 4 * i) ^ (row & 7)) << 4));
      float f[TT][NF];
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int j = 0; j < NF / 4; ++j) {
          float4_t v;
          if constexpr (C == 1) v = *reinterpret_cast<const float4_t*>(stage + 2048 + (row & 7) * 256 + (((row & 8) + ((2 * quad + j) ^ (row & 7))) << 4));
          else v = __builtin_bit_cast(float4_t, x_of[s][t][j / 2][j % 2]);
#pragma unroll
          for (int n = 0; n < 4; ++n) f[t][4 * j + n] = v[n];
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (read, before the stage is loaded again)
      next(now);
      load(s);  // (in front of the arithmetic, so that it has this time as well)
      if (segment != current) {
        join();
        take(segment);
        current = segment;
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        if constexpr (!BF) fit(t, f[t]);
#pragma unroll
        for (int i = 0; i < NF / 8; ++i) {
          const DownPlanes<BF> p = down_planes<BF>(f[t] + 8 * i, scale[t]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int4_t& m = C == 1 ? w[0][u] : w[C - 1 < u ? 0 : u][i];
            acc[u][t] = dense_mfma<BF>(m, p.v[0], acc[u][t]);
            left[u][t] = dense_mfma<BF>(m, p.v[1], left[u][t]);
            if constexpr (BF) left[u][t] = dense_mfma<BF>(m, p.v[2], left[u][t]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // (and none of it behind the next wait)
    }
  }
  if (begin + wave < end) join();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  // The waves' sums in their order: a thread four columns of a token.
  for (int i = tid; i < T * 4 * C; i += kThreads) {
    const int n = n0 + 4 * (i % (4 * C));
    float4_t v = sums[i];
    for (int w = 1; w < kWaves; ++w) v += sums[w * T * 4 * C + i];
    sums[i] = v;
    if (gridDim.y == 1 && n < H) moe_store<BF>(a.out + static_cast<int64_t>(i / (4 * C)) * H + n, v);
  }
  if (gridDim.y == 1) return;
  // Shares of several workgroups: the one that comes last adds them all, in their order.  They go past the L2 of a die (agent-scope stores
  // and loads) and are there before the ticket is drawn; a fence would write back the die's whole L2 instead, which took 100 us.
  float* const shares = reinterpret_cast<float*>(ws + layout.shares);  // [shares][tiles][T][16 C]
  auto share_of = [&](int s) { return shares + (static_cast<int64_t>(s) * gridDim.x + blockIdx.x) * T * 16 * C; };
  for (int i = tid; i < T * 4 * C; i += kThreads)
#pragma unroll
    for (int v = 0; v < 4; ++v) __hip_atomic_store(share_of(blockIdx.y) + 4 * i + v, sums[i][v], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int* const last_one = reinterpret_cast<int*>(smem);  // (the rings are done with)
  if (tid == 0)
    *last_one = __hip_atomic_fetch_add(reinterpret_cast<int*>(ws + layout.tickets) + blockIdx.x, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
               static_cast<int>(gridDim.y) - 1;
  __syncthreads();
  if (!*last_one) return;
  for (int i = tid; i < T * 4 * C; i += kThreads) {
    float4_t v = {};
    for (int s = 0; s < static_cast<int>(gridDim.y); ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += __hip_atomic_load(share_of(s) + 4 * i + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int n = n0 + 4 * (i % (4 * C));
    if (n < H) moe_store<BF>(a.out + static_cast<int64_t>(i / (4 * C)) * H + n, v);
  }
}

int64_t dense_moe_workspace_bytes(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t k) { return moe_layout(T, hidden, inter, experts, k).bytes; }

template <class Kernel>
static hipError_t may_use(Kernel* kern, size_t lds) {
  return lds > 65536 ? allow_large_lds(reinterpret_cast<const void*>(kern)) : hipSuccess;
}

template <bool BF, int NC, int XG, int D, int NB>
static hipError_t launch_up(const DenseMoeArgs& a, const MoeLayout& layout, int down_rows, hipStream_t s) {
  const int slots = a.T * a.k, n_tiles = a.inter / 8;
  const StreamPlan plan = stream_plan(experts_chosen(a.T, a.experts, a.k) * n_tiles, a.hidden, D, false);
  const int64_t most = static_cast<int64_t>(slots < a.experts ? slots : a.experts + slots / (8 * XG)) * n_tiles;  // items
  const int nw = NB > 0 ? 1 : kWaves >> plan.kw_log2;
  const int64_t sets = (most + nw - 1) / nw;
  const size_t tables = moe_tables_bytes(a.experts, slots), gate = kWaves * sizeof(GateScratch<NC>);
  const size_t rings = kWaves * ((NB > 0 ? D * kKeptStage : stream_ring<XG, D>()) + 2 * ((XG + 1) / 2) * 1024), lds = tables + (rings > gate ? rings : gate);
  if (lds > 160 * 1024) return hipErrorNotSupported;
  auto* kern = dense_moe_up_kernel<BF, NC, XG, D, NB>;
  const hipError_t e = may_use(kern, lds);
  if (e != hipSuccess) return e;
  const int vec = a.experts % 8 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15u) == 0;
  const int64_t at_a_time = kStreamUnits * (lds > 80 * 1024 || NB > 0 ? 1 : 2);
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(sets < at_a_time ? sets : at_a_time)), dim3(kThreads), lds, s, a.logits, a.T, a.experts,
                     a.k, a.logits_dtype, vec, static_cast<int>(tables), gate_group_inv(a.experts, a.groups), plan.kw_log2, plan.nb, down_rows, a, layout);
  return hipGetLastError();
}

template <bool BF, int XG, int C>
static hipError_t launch_down(const DenseMoeArgs& a, const MoeLayout& layout, hipStream_t s) {
  constexpr int D = 2;  // (three blocks ahead, C 1: one token of 64 experts of 2048 x 1408 10.5 -> 11.5 us)
  const int shares = moe_shares(a.T, a.hidden, a.inter, a.experts, a.k);
  const dim3 grid(static_cast<unsigned>((a.hidden + 16 * C - 1) / (16 * C)), static_cast<unsigned>(shares));
  note_kernel("dense_moe up to %d rows, %d shares%s", 8 * XG, shares, moe_keeps(a) ? ", x kept" : "");
  const size_t lds = kWaves * (D * down_stage<XG, C>() + static_cast<size_t>(a.T) * 64 * C) + static_cast<size_t>(a.T) * a.k * (4 + sizeof(MoeSegment));
  static_assert(kWaves * (D * down_stage<XG, C>() + kMoeTokens * 64 * C) + kMoeTokens * 32 * (4 + sizeof(MoeSegment)) <= 160 * 1024, "LDS of a unit");
  auto* kern = dense_moe_down_kernel<BF, XG, D, C>;
  const hipError_t e = may_use(kern, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, grid, dim3(kThreads), lds, s, a.workspace,
                     reinterpret_cast<const int*>(static_cast<const char*>(a.workspace) + layout.row_token), a.w2, a.T, a.T * a.k, a.hidden, a.inter, a,
                     layout);
  return hipGetLastError();
}

template <bool BF, int XG>
static hipError_t launch(const DenseMoeArgs& a, hipStream_t s) {
  const MoeLayout layout = moe_layout(a.T, a.hidden, a.inter, a.experts, a.k);
  const int down_rows = moe_down_rows(a);
  auto up = [&](auto xg, auto d, auto nb) {
    constexpr int U = decltype(xg)::value, D = decltype(d)::value, NB = decltype(nb)::value;
    return a.experts <= 64    ? launch_up<BF, 2, U, D, NB>(a, layout, down_rows, s)
           : a.experts <= 128 ? launch_up<BF, 4, U, D, NB>(a, layout, down_rows, s)
           : a.experts <= 256 ? launch_up<BF, 8, U, D, NB>(a, layout, down_rows, s)
                              : launch_up<BF, 16, U, D, NB>(a, layout, down_rows, s);
  };
  const std::integral_constant<int, 0> none{};
  const std::integral_constant<int, 2> two{};
  const std::integral_constant<int, 4> four{};
  const std::integral_constant<int, 8> eight{};
  const std::integral_constant<int, XG> rows{};
  hipError_t e = hipErrorNotSupported;
  if (moe_keeps(a)) e = moe_blocks(a.hidden) == 4 ? up(four, four, four) : up(four, four, eight);
  if (e == hipErrorNotSupported) e = up(rows, four, none);
  if constexpr (XG == 2)
    if (e == hipErrorNotSupported) e = up(rows, two, none);  // (many slots: their tables take the room)
  if (e != hipSuccess) return e;
  if constexpr (XG == 1) return launch_down<BF, 1, 1>(a, layout, s);  // (one token)
  else return down_rows == 32 ? launch_down<BF, 4, 2>(a, layout, s) : launch_down<BF, 2, 2>(a, layout, s);
}

hipError_t launch_dense_moe(const DenseMoeArgs& a, hipStream_t s) {
  const int eights = moe_eights(a.T);
  if (a.bf16) return eights == 1 ? launch<true, 1>(a, s) : launch<true, 2>(a, s);
  return eights == 1 ? launch<false, 1>(a, s) : launch<false, 2>(a, s);
}

}  // namespace gq
