// A mixture-of-experts layer with 16-bit weights on a few tokens, in two kernels.
//
//   y_t = sum over j of w_tj  W2[e_tj] h_tj,  h_tj = act(Wg[e_tj] x_t) * (Wu[e_tj] x_t),  (w, e)_t the routing of token t
//
// The first routes (every workgroup all tokens for itself: a microsecond, where a launch of its own and its results' way through memory
// are three) and streams the gate and up rows of the experts that some token chose past these experts' tokens.  A row of w h, the
// weighted activation of one token and expert, goes to the workspace as two 16-bit numbers, the rounded value and what the rounding
// left, so that the second product loses nothing to it.
// The second streams the down rows.  Its columns of x are the tokens, for every expert: a token that did not choose an expert reads zeros there
// (and its sums of that expert's part are dropped, whatever W holds), so that the sum over a token's experts is the accumulator's.
#include "gq_dense_stream.hpp"
#include "gq_gating.hpp"

namespace gq {

namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr double kTarget = 3000;

struct MoeExpert {
  int e, row0;    // the expert and the first of its rows of h
  uint64_t mask;  // its tokens
};
// The workspace: what the first kernel leaves for the second.
struct MoeLayout {
  int64_t count = 0, experts, tickets, shares, h, bytes;  // offsets; h: [2][T k][inter]
};
__host__ __device__ inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
inline int moe_shares(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t k);
inline MoeLayout moe_layout(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t k) {
  const int64_t slots = T * k, tiles = (hidden + 15) / 16;
  MoeLayout l;
  l.experts = 256;
  l.tickets = l.experts + up256((experts < slots ? experts : slots) * static_cast<int64_t>(sizeof(MoeExpert)));
  l.shares = l.tickets + up256(tiles * 4);
  const int shares = moe_shares(T, hidden, inter, experts, k);
  l.h = l.shares + (shares > 1 ? up256(static_cast<int64_t>(shares) * tiles * T * 64) : 0);
  l.bytes = l.h + up256(2 * slots * inter * 2);
  return l;
}
// experts that some token chooses, where all are alike
inline double experts_chosen(int64_t T, int64_t experts, int64_t k) {
  double none = 1;
  for (int64_t t = 0; t < T; ++t) none *= 1 - static_cast<double>(k) / static_cast<double>(experts);
  return static_cast<double>(experts) * (1 - none);
}
// Workgroups that share the K (all chosen experts' inter) of sixteen columns in the second kernel: about two a unit.
inline int moe_shares(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t k) {
  const int64_t tiles = (hidden + 15) / 16;
  const double blocks = experts_chosen(T, experts, k) * static_cast<double>((inter + kStreamBlock - 1) / kStreamBlock);
  int s = 1;
  while (s < 8 && tiles * s < 400 && blocks / (2 * s) >= 4 * kWaves) s *= 2;
  return s;
}

struct MoeTables {  // in LDS, in front of the rest
  uint64_t* mask;      // [experts] tokens of each
  int* slot_id;        // [T k]
  float* slot_w;       // [T k]
  int* row_token;      // [T k] in the order of the experts
  float* row_w;        // [T k]
  int2* segs;          // [T k at most] up to 16 TT rows of one expert: (expert, first row | rows << 16)
  int* totals;         // [32]
};
__host__ __device__ inline size_t moe_tables_bytes(int experts, int slots) { return (static_cast<size_t>(experts) * 8 + static_cast<size_t>(slots) * 24 + 256 + 15) / 16 * 16; }

}  // namespace

// NC: experts a lane in the routing.  TT: 16 TT tokens of an expert at a time.
template <bool BF, int NC, int TT>
__global__ __launch_bounds__(kThreads, 4) void dense_moe_up_kernel(DenseMoeArgs a, MoeLayout layout, int group_inv, int logits_vec, int kw_log2, int nb) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int NR = 2, D = 2, kTiles = NR * TT;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slots = a.T * a.k, E = a.experts, K = a.hidden, I = a.inter;
  MoeTables tab;
  tab.mask = reinterpret_cast<uint64_t*>(smem);
  tab.slot_id = reinterpret_cast<int*>(tab.mask + E);
  tab.slot_w = reinterpret_cast<float*>(tab.slot_id + slots);
  tab.row_token = reinterpret_cast<int*>(tab.slot_w + slots);
  tab.row_w = reinterpret_cast<float*>(tab.row_token + slots);
  tab.segs = reinterpret_cast<int2*>(tab.row_w + slots);
  tab.totals = reinterpret_cast<int*>(tab.segs + slots);
  uint8_t* const rest = smem + moe_tables_bytes(E, slots);
  GateScratch<NC>& gate = reinterpret_cast<GateScratch<NC>*>(rest)[wave];
  float4_t* const sums = reinterpret_cast<float4_t*>(rest);  // [2][waves][kTiles][64]

  // ---- routing ----
  if (tid < E) tab.mask[tid] = 0;
  __syncthreads();
  const GateRule rule{a.score_bias, E, a.k, a.sigmoid, a.groups, a.top_groups, group_inv, a.renormalize, a.scale};
  for (int t0 = 2 * wave; t0 < a.T; t0 += 2 * kWaves) {
    const int t = t0 + (lane >> 5), r = lane & 31;
    const int from = t < a.T ? t : a.T - 1;
    float score[NC];
    if (a.logits_dtype == MODEL_F32) gate_load<NC, MODEL_F32>(a.logits, from, E, r, logits_vec, score);
    else if (a.logits_dtype == MODEL_BF16) gate_load<NC, MODEL_BF16>(a.logits, from, E, r, logits_vec, score);
    else gate_load<NC, MODEL_F16>(a.logits, from, E, r, logits_vec, score);
    int id;
    const float w = gate_pair<NC>(gate, score, rule, &id);
    if (r < a.k && t < a.T) {
      tab.slot_id[t * a.k + r] = id;
      tab.slot_w[t * a.k + r] = w;
      atomicOr(reinterpret_cast<unsigned long long*>(tab.mask) + id, 1ull << t);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // Rows, segments and chosen experts in front of each expert: three sums in one number of 16 bits each.
  const uint64_t mine = tid < E ? tab.mask[tid] : 0;
  const int n_rows = __popcll(mine), n_segs = (n_rows + 16 * TT - 1) / (16 * TT);
  const uint64_t own = static_cast<uint64_t>(n_rows) | static_cast<uint64_t>(n_segs) << 16 | static_cast<uint64_t>(mine != 0) << 32;
  uint64_t upto = own;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t other = __shfl_up(upto, d);
    if (lane >= d) upto += other;
  }
  uint64_t* const wave_sums = reinterpret_cast<uint64_t*>(tab.totals);  // [8]
  if (lane == 63) wave_sums[wave] = upto;
  __syncthreads();
  uint64_t before = upto - own, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const uint64_t v = wave_sums[w];
    if (w < wave) before += v;
    all += v;
  }
  const int row0 = static_cast<int>(before & 0xffff), segs_all = static_cast<int>(all >> 16 & 0xffff);
  for (int s = 0; s < n_segs; ++s) {
    const int n = n_rows - 16 * TT * s < 16 * TT ? n_rows - 16 * TT * s : 16 * TT;
    tab.segs[static_cast<int>(before >> 16 & 0xffff) + s] = int2{tid, (row0 + 16 * TT * s) | n << 16};
  }
  {
    uint64_t left = mine;
    for (int i = 0; i < n_rows; ++i) {
      const int t = __builtin_ctzll(left);
      left &= left - 1;
      tab.row_token[row0 + i] = t;
      for (int j = 0; j < a.k; ++j)
        if (tab.slot_id[t * a.k + j] == tid) tab.row_w[row0 + i] = tab.slot_w[t * a.k + j];
    }
  }
  char* const ws = static_cast<char*>(a.workspace);
  if (blockIdx.x == 0) {
    if (mine != 0) reinterpret_cast<MoeExpert*>(ws + layout.experts)[before >> 32 & 0xffff] = MoeExpert{tid, row0, mine};
    if (tid == 0) *reinterpret_cast<int*>(ws) = static_cast<int>(all >> 32 & 0xffff);
    for (int i = tid; i < (K + 15) / 16; i += kThreads) reinterpret_cast<int*>(ws + layout.tickets)[i] = 0;
  }
  __syncthreads();

  // ---- the product: items of 16 gate rows and their up rows of one segment ----
  const int KW = 1 << kw_log2, kw = wave & (KW - 1), nw = wave >> kw_log2, NW = kWaves >> kw_log2, stride = gridDim.x * NW;
  const int n_tiles = (I + 15) / 16, items = segs_all * n_tiles, first = blockIdx.x * NW + nw;
  const int rounds = (items + stride - 1) / stride;
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
    const int2 seg = tab.segs[s];
    it.e = __builtin_amdgcn_readfirstlane(seg.x);
    const int v = __builtin_amdgcn_readfirstlane(seg.y);
    it.row0 = v & 0xffff;
    it.rows = v >> 16;
    it.n0 = it.there ? (i - s * n_tiles) * 16 : 0;
    return it;
  };
  auto place_of = [&](int round) {
    const Item it = item_of(round);
    StreamPlace<NR, TT> p;
    p.end = it.there ? K : 0;
    const int64_t left = I - it.n0 < 16 ? I - it.n0 : 16;
#pragma unroll
    for (int i = 0; i < NR; ++i)
      p.w[i] = dense_buffer(reinterpret_cast<const char*>(a.w13) + (static_cast<int64_t>(it.e) * 2 * I + static_cast<int64_t>(i) * I + it.n0) * pitch, left * pitch);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int c = 16 * t + (lane & 15);
      p.x_at[t] = static_cast<uint32_t>(tab.row_token[it.row0 + (c < it.rows ? c : it.rows - 1)]) * static_cast<uint32_t>(pitch);
    }
    return p;
  };
  auto done = [&](int round, float4_t (&acc)[NR][TT]) {
    if (KW > 1) {
      float4_t* const buf = sums + (round & 1) * kWaves * kTiles * 64;
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int t = 0; t < TT; ++t) buf[(wave * kTiles + i * TT + t) * 64 + lane] = acc[i][t];
      __syncthreads();
      if (kw != 0) return;
      for (int w = 1; w < KW; ++w)
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int t = 0; t < TT; ++t) acc[i][t] += buf[((wave + w) * kTiles + i * TT + t) * 64 + lane];
    }
    const Item it = item_of(round);
    const int n = it.n0 + 4 * (lane >> 4);
    uint16_t* const h = reinterpret_cast<uint16_t*>(ws + layout.h);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int c = 16 * t + (lane & 15);
      if (!it.there || c >= it.rows || n >= I) continue;
      const int64_t row = it.row0 + c, at = row * I + n;
      const float w = tab.row_w[row];
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float f = w * (dense_act(acc[0][t][v], a.act) * acc[1][t][v]);
        hi[v] = BF ? f2bf(f) : f2h(f);
        const float rounded = BF ? bf2f(hi[v]) : h2f(hi[v]), rest = f - rounded;
        lo[v] = __builtin_fabsf(rounded) <= 3.402823466e38f ? (BF ? f2bf(rest) : f2h(rest)) : 0u;  // (nothing is left of an infinity)
      }
      *reinterpret_cast<uint2*>(h + at) = uint2{hi[0] | hi[1] << 16, hi[2] | hi[3] << 16};
      *reinterpret_cast<uint2*>(h + static_cast<int64_t>(slots) * I + at) = uint2{lo[0] | lo[1] << 16, lo[2] | lo[3] << 16};
    }
  };
  dense_stream<BF, NR, TT, D>(K, kw, KW, nb, rounds, dense_buffer(a.x, a.T * pitch), place_of, done);
}

// Sixteen columns of the output and all tokens a workgroup, 16 TT of them at most; gridDim.y workgroups share the chosen experts' K.
template <bool BF, int TT>
__global__ __launch_bounds__(kThreads, TT == 1 ? 4 : 2) void dense_moe_down_kernel(DenseMoeArgs a, MoeLayout layout) {
  constexpr int D = 2;
  __shared__ MoeExpert experts[512];
  __shared__ __attribute__((aligned(16))) float4_t sums[kWaves][TT][64];
  __shared__ int last_one;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
  char* const ws = static_cast<char*>(a.workspace);
  const int chosen = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const int*>(ws));
  for (int i = tid; i < chosen; i += kThreads) experts[i] = reinterpret_cast<const MoeExpert*>(ws + layout.experts)[i];
  __syncthreads();
  const int H = a.hidden, I = a.inter, n0 = blockIdx.x * 16, per = (I + kStreamBlock - 1) / kStreamBlock;  // blocks an expert
  const int64_t blocks = static_cast<int64_t>(chosen) * per;
  const int64_t begin = blocks * blockIdx.y / gridDim.y, end = blocks * (blockIdx.y + 1) / gridDim.y;
  const int64_t pitch = static_cast<int64_t>(I) * 2, plane = static_cast<int64_t>(a.T) * a.k * pitch;
  const rsrc_t h_hi = dense_buffer(ws + layout.h, plane), h_lo = dense_buffer(ws + layout.h + plane, plane);
  const int64_t w_bytes = (H - n0 < 16 ? H - n0 : 16) * pitch;
  const uint32_t w_at = static_cast<uint32_t>(lane & 15) * static_cast<uint32_t>(pitch);

  // this wave's blocks: every kWaves-th; (expert, block of it) of the next one to load, and of the one to compute
  struct At {
    int64_t b;
    int i, kb;
  };
  auto next = [&](At& at) {
    at.b += kWaves;
    at.kb += kWaves;
    while (at.kb >= per) {
      at.kb -= per;
      ++at.i;
    }
  };
  At load_at{begin + wave, static_cast<int>((begin + wave) / per), static_cast<int>((begin + wave) % per)}, now = load_at;
  int4_t wq[D][2], hq[D][TT][2], lq[D][TT][2];
  auto load = [&](int s) {
    const bool there = load_at.b < end;
    const MoeExpert ex = experts[there ? load_at.i : 0];
    const int e = __builtin_amdgcn_readfirstlane(ex.e);
    const rsrc_t w = dense_buffer(reinterpret_cast<const char*>(a.w2) + (static_cast<int64_t>(e) * H + n0) * pitch, there ? w_bytes : 0);
    uint32_t row_at[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int token = 16 * t + (lane & 15);
      row_at[t] = there && (ex.mask >> token & 1) ? static_cast<uint32_t>(ex.row0 + __popcll(ex.mask & ((1ull << token) - 1))) * static_cast<uint32_t>(pitch) : kNowhere;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = load_at.kb * kStreamBlock + 32 * h + 8 * quad;
      const bool in = k < I;
      wq[s][h] = dense_chunk(w, in ? w_at + 2u * k : kNowhere);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const uint32_t at = in && row_at[t] != kNowhere ? row_at[t] + 2u * k : kNowhere;
        hq[s][t][h] = dense_chunk(h_hi, at);
        lq[s][t][h] = dense_chunk(h_lo, at);
      }
    }
    next(load_at);
  };
  float4_t acc[TT], part[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) acc[t] = part[t] = float4_t{};
  auto join = [&](int i) {  // the sums of expert i go to the tokens that chose it
    const uint64_t mask = experts[i].mask;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const bool mine = mask >> (16 * t + (lane & 15)) & 1;
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[t][v] += mine ? part[t][v] : 0.f;
      part[t] = float4_t{};
    }
  };
#pragma unroll
  for (int s = 0; s < D; ++s) load(s);
  int current = now.i;
  while (now.b < end) {
#pragma unroll
    for (int s = 0; s < D; ++s) {
      if (now.b < end && now.i != current) {
        join(current);
        current = now.i;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          part[t] = dense_mfma<BF>(wq[s][h], hq[s][t][h], part[t]);
          part[t] = dense_mfma<BF>(wq[s][h], lq[s][t][h], part[t]);
        }
      next(now);
      load(s);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (begin + wave < end) join(current);

#pragma unroll
  for (int t = 0; t < TT; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  // The waves' sums in their order: thread (token, four columns).
  const int token = 16 * (tid >> 6) + (lane & 15), n = n0 + 4 * quad;
  const bool mine = tid < 64 * TT && token < a.T && n < H;
  float4_t v = {};
  if (mine) {
    for (int w = 0; w < kWaves; ++w) v += sums[w][tid >> 6][lane];
  }
  auto store = [&](const float4_t& o) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = BF ? f2bf(o[i]) : f2h(o[i]);
    *reinterpret_cast<uint2*>(a.out + static_cast<int64_t>(token) * H + n) = uint2{u[0] | u[1] << 16, u[2] | u[3] << 16};
  };
  if (gridDim.y == 1) {
    if (mine) store(v);
    return;
  }
  // Shares of several workgroups: the one that comes last adds them all, in their order.
  float4_t* const shares = reinterpret_cast<float4_t*>(ws + layout.shares);  // [shares][tiles][T][4]
  auto place = [&](int s) { return ((static_cast<int64_t>(s) * gridDim.x + blockIdx.x) * a.T + token) * 4 + quad; };
  if (mine) shares[place(blockIdx.y)] = v;
  __threadfence();
  __syncthreads();
  if (tid == 0) last_one = atomicAdd(reinterpret_cast<int*>(ws + layout.tickets) + blockIdx.x, 1) == static_cast<int>(gridDim.y) - 1;
  __syncthreads();
  if (!last_one) return;
  __threadfence();
  if (mine) {
    v = float4_t{};
    for (int s = 0; s < static_cast<int>(gridDim.y); ++s) v += shares[place(s)];
    store(v);
  }
}

int64_t dense_moe_workspace_bytes(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t k) { return moe_layout(T, hidden, inter, experts, k).bytes; }

template <bool BF, int NC, int TT>
static hipError_t launch_up(const DenseMoeArgs& a, const MoeLayout& layout, hipStream_t s) {
  const int slots = a.T * a.k, n_tiles = (a.inter + 15) / 16;
  const StreamPlan plan = stream_plan(experts_chosen(a.T, a.experts, a.k) * n_tiles, a.hidden, 2, kTarget);
  const int64_t most = static_cast<int64_t>(slots < a.experts ? slots : a.experts + slots / (16 * TT)) * n_tiles;  // items
  const int nw = kWaves >> plan.kw_log2;
  const int64_t sets = (most + nw - 1) / nw;
  const size_t sums = plan.kw_log2 > 0 ? 2 * kWaves * 2 * TT * 1024 : 0, gate = kWaves * sizeof(GateScratch<NC>);
  const size_t lds = moe_tables_bytes(a.experts, slots) + (sums > gate ? sums : gate);
  auto* kern = dense_moe_up_kernel<BF, NC, TT>;
  if (lds > 65536) {
    const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern));
    if (e != hipSuccess) return e;
  }
  const int vec = a.experts % 8 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15u) == 0;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(sets < 512 ? sets : 512)), dim3(kThreads), lds, s, a, layout, gate_group_inv(a.experts, a.groups),
                     vec, plan.kw_log2, plan.nb);
  return hipGetLastError();
}

template <bool BF>
static hipError_t launch(const DenseMoeArgs& a, hipStream_t s) {
  const MoeLayout layout = moe_layout(a.T, a.hidden, a.inter, a.experts, a.k);
  auto up = [&](auto nc) {
    constexpr int NC = decltype(nc)::value;
    return a.T <= 16 ? launch_up<BF, NC, 1>(a, layout, s) : launch_up<BF, NC, 2>(a, layout, s);
  };
  hipError_t e = a.experts <= 64    ? up(std::integral_constant<int, 2>{})
                 : a.experts <= 128 ? up(std::integral_constant<int, 4>{})
                 : a.experts <= 256 ? up(std::integral_constant<int, 8>{})
                                    : up(std::integral_constant<int, 16>{});
  if (e != hipSuccess) return e;
  const int shares = moe_shares(a.T, a.hidden, a.inter, a.experts, a.k);
  const dim3 grid(static_cast<unsigned>((a.hidden + 15) / 16), static_cast<unsigned>(shares));
  note_kernel("dense_moe, %d shares", shares);
  auto down = [&](auto* kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, s, a, layout); };
  if (a.T <= 16) down(dense_moe_down_kernel<BF, 1>);
  else if (a.T <= 32) down(dense_moe_down_kernel<BF, 2>);
  else down(dense_moe_down_kernel<BF, 4>);
  return hipGetLastError();
}

hipError_t launch_dense_moe(const DenseMoeArgs& a, hipStream_t s) { return a.bf16 ? launch<true>(a, s) : launch<false>(a, s); }

}  // namespace gq
