// Products with 16-bit weights of more than a few rows: tiles through LDS on v_mfma_f32_16x16x32.
//
// Large ones are bound by the matrix pipe and the card's power: 256 x 256 tiles of 8192 x 8192 x 8192 keep the pipe 66 % busy at 1.79 GHz, 1395 TFLOP/s;
// 2048 rows of 28672 x 4096, gated, 355 to 369 us, by card (1305 to 1355 TFLOP/s), of 14336 x 4096 with bias and gelu 205 to 218.  The 32x32x16 instruction, with half the reads of operands, lets the
// clock fall further and came out 3 to 8 % slower.  Below some 200 rows the bound is HBM: 48 rows of 4096 x 14336 26.0 us (4.5 TB/s of weights, the join
// included), 16 of 128256 x 4096 163 (6.4).
#pragma once

#include "gq_dense_common.hpp"

namespace gq {

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr int kBlock = 64;                  // numbers of K, 128 bytes of a row
constexpr uint32_t kNowhere = 0xfffffff0u;  // past the end of any buffer here, or inside of it

template <bool ONCE>
__device__ __forceinline__ void load_to_lds(rsrc_t rsrc, uint32_t off, uint8_t* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, off, 0, 0, ONCE ? 2 : 0);
}
__device__ __forceinline__ rsrc_t buffer_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes), 0x00027000);
}
// bytes that a tile may reach: rows are below 2^24 bytes, so that a tile's 256 end below what is left of 2^32 at any block of K
__device__ __forceinline__ uint32_t reach(int64_t bytes) { return bytes > 0xffffffffll ? 0xffffffffu : static_cast<uint32_t>(bytes); }

// loads that go out at a time where there are `rows` times to send them
constexpr int burst_of(int w_loads, int x_loads, int rows) {
  int burst = 2;
  while ((w_loads + burst - 1) / burst + (x_loads + burst - 1) / burst > rows) burst *= 2;
  return burst;
}
}  // namespace

// WN x WM waves, each TN x TM results of 16 x 16: a tile of BN = 16 WN TN rows of W by BM = 16 WM TM rows of x.
// GATED: half of a wave's rows of W are gate rows and half the up rows that belong to them.
// WS stages of W and XS of x in LDS: W is WS - 1 blocks ahead, x XS - 1.
// ONCE: no other workgroup reads these rows of W.
template <bool BF, bool GATED, int WN, int WM, int TN, int TM, int WS, int XS, bool ONCE>
__global__ __launch_bounds__(64 * WN * WM, 2) void dense_tile_kernel(DenseArgs p, int n_first, int n_tiles, int m_tiles, int splits, int per_split) {
  constexpr int kWaves = WN * WM, BN = 16 * WN * TN, BM = 16 * WM * TM;
  constexpr int kWLoads = BN / 8 / kWaves, kXLoads = (BM / 8 + kWaves - 1) / kWaves;  // of 1 KiB, eight rows, a wave and block of K
  constexpr int P = GATED ? 2 : 1, kPart = 16 * TN / P;  // parts of a wave's rows of W
  constexpr int kWStage = BN * 128, kXStage = kXLoads * kWaves * 1024;  // of a block
  static_assert(XS == WS || XS == WS - 1, "hand_over's count");
  static_assert(BN / 8 % kWaves == 0 && kPart % 8 == 0, "whole loads");
  static_assert(TN % 2 == 0, "the first row of a block uses fw[0], and half of the rows are gates");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = static_cast<int>(p.K), N = static_cast<int>(p.N), half = N / P;
  const int blocks = (K + kBlock - 1) / kBlock;

  // Workgroups go to the eight dies in turn; each die takes a run of tiles, one share of K after the other and x tiles fastest in groups of kGroup:
  // what runs on it at a time is about as many rows of W as of x, which its L2 then holds for all of them.
  const int tiles = n_tiles * m_tiles, per = (tiles * splits + 7) / 8, at = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || at >= tiles * splits) return;
  const int part = at / tiles, id = at - part * tiles;  // this workgroup's share
  constexpr int kGroup = 8;
  const int group = id / (kGroup * n_tiles), m_first = group * kGroup, m_here = m_tiles - m_first < kGroup ? m_tiles - m_first : kGroup;
  const int in_group = id - group * kGroup * n_tiles, nt = in_group / m_here, mt = m_first + in_group - nt * m_here, n0 = n_first + nt * (BN / P);
  const int64_t r0 = static_cast<int64_t>(mt) * BM;
  const int rows = p.rows - r0 < BM ? static_cast<int>(p.rows - r0) : BM;  // of x in this tile
  // this workgroup's blocks of K
  const int first = part * per_split, last = (first + per_split < blocks ? first + per_split : blocks) - 1;

  // Rows past the end are read from the last one.  A block's loads see the matrix from that block on, and nothing past its end: the last
  // row's bytes past K are zeros, another row's are the next row's, and the last block is masked where it is used.
  const uint32_t pitch = static_cast<uint32_t>(K) * 2u;
  const char* const w0 = reinterpret_cast<const char*>(p.w) + static_cast<int64_t>(n0) * pitch;
  const char* const x0 = reinterpret_cast<const char*>(p.x) + r0 * pitch;
  const uint32_t w_bytes = reach(static_cast<int64_t>(half - n0) * pitch), x_bytes = reach((p.rows - r0) * pitch);
  // row of the tile -> (gate or up, row of W from n0 on)
  auto w_part = [&](int row) { return row % (16 * TN) / kPart; };
  auto w_row = [&](int row) {
    const int n = row / (16 * TN) * kPart + row % kPart;
    return n0 + n < half ? n : half - 1 - n0;
  };

  // A row of a stage is 128 bytes, its chunk c of 16 at place c ^ (row & 7), and a lane loads the chunk that belongs at its
  // place: eight rows of a chunk, which LDS serves at a time, meet all banks.
  uint32_t w_off[kWLoads], x_off[kXLoads];
  const int my_chunk = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
  for (int i = 0; i < kWLoads; ++i) {
    w_off[i] = static_cast<uint32_t>(w_row((i * kWaves + wave) * 8 + (lane >> 3))) * pitch + my_chunk;
    asm volatile("" : "+v"(w_off[i]));  // (kept as it is, not computed again at every load)
  }
#pragma unroll
  for (int i = 0; i < kXLoads; ++i) {
    const int r = (i * kWaves + wave) * 8 + (lane >> 3);
    x_off[i] = static_cast<uint32_t>(r < rows ? r : rows - 1) * pitch + my_chunk;
    if (BM % (8 * kWaves) != 0 && r >= BM) x_off[i] = kNowhere;  // (a load for the count of loads alone)
    asm volatile("" : "+v"(x_off[i]));
  }
  // Loads [from, to) of block g; past the last block, that one's again (nobody reads them).  No branches and no vector instructions
  // for addresses: the loop below is to stay one run of matrix instructions.
  auto issue_w = [&](int g, int slot, int from, int to) {
    const uint32_t k = (g < last ? g : last) * 128u;
#pragma unroll
    for (int i = from; i < to; ++i) {
      const int64_t up = GATED && w_part((i * kWaves + wave) * 8) != 0 ? static_cast<int64_t>(half) * pitch : 0;
      load_to_lds<ONCE>(buffer_of(w0 + up + k, w_bytes - k), w_off[i], smem + slot + (i * kWaves + wave) * 1024);
    }
  };
  auto issue_x = [&](int g, int slot, int from, int to) {
    const uint32_t k = (g < last ? g : last) * 128u;
    const rsrc_t rsrc = buffer_of(x0 + k, x_bytes - k);
#pragma unroll
    for (int i = from; i < to; ++i) load_to_lds<false>(rsrc, x_off[i], smem + WS * kWStage + slot + (i * kWaves + wave) * 1024);
  };

  const int wn = (wave % WN) * 16 * TN, wm = (wave / WN) * 16 * TM, frow = lane & 15, fpart = lane >> 4;
  float4_t acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = float4_t{};

  struct Operand {
    int4_t v[2];  // chunks fpart and fpart + 4 of a row
  };
  auto frag = [&](const uint8_t* stage, int g, int row, auto tail) {
    const uint8_t* base = stage + row * 128;
    Operand o;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int c = fpart + 4 * s;
      o.v[s] = *reinterpret_cast<const int4_t*>(base + ((c ^ (row & 7)) << 4));
      if constexpr (decltype(tail)::value) {  // (K is a multiple of 8)
        if (g * kBlock + 8 * c >= K) o.v[s] = int4_t{};
      }
    }
    return o;
  };
  Operand fx[TM], fw[2];
  // Where block g's stages are, the next block's, and those of the block before, which take the loads of block g + WS - 1 (XS - 1).
  int w_now = 0, x_now = 0;
  auto after = [](int slot, int stage, int count) { return slot + stage == count * stage ? 0 : slot + stage; };
  auto before = [](int slot, int stage, int count) { return (slot == 0 ? count * stage : slot) - stage; };
  auto frag_w = [&](int g, int slot, int i, auto tail) { return frag(smem + slot, g, wn + 16 * i + frow, tail); };
  auto frag_x = [&](int g, int slot, int j, auto tail) { return frag(smem + WS * kWStage + slot, g, wm + 16 * j + frow, tail); };
  // Waits for the next block's stages and hands them over.  Loads come back in order; those of the blocks behind it may still be on
  // their way.  Every wave has read the block before by then, whose stages take the next loads.
  auto hand_over = [&] {
    constexpr int kNewer = XS == WS ? (XS - 2) * (kWLoads + kXLoads) : kWLoads + (XS - 2) * (kWLoads + kXLoads);
    static_assert(kNewer < 64, "the counter of loads");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kNewer) : "memory");
    __builtin_amdgcn_s_barrier();
  };
  // One block.  The next stage is handed over in front of the last row of results, so that its first operands arrive while that row is
  // computed.  The next loads go out kBurst at a time, the first behind the hand-over and the others in front of the rows: all at
  // once they fill the queue to the vector cache, and every wave waits there in front of its matrix instructions.
  constexpr int kBurst = burst_of(kWLoads, kXLoads, TN), kXBursts = (kXLoads + kBurst - 1) / kBurst, kBursts = kXBursts + (kWLoads + kBurst - 1) / kBurst;
  static_assert(kBursts <= TN, "every burst has a row");
  auto burst = [&](int i, int g, int w_slot, int x_slot) {  // burst i of those that go out while block g is computed
    const int from = (i < kXBursts ? i : i - kXBursts) * kBurst, to = from + kBurst;
    if (i < kXBursts) issue_x(g + XS - 1, x_slot, from, to < kXLoads ? to : kXLoads);
    else if (i < kBursts) issue_w(g + WS - 1, w_slot, from, to < kWLoads ? to : kWLoads);
  };
  auto next_stage = [&] {
    w_now = after(w_now, kWStage, WS);
    x_now = after(x_now, kXStage, XS);
  };
  auto step = [&](int g, auto tail, auto next_tail, auto has_next) {
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      if (i + 1 < TN) {
        fw[(i + 1) & 1] = frag_w(g, w_now, i + 1, tail);
      } else if (decltype(has_next)::value) {
        hand_over();
        fw[0] = frag_w(g + 1, after(w_now, kWStage, WS), 0, next_tail);
        burst(0, g + 1, w_now, x_now);
      }
      if (decltype(has_next)::value && i + 1 < TN) burst(i + 1, g, before(w_now, kWStage, WS), before(x_now, kXStage, XS));
      __builtin_amdgcn_sched_barrier(0);  // (loads first: they have the row's time)
      __builtin_amdgcn_s_setprio(1);      // (a wave with its operands goes before one that asks for them)
#pragma unroll
      for (int j = 0; j < TM; ++j) {
#pragma unroll
        for (int s = 0; s < 2; ++s) acc[i][j] = dense_mfma<BF>(fw[i & 1].v[s], fx[j].v[s], acc[i][j]);
        if (i + 1 == TN && decltype(has_next)::value) {
          fx[j] = frag_x(g + 1, after(x_now, kXStage, XS), j, next_tail);
          __builtin_amdgcn_sched_barrier(0);  // (at once, not behind the row's other instructions)
        }
      }
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);  // rows in this order: operands of all rows at once would not fit the registers
    }
    next_stage();
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
#pragma unroll
  for (int i = 0; i < WS - 1; ++i) {  // the blocks that are on their way, x in front of the W that is asked for with it
    if (XS == WS || i < XS - 1) issue_x(first + i, i * kXStage, 0, kXLoads);
    asm volatile("" ::: "memory");  // (in this order)
    issue_w(first + i, i * kWStage, 0, kWLoads);
    asm volatile("" ::: "memory");
  }
  hand_over();
  burst(0, first, (WS - 1) * kWStage, (XS - 1) * kXStage);
  if (wm < rows) {
    auto begin = [&](auto tail) {
      fw[0] = frag_w(first, w_now, 0, tail);
#pragma unroll
      for (int j = 0; j < TM; ++j) fx[j] = frag_x(first, x_now, j, tail);
    };
    // the last block is masked, whether K ends inside it or not: one form of it, once a tile
    if (first == last) begin(yes);
    else begin(no);
    for (int g = first; g < last - 1; ++g) step(g, no, no, yes);
    if (first < last) step(last - 1, no, yes, yes);
    step(last, yes, no, no);
  } else {
    // none of this wave's rows of x exist: it only brings its part of the stages
    for (int g = first; g < last; ++g) {
#pragma unroll
      for (int i = 1; i < kBursts; ++i) burst(i, g, before(w_now, kWStage, WS), before(x_now, kXStage, XS));
      hand_over();
      burst(0, g + 1, w_now, x_now);
      next_stage();
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads that nobody reads may still land in the stages
  __syncthreads();  // (and the last stage has been read)

  // The results change hands through LDS, 16 rows of x at a time and each wave in a part of its own, so that a row's columns go out as runs of
  // eight a lane; float32 until the epilogue is through.
  constexpr int kRow = 16 * TN + 4, kLanes = kPart / 8, kRows = 64 / kLanes < 16 ? 64 / kLanes : 16;
  float* const mine = reinterpret_cast<float*>(smem) + wave * 16 * kRow;
  const bool share = splits > 1;
  const int n = n0 + (wave % WN) * kPart + (lane % kLanes) * 8;  // this lane's eight columns, in every row that it stores
  float bias[P][8] = {};
  const bool biased = !share && p.bias != nullptr;
  if (biased && n < half) {
#pragma unroll
    for (int i = 0; i < P; ++i) dense_add_run<BF, 8>(p, p.bias + i * half + n, half - n < 8 ? half - n : 8, bias[i]);
  }
  float* const to = static_cast<float*>(p.workspace) + (part * p.rows + r0) * N;
#pragma unroll
  for (int j = 0; j < TM; ++j) {
#pragma unroll
    for (int i = 0; i < TN; ++i) *reinterpret_cast<float4_t*>(mine + frow * kRow + 16 * i + 4 * fpart) = acc[i][j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < (16 + kRows - 1) / kRows; ++t) {
      const int row = t * kRows + lane / kLanes, col = (lane % kLanes) * 8, r = wm + 16 * j + row;
      if (row < 16 && lane / kLanes < kRows && r < rows && n < half) {
        float o[2][8];
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
          for (int v = 0; v < 8; v += 4) {
            const float4_t a = *reinterpret_cast<const float4_t*>(mine + row * kRow + i * kPart + col + v);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][v + e] = a[e];
          }
        if (!share) {
          if (biased) {
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
              for (int v = 0; v < 8; ++v) o[i][v] += bias[i][v];
          }
          dense_finish<BF, 8, GATED>(p, r0 + r, n, o[0], o[P - 1]);
        } else {  // a share of K: its sums go to the scratch as they are
          for (int i = 0; i < P; ++i) {
            float* const at = to + static_cast<int64_t>(r) * N + i * half + n;
            if (half % 4 == 0) {
#pragma unroll
              for (int v = 0; v < 8; v += 4)
                if (n + v < half) *reinterpret_cast<float4_t*>(at + v) = float4_t{o[i][v], o[i][v + 1], o[i][v + 2], o[i][v + 3]};
            } else {
#pragma unroll
              for (int v = 0; v < 8; ++v)
                if (n + v < half) at[v] = o[i][v];
            }
          }
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// A tile form and the shares of K; from column n_rest on (of W's rows), another form without shares.
struct DensePlan {
  int form = 0, splits = 1, per_split = 0;
  int64_t n_rest = 0;
  int form_rest = 0;
  float ns = 0.f;
};
// part 0: the columns of `form`; part 1: those of `form_rest`
hipError_t launch_dense_part_f16(const DenseArgs& a, const DensePlan& plan, int part, hipStream_t s);
hipError_t launch_dense_part_bf16(const DenseArgs& a, const DensePlan& plan, int part, hipStream_t s);
hipError_t launch_dense_join(const DenseArgs& a, int splits, hipStream_t s);

namespace {

template <bool BF, bool GATED, int WN, int WM, int TN, int TM, int WS, int XS, bool ONCE>
hipError_t launch_tile(const DenseArgs& a, const DensePlan& plan, int part, hipStream_t s) {
  constexpr int P = GATED ? 2 : 1, BN = 16 * WN * TN / P, BM = 16 * WM * TM, kWaves = WN * WM;  // (BN: columns of y)
  constexpr size_t stages = size_t(WS * BN * P) * 128 + XS * ((BM / 8 + kWaves - 1) / kWaves * kWaves * 1024), results = size_t(kWaves) * 16 * (16 * TN + 4) * 4;
  constexpr size_t lds = stages > results ? stages : results;
  static_assert(lds <= 160 * 1024, "LDS of a unit");
  const int64_t blocks = (a.K + kBlock - 1) / kBlock, cols = a.N / P, m_tiles = (a.rows + BM - 1) / BM;
  const int64_t n_first = part == 0 ? 0 : plan.n_rest / P, n_end = part == 0 && plan.n_rest > 0 ? plan.n_rest / P : cols, n_tiles = (n_end - n_first + BN - 1) / BN;
  int splits = 1, per_split = static_cast<int>(blocks);
  const int64_t joined = a.rows * ((cols + 3) / 4);  // work items of the join; 2^32 or more in a launch would wrap, without an error
  if (plan.splits > 1 && a.workspace != nullptr && a.workspace_bytes >= plan.splits * a.rows * a.N * 4 && joined < 0xffffff00ll) {
    splits = plan.splits;
    per_split = plan.per_split;
  }
  auto* kern = dense_tile_kernel<BF, GATED, WN, WM, TN, TM, WS, XS, ONCE>;
  if (lds > 65536) {
    const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern));
    if (e != hipSuccess) return e;
  }
  if (part == 0) note_kernel("dense_tile %dx%d%s, %d shares of K", BN * P, BM, GATED ? " gated" : "", splits);
  else note_kernel("dense_tile %dx%d%s, %d shares of K, rows of W from %lld on", BN * P, BM, GATED ? " gated" : "", splits, static_cast<long long>(plan.n_rest));
  const int64_t most = (0xffffffffll / (64 * kWaves) - 8) / (m_tiles * splits);  // columns of tiles a launch, likewise
  if (most < 1) return hipErrorNotSupported;
  for (int64_t t0 = 0; t0 < n_tiles; t0 += most) {
    const int64_t here = n_tiles - t0 < most ? n_tiles - t0 : most;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((here * m_tiles * splits + 7) / 8 * 8)), dim3(64 * kWaves), lds, s, a,
                       static_cast<int>(n_first + t0 * BN), static_cast<int>(here), static_cast<int>(m_tiles), splits, per_split);
  }
  return splits > 1 ? launch_dense_join(a, splits, s) : hipGetLastError();
}

template <bool BF, bool GATED>
hipError_t launch_form(const DenseArgs& a, const DensePlan& plan, int part, hipStream_t s) {
  switch (part == 0 ? plan.form : plan.form_rest) {  // rows of W x rows of x
    case 0: return launch_tile<BF, GATED, 2, 4, 8, 4, 3, 2, false>(a, plan, part, s);  // 256 x 256
    case 1: return launch_tile<BF, GATED, 4, 2, 4, 6, 3, 2, false>(a, plan, part, s);  // 256 x 192
    case 2: return launch_tile<BF, GATED, 4, 2, 4, 4, 3, 2, false>(a, plan, part, s);  // 256 x 128
    case 3: return launch_tile<BF, GATED, 2, 4, 4, 3, 3, 2, false>(a, plan, part, s);  // 128 x 192
    case 4:  // 128 x 128
      return a.rows <= 128 ? launch_tile<BF, GATED, 4, 2, 2, 4, 4, 4, true>(a, plan, part, s)
                           : launch_tile<BF, GATED, 4, 2, 2, 4, 4, 4, false>(a, plan, part, s);
    case 5: return launch_tile<BF, GATED, 2, 2, 4, 4, 3, 2, false>(a, plan, part, s);  // 128 x 128, two a unit
    case 6:  // 64 x 128
      return a.rows <= 128 ? launch_tile<BF, GATED, 2, 4, 2, 2, 4, 4, true>(a, plan, part, s)
                           : launch_tile<BF, GATED, 2, 4, 2, 2, 4, 4, false>(a, plan, part, s);
    case 7:  // 64 x 64, two a unit
      return a.rows <= 64 ? launch_tile<BF, GATED, 2, 2, 2, 2, 5, 5, true>(a, plan, part, s)
                          : launch_tile<BF, GATED, 2, 2, 2, 2, 5, 5, false>(a, plan, part, s);
    case 8: return launch_tile<BF, GATED, 2, 2, 2, 1, 6, 6, true>(a, plan, part, s);    // 64 x 32, two a unit
    case 9: return launch_tile<BF, GATED, 4, 2, 2, 5, 4, 3, false>(a, plan, part, s);   // 128 x 160
    default: return launch_tile<BF, GATED, 4, 2, 4, 5, 3, 2, false>(a, plan, part, s);  // 256 x 160
  }
}

}  // namespace

}  // namespace gq
