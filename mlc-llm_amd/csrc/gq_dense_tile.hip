// Products with 16-bit weights of more than a few rows: tiles through LDS on v_mfma_f32_16x16x32 or 32x32x16.
#include "gq_dense_common.hpp"

namespace gq {

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr int kBlock = 64;  // numbers of K, 128 bytes of a row

template <bool ONCE>
__device__ __forceinline__ void load_to_lds(rsrc_t rsrc, uint32_t off, uint8_t* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, off, 0, 0, ONCE ? 2 : 0);
}
__device__ __forceinline__ rsrc_t buffer_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes), 0x00027000);
}
// bytes that a tile may reach: rows are below 2^24 bytes, so that a tile's 256 end below what is left of 2^32 at any block of K
__device__ __forceinline__ uint32_t reach(int64_t bytes) { return bytes > 0xffffffffll ? 0xffffffffu : static_cast<uint32_t>(bytes); }

template <int MI>
using TileSums = std::conditional_t<MI == 16, float4_t, float16_t>;  // of a lane
template <bool BF>
__device__ __forceinline__ float4_t tile_mfma(int4_t w, int4_t x, float4_t acc) {
  return dense_mfma<BF>(w, x, acc);
}
template <bool BF>
__device__ __forceinline__ float16_t tile_mfma(int4_t w, int4_t x, float16_t acc) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, w), __builtin_bit_cast(bf16x8_t, x), acc, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, w), __builtin_bit_cast(half8_t, x), acc, 0, 0, 0);
}

}  // namespace

// WN x WM waves, each TN x TM results of MI x MI: a tile of BN = MI WN TN rows of W by BM = MI WM TM rows of x.
// GATED: half of a wave's rows of W are gate rows and half the up rows that belong to them.
// WS stages of W in LDS: three, so that W is two blocks ahead; or two, one block ahead.
// ONCE: no other workgroup reads these rows of W.
template <bool BF, bool GATED, int MI, int WN, int WM, int TN, int TM, int WS, bool ONCE>
__global__ __launch_bounds__(64 * WN * WM, 2) void dense_tile_kernel(DenseArgs p, int n_first, int n_tiles, int m_tiles, int per_split) {
  constexpr int kWaves = WN * WM, BN = MI * WN * TN, BM = MI * WM * TM, KS = MI / 8;  // KS: instructions to a block
  constexpr int kWLoads = BN / 8 / kWaves, kXLoads = (BM / 8 + kWaves - 1) / kWaves;  // of 1 KiB, eight rows, a wave and block of K
  constexpr int P = GATED ? 2 : 1, kPart = MI * TN / P;  // parts of a wave's rows of W
  constexpr int kWStage = BN * 128, kXStage = kXLoads * kWaves * 1024;  // WS stages of W and two of x in LDS
  static_assert(BN / 8 % kWaves == 0 && kPart % 8 == 0, "whole loads");
  static_assert(TN % 2 == 0, "the first row of a block uses fw[0], and half of the rows are gates");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = static_cast<int>(p.K), N = static_cast<int>(p.N), half = N / P;
  const int blocks = (K + kBlock - 1) / kBlock;

  // Workgroups go to the eight dies in turn; each die takes a run of tiles, x tiles fastest, so that what runs on it at a time
  // shares rows of W and of x in its L2.
  const int tiles = n_tiles * m_tiles, per = (tiles + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || id >= tiles) return;
  const int nt = id / m_tiles, mt = id - nt * m_tiles, n0 = n_first + nt * (BN / P);
  const int64_t r0 = static_cast<int64_t>(mt) * BM;
  const int rows = p.rows - r0 < BM ? static_cast<int>(p.rows - r0) : BM;  // of x in this tile
  // this workgroup's blocks of K
  const int first = blockIdx.y * per_split, last = (first + per_split < blocks ? first + per_split : blocks) - 1;

  // Rows past the end are read from the last one.  A block's loads see the matrix from that block on, and nothing past its end: the last
  // row's bytes past K are zeros, another row's are the next row's, and the last block is masked where it is used.
  const uint32_t pitch = static_cast<uint32_t>(K) * 2u;
  const char* const w0 = reinterpret_cast<const char*>(p.w) + static_cast<int64_t>(n0) * pitch;
  const char* const x0 = reinterpret_cast<const char*>(p.x) + r0 * pitch;
  const uint32_t w_bytes = reach(static_cast<int64_t>(half - n0) * pitch), x_bytes = reach((p.rows - r0) * pitch);
  // row of the tile -> (gate or up, row of W from n0 on)
  auto w_part = [&](int row) { return row % (MI * TN) / kPart; };
  auto w_row = [&](int row) {
    const int n = row / (MI * TN) * kPart + row % kPart;
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
  auto issue_x = [&](int g, int from, int to) {
    const uint32_t k = (g < last ? g : last) * 128u;
    const rsrc_t rsrc = buffer_of(x0 + k, x_bytes - k);
#pragma unroll
    for (int i = from; i < to; ++i) load_to_lds<false>(rsrc, x_off[i], smem + WS * kWStage + (g & 1) * kXStage + (i * kWaves + wave) * 1024);
  };

  const int wn = (wave % WN) * MI * TN, wm = (wave / WN) * MI * TM, frow = lane & (MI - 1), fpart = lane / MI;
  typedef TileSums<MI> Acc;
  Acc acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = Acc{};

  struct Operand {
    int4_t v[KS];  // chunks fpart, fpart + 64 / MI, ... of a row
  };
  auto frag = [&](const uint8_t* stage, int g, int row, auto tail) {
    const uint8_t* base = stage + row * 128;
    Operand o;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int c = fpart + s * (64 / MI);
      o.v[s] = *reinterpret_cast<const int4_t*>(base + ((c ^ (row & 7)) << 4));
      if constexpr (decltype(tail)::value) {  // (K is a multiple of 8)
        if (g * kBlock + 8 * c >= K) o.v[s] = int4_t{};
      }
    }
    return o;
  };
  Operand fx[TM], fw[2];
  int w_now = 0, w_then = kWStage, w_last = 2 * kWStage;  // stages of W of this block, the next and the one behind it
  auto frag_w = [&](int g, int slot, int i, auto tail) { return frag(smem + slot, g, wn + MI * i + frow, tail); };
  auto frag_x = [&](int g, int j, auto tail) { return frag(smem + WS * kWStage + (g & 1) * kXStage, g, wm + MI * j + frow, tail); };
  // Waits for block g's stages and hands them over.  Loads come back in order, and the last ones asked for (WS 3) are W of the block behind
  // it, which may still be on their way: W comes from memory and is two blocks ahead, x from the L2 and one.  Every wave has read the
  // block before by then, whose stages take the next loads.
  auto hand_over = [&] {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(WS == 2 ? 0 : kWLoads) : "memory");
    __builtin_amdgcn_s_barrier();
  };
  // One block.  The next stage is handed over in front of the last row of results, so that its first operands arrive while that row is
  // computed.  The next block's loads go out kBurst at a time, the first behind the hand-over and the others in front of the rows: all at
  // once they fill the queue to the vector cache, and every wave waits there in front of its matrix instructions.
  constexpr int kBurst = (kXLoads + 1) / 2 + kWLoads / 2 <= TN ? 2 : 4, kXBursts = (kXLoads + kBurst - 1) / kBurst, kBursts = kXBursts + kWLoads / kBurst;
  static_assert(kWLoads % kBurst == 0 && kBursts <= TN, "every burst has a row");
  auto burst = [&](int i, int g, int w_slot) {  // burst i of x of block g and W of block g + WS - 2
    if (i < kXBursts) issue_x(g, i * kBurst, (i + 1) * kBurst < kXLoads ? (i + 1) * kBurst : kXLoads);
    else if (i < kBursts) issue_w(g + WS - 2, w_slot, (i - kXBursts) * kBurst, (i - kXBursts + 1) * kBurst);
  };
  auto next_stage = [&] {
    const int freed = w_now;
    w_now = w_then;
    w_then = WS == 2 ? freed : w_last;
    w_last = freed;
  };
  auto step = [&](int g, auto tail, auto next_tail, auto has_next) {
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      if (i + 1 < TN) {
        fw[(i + 1) & 1] = frag_w(g, w_now, i + 1, tail);
      } else if (decltype(has_next)::value) {
        hand_over();
        fw[0] = frag_w(g + 1, w_then, 0, next_tail);
        burst(0, g + 2, w_now);
      }
      if (decltype(has_next)::value && i + 1 < TN) burst(i + 1, g + 1, WS == 2 ? w_then : w_last);
      __builtin_amdgcn_sched_barrier(0);  // (loads first: they have the row's time)
      __builtin_amdgcn_s_setprio(1);      // (a wave with its operands goes before one that asks for them)
#pragma unroll
      for (int j = 0; j < TM; ++j) {
#pragma unroll
        for (int s = 0; s < KS; ++s) acc[i][j] = tile_mfma<BF>(fw[i & 1].v[s], fx[j].v[s], acc[i][j]);
        if (i + 1 == TN && decltype(has_next)::value) {
          fx[j] = frag_x(g + 1, j, next_tail);
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
  issue_w(first, w_now, 0, kWLoads);
  issue_x(first, 0, kXLoads);
  asm volatile("" ::: "memory");  // (in this order)
  if (WS == 3) issue_w(first + 1, w_then, 0, kWLoads);
  hand_over();
  burst(0, first + 1, w_last);
  if (wm < rows) {
    auto begin = [&](auto tail) {
      fw[0] = frag_w(first, w_now, 0, tail);
#pragma unroll
      for (int j = 0; j < TM; ++j) fx[j] = frag_x(first, j, tail);
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
      for (int i = 1; i < kBursts; ++i) burst(i, g + 1, WS == 2 ? w_then : w_last);
      hand_over();
      burst(0, g + 2, w_now);
      next_stage();
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads that nobody reads may still land in the stages
  __syncthreads();  // (and the last stage has been read)

  // The results change hands through LDS, MI rows of x at a time and each wave in a part of its own, so that a row's columns go out as runs of
  // eight a lane; float32 until the epilogue is through.
  constexpr int kCols = MI * TN, kRow = kCols + 4, kLanes = kPart / 8, kRows = 64 / kLanes < MI ? 64 / kLanes : MI;
  float* const mine = reinterpret_cast<float*>(smem) + wave * MI * kRow;
  const bool share = gridDim.y > 1;
  float* const to = static_cast<float*>(p.workspace) + (blockIdx.y * p.rows + r0) * N;
#pragma unroll
  for (int j = 0; j < TM; ++j) {
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int q = 0; q < MI * MI / 256; ++q) {
        float4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
        *reinterpret_cast<float4_t*>(mine + frow * kRow + MI * i + (MI == 16 ? 4 * fpart : 8 * q + 4 * fpart)) = v;
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < (MI + kRows - 1) / kRows; ++t) {
      const int row = t * kRows + lane / kLanes, col = (lane % kLanes) * 8, r = wm + MI * j + row;
      const int n = n0 + (wave % WN) * kPart + col;
      if (row < MI && lane / kLanes < kRows && r < rows && n < half) {
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
          dense_store<8, GATED>(p, r0 + r, n, o[0], o[P - 1]);
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

// the sums of the shares of K, in their order, and the epilogue.  Four columns a thread.
template <bool GATED>
__global__ __launch_bounds__(256) void dense_join_kernel(DenseArgs p, int splits) {
  const int N = static_cast<int>(p.N), cols = GATED ? N / 2 : N, runs = (cols + 3) / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.rows * runs) return;
  const int64_t r = i / runs;
  const int n = static_cast<int>(i - r * runs) * 4;
  const float* from = static_cast<const float*>(p.workspace) + r * N + n;
  float o[2][4] = {};
  const bool vec = cols % 4 == 0;
  for (int s = 0; s < splits; ++s, from += p.rows * N) {
#pragma unroll
    for (int h = 0; h < (GATED ? 2 : 1); ++h) {
      if (vec) {
        const float4_t a = *reinterpret_cast<const float4_t*>(from + h * cols);
#pragma unroll
        for (int v = 0; v < 4; ++v) o[h][v] += a[v];
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (n + v < cols) o[h][v] += from[h * cols + v];
      }
    }
  }
  dense_store<4, GATED>(p, r, n, o[0], o[GATED ? 1 : 0]);
}

namespace {

// A tile form and the shares of K; from column n_rest on (of W's rows; of y's columns where gated), another form without shares.
struct Plan {
  int form = 0, splits = 1, per_split = 0;
  int64_t n_rest = 0;
  int form_rest = 0;
  float ns = 0.f;
};
// Tiles, workgroups that run at a time, and what a block of K of a round of them takes in ns: alone_ns where few run, full_ns where all
// of them do (L2 and clocks are shared).
struct Form {
  int bn, bm, at_a_time;
  float alone_ns, full_ns;
};
constexpr int kForms = 6;
constexpr Form kForm[kForms] = {{256, 256, 256, 875.f, 1687.f}, {256, 192, 256, 752.f, 1412.f}, {256, 128, 256, 619.f, 927.f},
                                {128, 128, 512, 436.f, 1046.f}, {128, 64, 512, 358.f, 700.f}, {128, 32, 512, 300.f, 500.f}};
constexpr float kRoundNs = 1140.f, kJoinNs = 2000.f, kShareNs = 1.42e-3f;  // a round's ends, the launch that joins, an element of a share
float ns_of(const Form& f, int64_t tiles, int64_t blocks) {
  const int64_t full = tiles / f.at_a_time, rest = tiles - full * f.at_a_time;
  float ns = full * (blocks * f.full_ns + kRoundNs);
  if (rest > 0) ns += blocks * (f.alone_ns + (f.full_ns - f.alone_ns) * rest / f.at_a_time) + kRoundNs;
  return ns;
}
bool may_take(int form) { return options().gemm_variant < 0 || options().gemm_variant >= kForms || options().gemm_variant == form; }
// N: rows of W
Plan plan_of(int64_t rows, int64_t N, int64_t K, bool only_whole = false) {
  const int64_t blocks = (K + kBlock - 1) / kBlock;
  Plan best;
  for (int f = 0; f < kForms; ++f) {
    if (!may_take(f)) continue;
    const int64_t m_tiles = (rows + kForm[f].bm - 1) / kForm[f].bm, n_tiles = (N + kForm[f].bn - 1) / kForm[f].bn, tiles = m_tiles * n_tiles;
    for (int64_t want = 1; want <= 16 && want <= (only_whole || blocks < 4 ? 1 : blocks / 4); ++want) {
      if (options().gemm_split_k > 0 && options().gemm_split_k != want) continue;
      const int64_t per = (blocks + want - 1) / want, splits = (blocks + per - 1) / per;
      const float ns = ns_of(kForm[f], tiles * splits, per) + (splits > 1 ? kJoinNs + splits * rows * N * kShareNs : 0.f);
      if (best.per_split == 0 || ns < best.ns) {
        best = Plan{};
        best.form = f;
        best.splits = static_cast<int>(splits);
        best.per_split = static_cast<int>(per);
        best.ns = ns;
      }
    }
    // whole rounds of this form, and what is left of the last in a form that fills a round of its own
    const int64_t whole = tiles / kForm[f].at_a_time * kForm[f].at_a_time / m_tiles;
    if (!only_whole && options().gemm_split_k <= 1 && whole > 0 && whole < n_tiles) {
      const Plan rest = plan_of(rows, N - whole * kForm[f].bn, K, true);
      const float ns = ns_of(kForm[f], whole * m_tiles, blocks) + rest.ns + 2000.f;
      if (ns < best.ns) {
        best = Plan{};
        best.form = f;
        best.per_split = static_cast<int>(blocks);
        best.n_rest = whole * kForm[f].bn;
        best.form_rest = rest.form;
        best.ns = ns;
      }
    }
  }
  return best;
}

template <bool BF, bool GATED, int MI, int WN, int WM, int TN, int TM, int WS, bool ONCE>
hipError_t launch_tile(const DenseArgs& a, const Plan& plan, int part, hipStream_t s) {
  constexpr int P = GATED ? 2 : 1, BN = MI * WN * TN / P, BM = MI * WM * TM, kWaves = WN * WM;  // (BN: columns of y)
  constexpr size_t stages = size_t(WS * BN * P) * 128 + 2 * ((BM / 8 + kWaves - 1) / kWaves * kWaves * 1024), results = size_t(kWaves) * MI * (MI * TN + 4) * 4;
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
  auto* kern = dense_tile_kernel<BF, GATED, MI, WN, WM, TN, TM, WS, ONCE>;
  if (lds > 65536) {
    const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern));
    if (e != hipSuccess) return e;
  }
  note_kernel("dense_tile %dx%d%s, %d shares of K", BN * P, BM, GATED ? " gated" : "", splits);
  const int64_t most = (0xffffffffll / (64 * kWaves) - 8) / m_tiles;  // columns of tiles a launch, likewise
  if (most < 1) return hipErrorNotSupported;
  for (int64_t t0 = 0; t0 < n_tiles; t0 += most) {
    const int64_t here = n_tiles - t0 < most ? n_tiles - t0 : most;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((here * m_tiles + 7) / 8 * 8), splits), dim3(64 * kWaves), lds, s, a,
                       static_cast<int>(n_first + t0 * BN), static_cast<int>(here), static_cast<int>(m_tiles), per_split);
  }
  if (splits > 1) hipLaunchKernelGGL(dense_join_kernel<GATED>, dim3(static_cast<unsigned>((joined + 255) / 256)), dim3(256), 0, s, a, splits);
  return hipGetLastError();
}

template <bool BF, bool GATED>
hipError_t launch_part(const DenseArgs& a, const Plan& plan, int part, hipStream_t s) {
  const int form = part == 0 ? plan.form : plan.form_rest;
  switch (form) {
    case 0: return launch_tile<BF, GATED, 16, 2, 4, 8, 4, 3, false>(a, plan, part, s);
    case 1: return launch_tile<BF, GATED, 16, 4, 2, 4, 6, 3, false>(a, plan, part, s);
    case 2: return launch_tile<BF, GATED, 16, 4, 2, 4, 4, 3, false>(a, plan, part, s);
    case 3: return launch_tile<BF, GATED, 16, 2, 2, 4, 4, 3, false>(a, plan, part, s);
    case 4: return a.rows <= 64 ? launch_tile<BF, GATED, 16, 2, 2, 4, 2, 3, true>(a, plan, part, s) : launch_tile<BF, GATED, 16, 2, 2, 4, 2, 3, false>(a, plan, part, s);
    default: return a.rows <= 32 ? launch_tile<BF, GATED, 16, 4, 1, 2, 2, 3, true>(a, plan, part, s) : launch_tile<BF, GATED, 16, 4, 1, 2, 2, 3, false>(a, plan, part, s);
  }
}

}  // namespace

int64_t dense_tile_workspace_bytes(int64_t rows, int64_t N, int64_t K) {
  const Plan p = plan_of(rows, N, K);
  return p.splits > 1 ? p.splits * rows * N * 4 : 0;
}

hipError_t launch_dense_tile(const DenseArgs& a, hipStream_t s) {
  const Plan plan = plan_of(a.rows, a.N, a.K);
  auto go = [&](int part) {
    if (a.bf16) return a.gated ? launch_part<true, true>(a, plan, part, s) : launch_part<true, false>(a, plan, part, s);
    return a.gated ? launch_part<false, true>(a, plan, part, s) : launch_part<false, false>(a, plan, part, s);
  };
  const hipError_t e = go(0);
  return e != hipSuccess || plan.n_rest == 0 ? e : go(1);
}

}  // namespace gq
