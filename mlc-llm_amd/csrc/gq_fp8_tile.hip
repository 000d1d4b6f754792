// e4m3 block-scaled matrix product on the 8-bit matrix instruction (v_mfma_f32_16x16x128_f8f6f4), dense or by expert segments.
//
//   y[r, n] = sum over blocks g of 128 of  xs[g, r] ws[n / 128, g] sum_{k in g} xq[r, k] wq[n, k]
//
// W is the instruction's A operand and x its B operand, so a lane of a 16 x 16 result holds one row r of x and four rows n of
// W: both scales of a block are one number per lane, and a block's sum joins the float32 accumulator with four multiply-adds
// beside its one matrix instruction (32 cycles, the multiply-adds another 16 of the vector unit, which runs beside it).
// What the instruction sums itself is one block of 128: of eight neighbouring products it drops what lies more than 13 bits below
// the largest, and adds such sums in float32 (seen with single products over all positions and sizes); about 1e-5 of a typical
// result, a fiftieth of a float16 rounding.  Blocks join in float32.
#include "gq_fp8_common.hpp"
#include "gq_topk.hpp"

namespace gq {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;

// 16 bytes per lane from global memory into LDS at lds + 16 * lane, past the registers.  The compiler does not wait for them: the
// loop below does (vmcnt), in front of the barrier that hands the stage over.
__device__ __forceinline__ void load_to_lds(rsrc_t rsrc, uint32_t voff, uint32_t soff, uint8_t* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, voff, soff, 0, 0);
}

__device__ __forceinline__ rsrc_t buffer_of(const void* base, int64_t bytes) {
  const uint32_t n = bytes < 0 ? 0u : bytes > 0xffffffffll ? 0xffffffffu : static_cast<uint32_t>(bytes);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(n), 0x00027000);
}

// the bytes of a chunk of 16 at k that lie below K
__device__ __forceinline__ int4_t mask_chunk(int4_t v, int left) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = left - 4 * i;
    v[i] = b >= 4 ? v[i] : b <= 0 ? 0 : v[i] & ((1 << (8 * b)) - 1);
  }
  return v;
}

// eight neighbouring results of row r: bias, residual, one rounding; vec: rows of y and residual start at 16 bytes
template <int OUT, int MODEL>
__device__ __forceinline__ void store_run(const Fp8Args& p, int64_t r, int n, int N, bool vec, float (&o)[8]) {
  const int64_t at = r * N + n;
  const int count = N - n < 8 ? N - n : 8;
#pragma unroll
  for (int v = 0; v < 8; ++v) {
    if (v < count) {
      if (p.bias) o[v] += Elem<MODEL>::load(p.bias, n + v);
      if (p.residual) o[v] += Elem<MODEL>::load(p.residual, at + v);
    }
  }
  if (vec) {
    if constexpr (OUT == MODEL_F32) {
      float4_t* q = reinterpret_cast<float4_t*>(static_cast<float*>(p.y) + at);
      q[0] = float4_t{o[0], o[1], o[2], o[3]};
      q[1] = float4_t{o[4], o[5], o[6], o[7]};
    } else {
      uint32_t u[4];
#pragma unroll
      for (int v = 0; v < 4; ++v)
        u[v] = OUT == MODEL_BF16 ? f2bf(o[2 * v]) | static_cast<uint32_t>(f2bf(o[2 * v + 1])) << 16
                                 : f2h(o[2 * v]) | static_cast<uint32_t>(f2h(o[2 * v + 1])) << 16;
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + at) = uint4{u[0], u[1], u[2], u[3]};
    }
  } else {
#pragma unroll
    for (int v = 0; v < 8; ++v)
      if (v < count) Elem<OUT>::store(p.y, at + v, o[v]);
  }
}

}  // namespace

// WN x WM waves, each TN x TM results of 16 x 16: a tile of BN = 16 WN TN rows of W by BM = 16 WM TM rows of x.
template <int WN, int WM, int TN, int TM, int OUT, int MODEL>
__global__ __launch_bounds__(64 * WN * WM, 2) void fp8_tile_kernel(Fp8Args p, int n_tiles, int m_tiles) {
  constexpr int kWaves = WN * WM, BN = 16 * WN * TN, BM = 16 * WM * TM, kStage = (BN + BM) * 128;
  constexpr int kLoads = (BN + BM) / 8 / kWaves;  // of 1 KiB, eight rows, a wave and stage
  static_assert((BN + BM) / 8 % kWaves == 0 && BN / 8 % kWaves == 0, "whole loads");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = static_cast<int>(p.K), N = static_cast<int>(p.N);
  const int groups = (K + kFp8Block - 1) / kFp8Block, n_blocks = (N + kFp8Block - 1) / kFp8Block;

  // Workgroups go to the eight dies in turn; each die takes a run of tiles, x tiles fastest, so that what runs on it at a time
  // shares rows of W and of x in its L2.
  const int tiles = n_tiles * m_tiles, per = (tiles + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || id >= tiles) return;
  const int nt = id / m_tiles, mt = id - nt * m_tiles, n0 = nt * BN;
  int e = 0, r0 = mt * BM, r_end = static_cast<int>(p.rows);
  if (p.indptr != nullptr) {
    // tiles of segment e are numbered from indptr[e] / BM + e on: no two segments share a number, and some numbers have no tile
    int before = 0;
    for (int i0 = 0; i0 < p.experts; i0 += 64) {
      const int i = i0 + lane;
      before += __popcll(__ballot(i < p.experts && p.indptr[i < p.experts ? i : 0] / BM + i <= mt));
    }
    e = before > 0 ? before - 1 : 0;
    const int begin = p.indptr[e], end = p.indptr[e + 1];
    r0 = begin + (mt - (begin / BM + e)) * BM;
    r_end = end < r_end ? end : r_end;
    e = __builtin_amdgcn_readfirstlane(e);
    r0 = __builtin_amdgcn_readfirstlane(r0);
    r_end = __builtin_amdgcn_readfirstlane(r_end);
  }
  if (r0 >= r_end || r0 < 0) return;

  const uint8_t* w0 = p.w + (static_cast<int64_t>(e) * N + n0) * p.w_pitch;
  const int k16 = (K + 15) & ~15;
  // (every address below lies inside its matrix: rows past the end are read from the last one)
  const rsrc_t w_rsrc = buffer_of(w0, static_cast<int64_t>(N - n0 - 1) * p.w_pitch + k16);
  const bool gather = p.x_row_index != nullptr;
  const uint8_t* x0 = p.x + (gather ? 0 : static_cast<int64_t>(r0) * p.x_pitch);
  const rsrc_t x_rsrc = buffer_of(x0, (p.x_rows - 1 - (gather ? 0 : r0)) * p.x_pitch + k16);
  auto source = [&](int r) {  // row of x behind row r of the result, within x
    int j = r < r_end ? r : r_end - 1;
    if (gather) j = p.x_row_index[j];
    return j < 0 ? 0 : j < p.x_rows ? j : static_cast<int>(p.x_rows) - 1;
  };

  // A row of a stage is 128 bytes, its chunk c of 16 at place c ^ (row & 7), and a lane loads the chunk that belongs at its
  // place.  An operand is chunks q and q + 4 of a row, q = lane / 16 (the order of K is free as long as both operands share it):
  // so the 16 lanes that LDS serves in a cycle, half of them of one quarter of the wave and half of the next, meet 16 places in
  // 16 different groups of banks.  With chunks 2 q and 2 q + 1 every read took two turns.
  const uint32_t w_pitch = static_cast<uint32_t>(p.w_pitch), x_pitch = static_cast<uint32_t>(p.x_pitch);
  uint32_t voff[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = (i * kWaves + wave) * 8 + (lane >> 3), chunk = (lane & 7) ^ (lane >> 3);
    if (i < BN / 8 / kWaves) voff[i] = static_cast<uint32_t>(n0 + row < N ? row : N - 1 - n0) * w_pitch + chunk * 16;
    else voff[i] = static_cast<uint32_t>(source(r0 + row - BN) - (gather ? 0 : r0)) * x_pitch + chunk * 16;
    asm volatile("" : "+v"(voff[i]));  // (kept as it is, not computed again at every load)
  }
  uint8_t* const lds0 = smem + wave * 1024;
  // Loads [from, to) of block g into its stage; past the last block, that one's again (nobody reads them).  A chunk past the row's
  // end is read from its start, and masked where it is used.  No branches: the loop below is to stay one run of instructions.
  const int last = groups - 1, my_chunk = ((lane & 7) ^ (lane >> 3)) * 16;
  auto issue = [&](int g, int from, int to) {
    uint8_t* const at = lds0 + (g & 1) * kStage;
    const int k = (g < last ? g : last) * 128;
    const int shift = k + my_chunk < k16 ? k : -my_chunk;
#pragma unroll
    for (int i = from; i < to; ++i)
      load_to_lds(i < BN / 8 / kWaves ? w_rsrc : x_rsrc, voff[i] + shift, 0, at + i * kWaves * 1024);
  };

  const int wn = (wave % WN) * 16 * TN, wm = (wave / WN) * 16 * TM, frow = lane & 15, fquad = lane >> 4;
  uint32_t xrow[TM];
#pragma unroll
  for (int j = 0; j < TM; ++j) xrow[j] = source(r0 + wm + 16 * j + frow);
  // a wave's rows of W lie in one block, or (64 rows and fewer) in part of one: tiles start at multiples of their size
  static_assert(16 * TN <= kFp8Block && kFp8Block % (16 * TN) == 0, "one block of W a wave");
  typedef const __attribute__((address_space(4))) float* scalar_floats;  // read through the scalar cache
  const int wb = (n0 + wn) / kFp8Block < n_blocks ? (n0 + wn) / kFp8Block : n_blocks - 1;
  const scalar_floats ws = (scalar_floats)(p.ws + (static_cast<int64_t>(e) * n_blocks + wb) * groups);

  float4_t acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = float4_t{};

  // Scales are two blocks ahead, and asked for in front of a stage's loads: the wait for a load takes all before it as well.
  float sx_next[TM], sw_next = 0.f;
  auto scales = [&](int g) {
    g = g < last ? g : last;
#pragma unroll
    for (int j = 0; j < TM; ++j) sx_next[j] = (p.xs + g * p.x_rows)[xrow[j]];
    sw_next = ws[g];
  };
  auto frag = [&](int g, int row, auto tail) {
    const uint8_t* base = smem + (g & 1) * kStage + row * 128;
    int4_t a = *reinterpret_cast<const int4_t*>(base + ((fquad ^ (row & 7)) << 4));
    int4_t b = *reinterpret_cast<const int4_t*>(base + (((fquad + 4) ^ (row & 7)) << 4));
    if constexpr (decltype(tail)::value) {
      a = mask_chunk(a, K - g * 128 - fquad * 16);
      b = mask_chunk(b, K - g * 128 - fquad * 16 - 64);
    }
    return int8_vt{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  };
  float4_t part[TM];                      // a row of results of one block, unscaled
  float sc[TM], sc_old[TM], sc_next[TM];  // scales of this block, the one before and the one behind it
  int8_vt fx[TM], fw[2];
  // Waits for stage g and hands it over: every wave has read the stage before it, which may take the loads of block g + 1.
  auto hand_over = [&](int g) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      sc_next[j] = sw_next * sx_next[j];
      asm volatile("" : "+v"(sc_next[j]));  // here, not behind the loads below
    }
    scales(g + 1);
  };
  // One block.  The multiply-adds of a result run beside the matrix instructions of the row of results behind it, and the last
  // row's beside the next block's first; the next stage is handed over in front of the last row, so that its first operands
  // arrive while that row is computed.
  // The next block's loads go out kBurst at a time, the first behind the hand-over and the others in front of the rows: all at
  // once they fill the queue to the vector cache (16 cycles a load), and every wave waits there in front of its matrix instructions.
  constexpr int kBurst = 2;
  static_assert((TN - 1) * kBurst >= kLoads - kBurst, "every load has a row");
  auto step = [&](int g, auto tail, auto next_tail, auto has_next) {
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      if (i + 1 < TN) {
        fw[(i + 1) & 1] = frag(g, wn + 16 * (i + 1) + frow, tail);
      } else if (decltype(has_next)::value) {
        hand_over(g + 1);
        fw[0] = frag(g + 1, wn + frow, next_tail);
        issue(g + 2, 0, kBurst < kLoads ? kBurst : kLoads);
      }
      if (decltype(has_next)::value && i + 1 < TN && (i + 1) * kBurst < kLoads)
        issue(g + 1, (i + 1) * kBurst, (i + 2) * kBurst < kLoads ? (i + 2) * kBurst : kLoads);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const float s = i == 0 ? sc_old[j] : sc[j];
        float4_t& to = acc[i == 0 ? TN - 1 : i - 1][j];
#pragma unroll
        for (int v = 0; v < 4; ++v) to[v] = __builtin_fmaf(part[j][v], s, to[v]);
        asm volatile("" : "+v"(to));  // here, not behind the last row with all partial results kept
        part[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[i & 1], fx[j], float4_t{}, 0, 0, 0, 0, 0, 0);
        if (i + 1 == TN && decltype(has_next)::value) fx[j] = frag(g + 1, BN + wm + 16 * j + frow, next_tail);
      }
      __builtin_amdgcn_sched_barrier(0);  // rows in this order: operands of all rows at once would not fit the registers
    }
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      sc_old[j] = sc[j];
      sc[j] = sc_next[j];
    }
  };
  static_assert(TN % 2 == 0, "the first row of a block uses fw[0]");
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  scales(0);
  issue(0, 0, kLoads);
  hand_over(0);
  issue(1, 0, kBurst < kLoads ? kBurst : kLoads);
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    part[j] = float4_t{};
    sc_old[j] = 0.f;
    sc[j] = sc_next[j];
  }
  auto first = [&](auto tail) {
    fw[0] = frag(0, wn + frow, tail);
#pragma unroll
    for (int j = 0; j < TM; ++j) fx[j] = frag(0, BN + wm + 16 * j + frow, tail);
  };
  // the last block is masked, whether K ends inside it or not: one form of it, once a tile
  if (last == 0) first(yes);
  else first(no);
  for (int g = 0; g < last - 1; ++g) step(g, no, no, yes);
  if (last > 0) step(last - 1, no, yes, yes);
  step(last, yes, no, no);
#pragma unroll
  for (int j = 0; j < TM; ++j)
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[TN - 1][j][v] = __builtin_fmaf(part[j][v], sc_old[j], acc[TN - 1][j][v]);

  // The results change hands through LDS, 16 rows of x at a time and each wave in a part of its own, so that a row's
  // columns go out as runs of 16 bytes per lane; float32 until bias and residual are in.
  constexpr int kCols = 16 * TN, kRow = kCols + 4, kLanes = kCols / 8, kRows = 64 / kLanes < 16 ? 64 / kLanes : 16;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads that nobody reads may still land in the stages
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(smem) + wave * 16 * kRow;
  const bool vec = N % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.residual)) & 15u) == 0;
#pragma unroll
  for (int j = 0; j < TM; ++j) {
#pragma unroll
    for (int i = 0; i < TN; ++i) *reinterpret_cast<float4_t*>(mine + frow * kRow + 16 * i + 4 * fquad) = acc[i][j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < 16 / kRows; ++t) {
      const int row = t * kRows + lane / kLanes, col = (lane % kLanes) * 8;
      const int64_t r = r0 + wm + 16 * j + row;
      const int n = n0 + wn + col;
      if (row < 16 && r < r_end && n < N) {
        const float4_t a = *reinterpret_cast<const float4_t*>(mine + row * kRow + col), b = *reinterpret_cast<const float4_t*>(mine + row * kRow + col + 4);
        float o[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        store_run<OUT, MODEL>(p, r, n, N, vec, o);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

template <int WN, int WM, int TN, int TM>
static hipError_t launch_tile(const Fp8Args& a, hipStream_t s) {
  constexpr int BN = 16 * WN * TN, BM = 16 * WM * TM;
  constexpr size_t stages = size_t(2) * (BN + BM) * 128, results = size_t(WN * WM) * 16 * (16 * TN + 4) * 4;
  constexpr size_t lds = stages > results ? stages : results;
  const int64_t m_tiles = a.indptr ? a.rows / BM + a.experts : (a.rows + BM - 1) / BM, n_tiles = (a.N + BN - 1) / BN;
  const unsigned grid = static_cast<unsigned>((n_tiles * m_tiles + 7) / 8 * 8);
  note_kernel("fp8_tile %dx%d", BN, BM);
  auto go = [&](auto out, auto model) {
    auto* kern = fp8_tile_kernel<WN, WM, TN, TM, decltype(out)::value, decltype(model)::value>;
    if (lds > 65536) {
      const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern));
      if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kern, dim3(grid), dim3(64 * WN * WM), lds, s, a, static_cast<int>(n_tiles), static_cast<int>(m_tiles));
    return hipGetLastError();
  };
  auto by_model = [&](auto out) {
    if (a.model_dtype == MODEL_F32) return go(out, std::integral_constant<int, MODEL_F32>{});
    if (a.model_dtype == MODEL_BF16) return go(out, std::integral_constant<int, MODEL_BF16>{});
    return go(out, std::integral_constant<int, MODEL_F16>{});
  };
  if (a.out_dtype == MODEL_F32) return by_model(std::integral_constant<int, MODEL_F32>{});
  if (a.out_dtype == MODEL_BF16) return by_model(std::integral_constant<int, MODEL_BF16>{});
  return by_model(std::integral_constant<int, MODEL_F16>{});
}

hipError_t launch_fp8_tile(const Fp8Args& a, hipStream_t s) {
  return launch_tile<2, 4, 8, 4>(a, s);
}

}  // namespace gq
