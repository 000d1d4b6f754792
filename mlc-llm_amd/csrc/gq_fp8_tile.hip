// e4m3 block-scaled matrix product on the 8-bit matrix instruction (v_mfma_f32_16x16x128_f8f6f4), dense or by expert segments.
//
//   y[r, n] = sum over blocks g of 128 of  xs[g, r] ws[n / 128, g] sum_{k in g} xq[r, k] wq[n, k]
//
// W is the instruction's A operand and x its B operand, so a lane of a 16 x 16 result holds one row r of x and four rows n of
// W: both scales of a block are one number per lane, and a block's sum joins the float32 accumulator with four multiply-adds
// beside its one matrix instruction (32 cycles, the multiply-adds another 16 of the vector unit).
// What the instruction sums itself is one block of 128: of eight neighbouring products it drops what lies more than 13 bits below
// the largest, and adds such sums in float32 (seen with single products over all positions and sizes).  That is a choice for speed: the error of
// a whole result is 1.5e-5 of its norm for normal operands, 2.7e-5 and 7.7e-5 where x's channels are spread by exp(0.7 N) and exp(2 N), 1.4e-3 to
// 2.3e-3 of the results' deviation at most, where float32 sums are 1e-7 off and a rounding to float16 2.1e-4.  Blocks join in float32.
//
// Measured, and what bounds it: 8192 x 8192 x 8192 485 to 505 us = 2.2 PFLOP/s, 2048 x 28672 x 4096 264 to 277 us in all (two launches).  The
// matrix pipe is busy 53 % of the cycles at 2.0 GHz; without its loads the large tile takes 419 us, without barriers as well 419, and without
// the reads of x from LDS 395, and an operand of W asked for two rows ahead in place of one changes nothing: multiply-adds (4 to a matrix
// instruction, 40 % of the vector unit), LDS and the caches share issue slots and power with the matrix pipe.  Matrix and vector cycles add up to
// 85 to 105 % of all, as if the two hardly ran at once; why is not found.
// 256 x 256 x 128 is a stage of 64 KiB for 8 waves; they read 192 KiB of operands from LDS for it.
//
// Precise products sum in float32 throughout: the operands are widened to bfloat16 (which holds them exactly) on their way from
// LDS, four instructions of 16 x 16 x 32 to a block, at half the rate.  So do products that are rounded to e4m3 again.
#include "gq_fp8_common.hpp"

namespace gq {

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;

// 16 bytes per lane from global memory into LDS at lds + 16 * lane, past the registers.  The compiler does not wait for them: the
// loop below does (vmcnt), in front of the barrier that hands the stage over.
__device__ __forceinline__ void load_to_lds(rsrc_t rsrc, uint32_t off, uint8_t* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, off, 0, 0, 0);
}

__device__ __forceinline__ rsrc_t buffer_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes), 0x00027000);
}
// bytes that a tile may reach: rows are below 2^24 bytes, so that a tile's 256 end below what is left of 2^32 at any block of K
__device__ __forceinline__ uint32_t reach(int64_t bytes) { return bytes > 0xffffffffll ? 0xffffffffu : static_cast<uint32_t>(bytes); }

// the bytes of a chunk of 16 at k that lie below K
__device__ __forceinline__ int4_t mask_chunk(int4_t v, int left) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = left - 4 * i;
    v[i] = b >= 4 ? v[i] : b <= 0 ? 0 : v[i] & ((1 << (8 * b)) - 1);
  }
  return v;
}

}  // namespace

// WN x WM waves, each TN x TM results of 16 x 16: a tile of BN = 16 WN TN rows of W by BM = 16 WM TM rows of x.
// SILU: half of a wave's rows of W are gate rows and half the up rows that belong to them.
// WS stages of W in LDS: three, so that W is two blocks ahead; or two, one block ahead, in the forms of 64 rows, two or three workgroups of which
// run on a unit then (expert layer of 509 tokens, 128 experts: 175 -> 163 us).
template <int WN, int WM, int TN, int TM, int WS, bool PRECISE, bool SILU>
__global__ __launch_bounds__(64 * WN * WM, WS == 2 ? 4 : 2) void fp8_tile_kernel(Fp8Args p, int n_first, int n_tiles, int m_tiles, int per_split) {
  constexpr int kWaves = WN * WM, BN = 16 * WN * TN, BM = 16 * WM * TM;
  constexpr int kWLoads = BN / 8 / kWaves, kXLoads = (BM / 8 + kWaves - 1) / kWaves;  // of 1 KiB, eight rows, a wave and block of K
  constexpr int P = SILU ? 2 : 1, kPart = 16 * TN / P;  // parts of a wave's rows of W
  constexpr int kWStage = BN * 128, kXStage = kXLoads * kWaves * 1024;  // WS stages of W and two of x in LDS
  static_assert(BN / 8 % kWaves == 0, "whole loads");
  static_assert(TN % 2 == 0, "the first row of a block uses fw[0]");
  static_assert(kPart <= kFp8Block && kFp8Block % kPart == 0, "a part lies in one block of W");
  static_assert(!SILU || BN == 2 * kFp8Block, "a tile holds one group of the activation");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = static_cast<int>(p.K), N = static_cast<int>(p.N), half = N / P;
  const int groups = (K + kFp8Block - 1) / kFp8Block, n_blocks = (N + kFp8Block - 1) / kFp8Block;

  // Workgroups go to the eight dies in turn; each die takes a run of tiles, x tiles fastest, so that what runs on it at a time
  // shares rows of W and of x in its L2.
  const int tiles = n_tiles * m_tiles, per = (tiles + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || id >= tiles) return;
  const int nt = id / m_tiles, mt = id - nt * m_tiles, n0 = n_first + nt * (BN / P);
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
  // this workgroup's blocks of K
  const int first = blockIdx.y * per_split, last = (first + per_split < groups ? first + per_split : groups) - 1;

  const uint8_t* w0 = p.w + (static_cast<int64_t>(e) * N + n0) * p.w_pitch;
  const int k16 = (K + 15) & ~15;
  // Rows past the end are read from the last one.  A block's loads see the matrix from that block on, and nothing past its end: the last
  // row's bytes past K are zeros, another row's are what lies there, and the last block is masked where it is used.
  const uint32_t w_bytes = reach(static_cast<int64_t>(N - n0 - 1) * p.w_pitch + k16);
  const bool gather = p.x_row_index != nullptr;
  const uint8_t* x0 = p.x + (gather ? 0 : static_cast<int64_t>(r0) * p.x_pitch);
  const uint32_t x_bytes = reach((p.x_rows - 1 - (gather ? 0 : r0)) * p.x_pitch + k16);
  auto source = [&](int r) {  // row of x behind row r of the result, within x
    int j = r < r_end ? r : r_end - 1;
    if (gather) j = p.x_row_index[j];
    return j < 0 ? 0 : j < p.x_rows ? j : static_cast<int>(p.x_rows) - 1;
  };
  auto w_row = [&](int row) {  // row of W, from n0, behind row `row` of the tile
    const int part = row % (16 * TN) / kPart, n = row / (16 * TN) * kPart + row % kPart;
    return (n0 + n < half ? n : half - 1 - n0) + part * half;
  };

  // A row of a stage is 128 bytes, its chunk c of 16 at place c ^ (row & 7), and a lane loads the chunk that belongs at its
  // place.  An operand is chunks q and q + 4 of a row, q = lane / 16 (the order of K is free as long as both operands share it):
  // so the 16 lanes that LDS serves in a cycle, half of them of one quarter of the wave and half of the next, meet 16 places in
  // 16 different groups of banks.  With chunks 2 q and 2 q + 1 every read took two turns.
  const uint32_t w_pitch = static_cast<uint32_t>(p.w_pitch), x_pitch = static_cast<uint32_t>(p.x_pitch);
  uint32_t w_off[kWLoads], x_off[kXLoads];
  const int my_chunk = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
  for (int i = 0; i < kWLoads; ++i) {
    w_off[i] = static_cast<uint32_t>(w_row((i * kWaves + wave) * 8 + (lane >> 3))) * w_pitch + my_chunk;
    asm volatile("" : "+v"(w_off[i]));  // (kept as it is, not computed again at every load)
  }
#pragma unroll
  for (int i = 0; i < kXLoads; ++i) {
    x_off[i] = static_cast<uint32_t>(source(r0 + (i * kWaves + wave) * 8 + (lane >> 3)) - (gather ? 0 : r0)) * x_pitch + my_chunk;
    asm volatile("" : "+v"(x_off[i]));
  }
  // Loads [from, to) of block g; past the last block, that one's again (nobody reads them).  No branches: the loop below is to
  // stay one run of instructions, and the vector unit's, which has a multiply-add to issue beside the matrix instructions nine times in ten,
  // has none for addresses.
  auto issue_w = [&](int g, int slot, int from, int to) {
    const uint32_t k = (g < last ? g : last) * 128u;
    const rsrc_t rsrc = buffer_of(w0 + k, w_bytes - k);
#pragma unroll
    for (int i = from; i < to; ++i) load_to_lds(rsrc, w_off[i], smem + slot + (i * kWaves + wave) * 1024);
  };
  auto issue_x = [&](int g, int from, int to) {
    const uint32_t k = (g < last ? g : last) * 128u;
    const rsrc_t rsrc = buffer_of(x0 + k, x_bytes - k);
#pragma unroll
    for (int i = from; i < to; ++i) load_to_lds(rsrc, x_off[i], smem + WS * kWStage + (g & 1) * kXStage + (i * kWaves + wave) * 1024);
  };

  const int wn = (wave % WN) * 16 * TN, wm = (wave / WN) * 16 * TM, frow = lane & 15, fquad = lane >> 4;
  const float* const xs0 = p.xs + (gather ? 0 : r0);
  uint32_t xs_off[TM];  // (rows by an index: x ends below 4 GiB)
#pragma unroll
  for (int j = 0; j < TM; ++j) xs_off[j] = static_cast<uint32_t>(source(r0 + wm + 16 * j + frow) - (gather ? 0 : r0)) * 4u;
  const float* ws[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int b = (n0 + (wave % WN) * kPart + i * half) / kFp8Block;
    ws[i] = p.ws + (static_cast<int64_t>(e) * n_blocks + (b < n_blocks ? b : n_blocks - 1)) * groups;
  }

  float4_t acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = float4_t{};

  // Scales are a block ahead.  Vector loads, also for W's: a scalar load counts with the reads of LDS and comes back in any order, so
  // that a wait for one is a wait for all.
  float sx_next[TM], sw_next[P];
  auto scales = [&](int g) {
    g = g < last ? g : last;
    const rsrc_t xs_rsrc = buffer_of(xs0 + g * p.x_rows, 0xffffffffu);
#pragma unroll
    for (int j = 0; j < TM; ++j) sx_next[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(xs_rsrc, xs_off[j], 0, 0));
#pragma unroll
    for (int i = 0; i < P; ++i) sw_next[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buffer_of(ws[i] + g, 4), 0, 0, 0));
  };
  struct Operand {
    int4_t a, b;  // chunks q and q + 4 of a row
  };
  auto frag = [&](const uint8_t* stage, int g, int row, auto tail) {
    const uint8_t* base = stage + row * 128;
    Operand o;
    o.a = *reinterpret_cast<const int4_t*>(base + ((fquad ^ (row & 7)) << 4));
    o.b = *reinterpret_cast<const int4_t*>(base + (((fquad + 4) ^ (row & 7)) << 4));
    if constexpr (decltype(tail)::value) {
      o.a = mask_chunk(o.a, K - g * 128 - fquad * 16);
      o.b = mask_chunk(o.b, K - g * 128 - fquad * 16 - 64);
    }
    return o;
  };
  struct Wide {
    bf16x8_t v[4];
  };
  auto wide = [](const Operand& o) {
    return Wide{{fp8_widen(o.a[0], o.a[1]), fp8_widen(o.a[2], o.a[3]), fp8_widen(o.b[0], o.b[1]), fp8_widen(o.b[2], o.b[3])}};
  };
  float4_t part[TM];                                   // a row of results of one block, unscaled
  float sc[P][TM];                                     // scales of its block
  Operand fx[TM], fw[2];
  Wide wx[PRECISE ? TM : 1];
  int w_now = 0, w_then = kWStage, w_last = 2 * kWStage;  // stages of W of this block, the next and the one behind it
  auto frag_w = [&](int g, int slot, int i, auto tail) { return frag(smem + slot, g, wn + 16 * i + frow, tail); };
  auto frag_x = [&](int g, int j, auto tail) { return frag(smem + WS * kWStage + (g & 1) * kXStage, g, wm + 16 * j + frow, tail); };
  // Waits for block g's stages and hands them over.  Loads come back in order, and the last ones asked for are the scales of block g
  // and (WS 3) W of block g + 1, which may still be on their way: W comes from memory and is two blocks ahead, x from the L2 and one.  Every
  // wave has read block g - 1 by then, whose stages take x of block g + 1 and W of block g + WS - 1.  The count takes every scale for a
  // load of its own, and in the order of this text.
  auto hand_over = [&](auto scale_loads) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(WS == 2 ? 0 : kWLoads + decltype(scale_loads)::value) : "memory");
    __builtin_amdgcn_s_barrier();
  };
  // One block.  The multiply-adds of a result run beside the matrix instructions of the row of results behind it, and the last
  // row's beside the next block's first; the next stage is handed over in front of the last row, so that its first operands
  // arrive while that row is computed.
  // The next block's loads go out kBurst at a time, the first behind the hand-over and the others in front of the rows: all at
  // once they fill the queue to the vector cache (16 cycles a load), and every wave waits there in front of its matrix instructions.
  constexpr int kBurst = 2, kXBursts = (kXLoads + kBurst - 1) / kBurst, kBursts = kXBursts + kWLoads / kBurst;
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
        hand_over(std::integral_constant<int, TM + P>{});
        fw[0] = frag_w(g + 1, w_then, 0, next_tail);
        burst(0, g + 2, w_now);
      }
      if (decltype(has_next)::value && i + 1 < TN) burst(i + 1, g + 1, WS == 2 ? w_then : w_last);
      __builtin_amdgcn_sched_barrier(0);  // (loads first: they have the row's time)
      Wide ww;
      if constexpr (PRECISE) ww = wide(fw[i & 1]);
      __builtin_amdgcn_s_setprio(1);  // (a wave with its operands goes before one that asks for them)
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int prev = i == 0 ? TN - 1 : i - 1;
        const float s = sc[prev * P / TN][j];  // (the block before's while i is 0)
        float4_t& to = acc[prev][j];
#pragma unroll
        for (int v = 0; v < 4; ++v) to[v] = __builtin_fmaf(part[j][v], s, to[v]);
        asm volatile("" : "+v"(to));  // here, not behind the last row with all partial results kept
        if constexpr (PRECISE) {
          if (i == 0) wx[j] = wide(fx[j]);
          part[j] = float4_t{};
#pragma unroll
          for (int h = 0; h < 4; ++h) part[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww.v[h], wx[j].v[h], part[j], 0, 0, 0);
        } else {
          auto both = [](const Operand& o) { return int8_vt{o.a[0], o.a[1], o.a[2], o.a[3], o.b[0], o.b[1], o.b[2], o.b[3]}; };
          part[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(both(fw[i & 1]), both(fx[j]), float4_t{}, 0, 0, 0, 0, 0, 0);
        }
        if (i + 1 == TN && decltype(has_next)::value) {
          fx[j] = frag_x(g + 1, j, next_tail);
          __builtin_amdgcn_sched_barrier(0);  // (at once, not behind the row's other instructions)
        }
      }
      if (i == 0) {  // nobody needs the scales of the block before any more
#pragma unroll
        for (int t = 0; t < P; ++t)
#pragma unroll
          for (int j = 0; j < TM; ++j) {
            sc[t][j] = sw_next[t] * sx_next[j];
            asm volatile("" : "+v"(sc[t][j]));  // here, in front of the loads
          }
        if (decltype(has_next)::value) scales(g + 1);
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
  scales(first);
  asm volatile("" ::: "memory");
  if (WS == 3) issue_w(first + 1, w_then, 0, kWLoads);
  hand_over(std::integral_constant<int, TM + P>{});
  burst(0, first + 1, w_last);
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    part[j] = float4_t{};
#pragma unroll
    for (int i = 0; i < P; ++i) sc[i][j] = 0.f;
  }
  if (r0 + wm < r_end) {
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
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[TN - 1][j][v] = __builtin_fmaf(part[j][v], sc[P - 1][j], acc[TN - 1][j][v]);
  } else {
    // none of this wave's rows of x exist: it only brings its part of the stages
    for (int g = first; g < last; ++g) {
#pragma unroll
      for (int i = 1; i < kBursts; ++i) burst(i, g + 1, WS == 2 ? w_then : w_last);
      hand_over(std::integral_constant<int, 0>{});
      burst(0, g + 2, w_now);
      next_stage();
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads that nobody reads may still land in the stages
  __syncthreads();  // (and the last stage has been read)

  if constexpr (SILU) {
    // silu(gate) * up in place of the gates; a group is the tile's 128 columns, of which this wave has kPart
    float* const tops = reinterpret_cast<float*>(smem);  // [WN][BM]
    uint8_t* const bytes = smem + WN * BM * 4;           // [BM][kBytes]
    constexpr int kBytes = kFp8Block + 16;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < TN / 2; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          acc[i][j][v] = silu_mul_f32(acc[i][j][v], acc[i + TN / 2][j][v]);
          top = fmaxf(top, fp8_magnitude(acc[i][j][v]));
        }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      if (fquad == 0) tops[(wave % WN) * BM + wm + 16 * j + frow] = top;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int row = wm + 16 * j + frow;
      float top = tops[row];
#pragma unroll
      for (int w = 1; w < WN; ++w) top = fmaxf(top, tops[w * BM + row]);
      const uint32_t bits = fp8_scale_bits(top);
      const float inv = fp8_inverse(bits);
#pragma unroll
      for (int i = 0; i < TN / 2; ++i)
        *reinterpret_cast<uint32_t*>(bytes + row * kBytes + (wave % WN) * kPart + 16 * i + 4 * fquad) =
            fp8_quad(acc[i][j][0] * inv, acc[i][j][1] * inv, acc[i][j][2] * inv, acc[i][j][3] * inv);
      if (wave % WN == 0 && fquad == 0 && r0 + row < r_end)
        p.scale_out[static_cast<int64_t>(n0 / kFp8Block) * p.rows + r0 + row] = __builtin_bit_cast(float, bits);
    }
    __syncthreads();
    for (int c = tid; c < BM * 8; c += 64 * kWaves) {
      const int row = c >> 3;
      if (r0 + row < r_end)
        *reinterpret_cast<uint4*>(p.q_out + static_cast<int64_t>(r0 + row) * half + n0 + (c & 7) * 16) =
            *reinterpret_cast<const uint4*>(bytes + row * kBytes + (c & 7) * 16);
    }
  } else {
    // The results change hands through LDS, 16 rows of x at a time and each wave in a part of its own, so that a row's
    // columns go out as runs of 16 bytes per lane; float32 until bias and residual are in.
    constexpr int kCols = 16 * TN, kRow = kCols + 4, kLanes = kCols / 8, kRows = 64 / kLanes < 16 ? 64 / kLanes : 16;
    float* const mine = reinterpret_cast<float*>(smem) + wave * 16 * kRow;
    Fp8Args to = p;
    if (gridDim.y > 1) {  // a share of K: its sums go to the scratch as they are
      to.y = static_cast<float*>(p.workspace) + blockIdx.y * p.rows * N;
      to.out_dtype = MODEL_F32;
      to.bias = to.residual = nullptr;
    }
    const bool vec = N % 8 == 0 && (reinterpret_cast<uintptr_t>(to.y) & 15u) == 0;
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
          fp8_store<8>(to, r, n, N, vec, o);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// the sums of the shares of K, in their order; bias, residual and the one rounding.  Four columns a thread, so that a wave's read of a
// share is 1 KiB in one piece.
__global__ __launch_bounds__(256) void fp8_join_kernel(Fp8Args p, int splits) {
  const int N = static_cast<int>(p.N), runs = (N + 3) / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.rows * runs) return;
  const int64_t r = i / runs;
  const int n = static_cast<int>(i - r * runs) * 4;
  const float* from = static_cast<const float*>(p.workspace) + r * N + n;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  const bool vec = N % 4 == 0;
  for (int s = 0; s < splits; ++s, from += p.rows * N) {
    if (vec) {
      const float4_t a = *reinterpret_cast<const float4_t*>(from);
#pragma unroll
      for (int v = 0; v < 4; ++v) o[v] += a[v];
    } else {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (n + v < N) o[v] += from[v];
    }
  }
  fp8_store<4>(p, r, n, N, vec && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0, o);
}

namespace {

// A tile form and the shares of K of a dense product; from column n_rest on, another form without shares.
struct Plan {
  int form = 0, splits = 1, per_split = 0;
  int64_t n_rest = 0;
  int form_rest = 0;
  float ns = 0.f;
};
// Tiles, workgroups that run at a time, and what a block of K of a round of them takes in ns: alone_ns where few run, full_ns where all
// of them do (L2 and clocks are shared).  Fitted to 5500 timings of 112 shapes, 18 to 2048 rows, all forms, 1 to 12 shares: the choice takes 1.7 %
// longer than the best one on average, 15 % at most.
struct Form {
  int bn, bm, at_a_time;
  float alone_ns, full_ns;
};
constexpr Form kForms[] = {{256, 256, 256, 875.f, 1687.f}, {256, 192, 256, 752.f, 1412.f}, {256, 160, 256, 822.f, 1203.f}, {256, 128, 256, 619.f, 927.f},
                           {128, 128, 512, 436.f, 1046.f}, {128, 64, 768, 358.f, 970.f}};
constexpr float kRoundNs = 1140.f, kJoinNs = 460.f, kShareNs = 1.42e-3f;  // a round's ends, the launch that joins, an element of a share
// float32 sums: widening, and four instructions for one.  Fitted alike (36 shapes: 1.4 % on average).  64 rows of 4096 x 14336 29 us in 16 shares, 119 in one; 300 of 4096 x 4096 29 and 52.
constexpr Form kPreciseForms[] = {{256, 192, 256, 1493.f, 2287.f}, {256, 128, 256, 962.f, 1765.f}, {256, 64, 512, 582.f, 2050.f}};
struct Forms {
  const Form* form;
  int count;
};
Forms forms_of(bool precise) { return precise ? Forms{kPreciseForms, 3} : Forms{kForms, 6}; }
float ns_of(const Form& f, int64_t tiles, int64_t blocks) {
  const int64_t full = tiles / f.at_a_time, rest = tiles - full * f.at_a_time;
  float ns = full * (blocks * f.full_ns + kRoundNs);
  if (rest > 0) ns += blocks * (f.alone_ns + (f.full_ns - f.alone_ns) * rest / f.at_a_time) + kRoundNs;
  return ns;
}
bool may_take(const Forms& forms, int form) {
  return options().gemm_variant < 0 || options().gemm_variant >= forms.count || options().gemm_variant == form;
}
Plan plan_of(const Forms& forms, int64_t rows, int64_t N, int64_t K, bool only_whole = false) {
  const int64_t groups = (K + kFp8Block - 1) / kFp8Block;
  Plan best;
  for (int f = 0; f < forms.count; ++f) {
    if (!may_take(forms, f)) continue;
    const int64_t m_tiles = (rows + forms.form[f].bm - 1) / forms.form[f].bm, n_tiles = (N + forms.form[f].bn - 1) / forms.form[f].bn, tiles = m_tiles * n_tiles;
    for (int64_t want = 1; want <= 16 && want <= (only_whole || groups < 4 ? 1 : groups / 4); ++want) {
      if (options().gemm_split_k > 0 && options().gemm_split_k != want) continue;
      const int64_t per = (groups + want - 1) / want, splits = (groups + per - 1) / per;
      const float ns = ns_of(forms.form[f], tiles * splits, per) + (splits > 1 ? kJoinNs + splits * rows * N * kShareNs : 0.f);
      if (best.per_split == 0 || ns < best.ns) {
        best = Plan{};
        best.form = f;
        best.splits = static_cast<int>(splits);
        best.per_split = static_cast<int>(per);
        best.ns = ns;
      }
    }
    // whole rounds of this form, and what is left of the last in a form that fills a round of its own
    const int64_t whole = tiles / forms.form[f].at_a_time * forms.form[f].at_a_time / m_tiles;
    if (!only_whole && options().gemm_split_k <= 1 && whole > 0 && whole < n_tiles) {
      const Plan rest = plan_of(forms, rows, N - whole * forms.form[f].bn, K, true);
      const float ns = ns_of(forms.form[f], whole * m_tiles, groups) + rest.ns + 2000.f;
      if (ns < best.ns) {
        best = Plan{};
        best.form = f;
        best.per_split = static_cast<int>(groups);
        best.n_rest = whole * forms.form[f].bn;
        best.form_rest = rest.form;
        best.ns = ns;
      }
    }
  }
  return best;
}
// With segments a tile in two, about, of each is short.  No shares of K.
int form_of(const Forms& forms, int64_t rows, int64_t experts, int64_t N, int64_t K) {
  int best = 0;
  float best_ns = 0.f;
  for (int f = 0; f < forms.count; ++f) {
    if (!may_take(forms, f)) continue;
    const int64_t tiles = (rows / forms.form[f].bm + (experts + 1) / 2) * ((N + forms.form[f].bn - 1) / forms.form[f].bn);
    const float ns = ns_of(forms.form[f], tiles, (K + kFp8Block - 1) / kFp8Block);
    if (best_ns == 0.f || ns < best_ns) {
      best_ns = ns;
      best = f;
    }
  }
  return best;
}

template <int WN, int WM, int TN, int TM, int WS, bool PRECISE, bool SILU>
hipError_t launch_tile(const Fp8Args& a, const Plan& plan, int part, hipStream_t s) {
  constexpr int BN = 16 * WN * TN, BM = 16 * WM * TM;
  constexpr size_t stages = size_t(WS * BN) * 128 + 2 * ((BM / 8 + WN * WM - 1) / (WN * WM) * WN * WM * 1024), results = SILU ? size_t(BM) * (4 * WN + kFp8Block + 16) : size_t(WN * WM) * 16 * (16 * TN + 4) * 4;
  constexpr size_t lds = stages > results ? stages : results;
  const int64_t groups = (a.K + kFp8Block - 1) / kFp8Block;
  const int64_t m_tiles = a.indptr ? a.rows / BM + a.experts : (a.rows + BM - 1) / BM;
  const int64_t n_first = part == 0 ? 0 : plan.n_rest, n_end = part == 0 && plan.n_rest > 0 ? plan.n_rest : a.N, n_tiles = (n_end - n_first + BN - 1) / BN;
  int splits = 1, per_split = static_cast<int>(groups);
  const int64_t joined = a.rows * ((a.N + 3) / 4);  // work items of the join; 2^32 or more in a launch would wrap, without an error
  if (plan.splits > 1 && a.workspace != nullptr && a.workspace_bytes >= plan.splits * a.rows * a.N * 4 && joined < 0xffffff00ll) {
    splits = plan.splits;
    per_split = plan.per_split;
  }
  auto* kern = fp8_tile_kernel<WN, WM, TN, TM, WS, PRECISE, SILU>;
  if (lds > 65536) {
    const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern));
    if (e != hipSuccess) return e;
  }
  note_kernel("fp8_tile %dx%d%s, %d shares of K", BN, BM, PRECISE ? " float32 sums" : "", splits);
  const int64_t most = (0xffffffffll / (64 * WN * WM) - 8) / m_tiles;  // columns of tiles a launch, likewise (m_tiles is 65535 at most)
  for (int64_t t0 = 0; t0 < n_tiles; t0 += most) {
    const int64_t here = n_tiles - t0 < most ? n_tiles - t0 : most;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((here * m_tiles + 7) / 8 * 8), splits), dim3(64 * WN * WM), lds, s, a,
                       static_cast<int>(n_first + t0 * (SILU ? BN / 2 : BN)), static_cast<int>(here), static_cast<int>(m_tiles), per_split);
  }
  if (splits > 1) hipLaunchKernelGGL(fp8_join_kernel, dim3(static_cast<unsigned>((joined + 255) / 256)), dim3(256), 0, s, a, splits);
  return hipGetLastError();
}

hipError_t launch_part(const Fp8Args& a, const Plan& plan, int part, hipStream_t s) {
  const int form = part == 0 ? plan.form : plan.form_rest;
  if (a.precise) {
    if (form == 0) return launch_tile<2, 4, 8, 3, 3, true, false>(a, plan, part, s);
    if (form == 1) return launch_tile<4, 2, 4, 4, 3, true, false>(a, plan, part, s);
    return launch_tile<4, 2, 4, 2, 2, true, false>(a, plan, part, s);
  }
  switch (form) {
    case 0: return launch_tile<2, 4, 8, 4, 3, false, false>(a, plan, part, s);
    case 1: return launch_tile<4, 2, 4, 6, 3, false, false>(a, plan, part, s);
    case 2: return launch_tile<4, 2, 4, 5, 3, false, false>(a, plan, part, s);
    case 3: return launch_tile<4, 2, 4, 4, 3, false, false>(a, plan, part, s);
    case 4: return launch_tile<2, 2, 4, 4, 3, false, false>(a, plan, part, s);
    default: return launch_tile<2, 2, 4, 2, 2, false, false>(a, plan, part, s);
  }
}

}  // namespace

int64_t fp8_tile_workspace_bytes(int64_t rows, int64_t N, int64_t K) {
  int64_t bytes = 0;
  for (const bool precise : {false, true}) {
    const Plan p = plan_of(forms_of(precise), rows, N, K);
    if (p.splits > 1 && p.splits * rows * N * 4 > bytes) bytes = p.splits * rows * N * 4;
  }
  return bytes;
}

hipError_t launch_fp8_tile(const Fp8Args& a, hipStream_t s) {
  if (a.q_out != nullptr) {
    if (!fp8_silu_takes(a.N, a.w_pitch)) return hipErrorNotSupported;
    // 64 rows in two workgroups a unit, or 192 in one: expert layers of 128 x 2048 x 768 at 64 rows an expert 227 / 246 us, at 128 312 / 327, at
    // 256 499 / 517; of 8 x 4096 x 14336 at 64 rows 387 / 396, at 192 689 / 727, at 256 852 / 822, at 384 1177 / 1125.  (A form of 128 rows,
    // whose waves widen a third more operands than 192's for a result, was behind one of them at all of these.)
    if (a.rows < 256 * a.experts) return launch_tile<4, 2, 4, 2, 2, true, true>(a, Plan{}, 0, s);
    return launch_tile<2, 4, 8, 3, 3, true, true>(a, Plan{}, 0, s);
  }
  Plan plan;
  if (!a.indptr) plan = plan_of(forms_of(a.precise), a.rows, a.N, a.K);
  else plan.form = form_of(forms_of(a.precise), a.rows, a.experts, a.N, a.K);
  const hipError_t e = launch_part(a, plan, 0, s);
  return e != hipSuccess || plan.n_rest == 0 ? e : launch_part(a, plan, 1, s);
}

}  // namespace gq
