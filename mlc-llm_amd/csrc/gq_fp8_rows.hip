// e4m3 block-scaled products of up to sixteen rows (a segment): the weights stream through once, bound by HBM.
//
//   y[r, n] = sum over blocks g of 128 of  xs[g, r] ws[n / 128, g] sum_{k in g} xq[r, k] wq[n, k]
//
// x lies in LDS as e4m3 groups and their scales; a wave takes rows of W sixteen at a time, straight from memory into registers
// (one load instruction covers 16 rows x 64 bytes), and has the next D blocks of 128 x 16 in flight while it computes one.
// KW of a workgroup's eight waves share the K of their rows, where there are too few rows to keep the memory busy otherwise,
// and their sums meet in LDS.
// Sums are float32 on v_mfma_f32_16x16x32_bf16 (W is operand A, x operand B; a bfloat16 holds an e4m3 number exactly): at these
// sizes the conversion costs nothing that the memory would not cost anyway.  A lane of a result holds one row of x and four of
// W, so both scales of a block are one number.
//
// x may arrive quantised, or as numbers that each workgroup quantises itself on their way to LDS (a launch less).
//
// Measured: 4096 x 4096 of 2 / 8 rows 8.8 / 11.8 us, 28672 x 4096 of 8 rows 28.7 us (4.1 TB/s; bound by HBM, and by the x that each of
// its workgroups quantises).  16 tokens over 128 experts of 2048 x 768: gate/up 44 us, down 27 us (about 390 MB, 5.5 TB/s).
#include "gq_fp8_common.hpp"

namespace gq {

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;

constexpr int kRowWaves = 8;
constexpr int kRowTarget = 2048;   // waves that keep the memory busy
constexpr int kRowDepth = 4;       // blocks of 16 x 128 that a wave has in flight
constexpr int kRowHead = 256;      // bytes of LDS in front of x
constexpr int kRowLds = 152 * 1024;  // of a workgroup: x and the sums

}  // namespace

// Sixteen rows of W a step, sixteen rows of x a pass.  SILU: sixteen gate rows and their sixteen up rows a step, the activation
// quantised in the epilogue; a workgroup's eight steps are one group of it, so that its waves share no K.
// nbw: blocks of K a wave and phase, a multiple of D; phase_blocks = KW nbw blocks of x lie in LDS at a time.
template <int X, bool SILU>
__global__ __launch_bounds__(64 * kRowWaves, 4) void fp8_rows_kernel(Fp8RowsArgs p, int kw_log2, int nbw, int steps, int phases) {
  constexpr int NR = SILU ? 2 : 1, D = kRowDepth / NR;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int32_t* const source_of = reinterpret_cast<int32_t*>(smem);  // [16] rows of x
  uint8_t* const x_lds = smem + kRowHead;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KW = 1 << kw_log2, NW = kRowWaves >> kw_log2, kw = wave & (KW - 1), nw = wave >> kw_log2;
  const int K = static_cast<int>(p.K), N = static_cast<int>(p.N);
  const int groups = (K + kFp8Block - 1) / kFp8Block, n_blocks = (N + kFp8Block - 1) / kFp8Block;
  const int col = lane & 15, quad = lane >> 4, phase_blocks = KW * nbw, x_pitch = phase_blocks * kFp8Block;

  // the segment: expert e, `rows` rows from row r0 on
  int e = 0, rows = static_cast<int>(p.rows), r0 = 0;
  if (p.indptr != nullptr) {
    int before = 0;
    e = -1;
    for (int i0 = 0; i0 < p.experts && e < 0; i0 += 64) {  // the segment that is the blockIdx.y-th with any rows
      const int i = i0 + lane;
      const unsigned long long m = __ballot(i < p.experts && p.indptr[i < p.experts ? i + 1 : 1] > p.indptr[i < p.experts ? i : 0]);
      const int c = __popcll(m);
      if (static_cast<int>(blockIdx.y) < before + c) {
        unsigned long long u = m;
        for (int t = before; t < static_cast<int>(blockIdx.y); ++t) u &= u - 1;
        e = i0 + __builtin_ctzll(u);
      }
      before += c;
    }
    if (e < 0) return;
    e = __builtin_amdgcn_readfirstlane(e);
    r0 = p.indptr[e];
    rows = p.indptr[e + 1] - r0;
    if (r0 < 0 || r0 + rows > p.rows) return;
  }

  const uint32_t pitch = static_cast<uint32_t>(p.w_pitch);
  const rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w + static_cast<int64_t>(e) * N * p.w_pitch), 0,
                                                          static_cast<int>((N - 1) * pitch + K), 0x00027000);
  const rsrc_t s_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p.ws + static_cast<int64_t>(e) * n_blocks * groups), 0,
                                                          n_blocks * groups * 4, 0x00027000);
  constexpr uint32_t kNowhere = 0xffffffffu;  // past any buffer's end: reads as zeros, and asks the memory for nothing
  const int half = N >> 1;
  const int stride = gridDim.x * NW, s_first = blockIdx.x * NW + nw, rounds = (steps + stride - 1) / stride;
  // D blocks of this wave from block `from` on (of the phase's share of K), for step s; and their scales, one a lane
  int4_t wq[NR][D][2];
  float wsc[NR];
  auto block_of = [&](int ph, int b) { return ph * phase_blocks + kw * nbw + b; };
  auto load_scales = [&](int s, int ph, int from) {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int kb = block_of(ph, from) + lane, wb = (16 * s + i * half) / kFp8Block;  // (half is a multiple of 16: sixteen rows share a block)
      const uint32_t at = lane < D && kb < groups && s < steps ? static_cast<uint32_t>(wb * groups + kb) * 4 : kNowhere;
      wsc[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(s_rsrc, at, 0, 0));
    }
  };
  auto row_at = [&](int s, int i) {  // where this lane's row of W of step s starts, if there is such a row
    const int n = 16 * s + col;
    return s < steps && n < (SILU ? half : N) ? static_cast<uint32_t>(n + i * half) * pitch : kNowhere;
  };
  auto load_w = [&](uint32_t at, int ph, int i, int b, int slot) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = block_of(ph, b) * kFp8Block + 64 * h + 16 * quad;  // a chunk of 16; K is a multiple of 16
      wq[i][slot][h] = __builtin_bit_cast(int4_t, __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, at != kNowhere && k < K ? at + k : kNowhere, 0, 0));
    }
  };

  for (int pass = 0; pass < rows; pass += 16) {
    load_scales(s_first, 0, 0);
#pragma unroll
    for (int b = 0; b < D; ++b)
#pragma unroll
      for (int i = 0; i < NR; ++i) load_w(row_at(s_first, i), 0, i, b, b);

    const int here = rows - pass < 16 ? rows - pass : 16;  // rows of x in LDS
    float* const xs = reinterpret_cast<float*>(x_lds + 16 * x_pitch);  // [phase_blocks][16]
    auto y_row = [&](int m) -> int64_t { return r0 + pass + m; };  // row of y behind row m of the pass
    auto x_row = [&](int m) -> int64_t {
      int64_t r = y_row(m);
      if (p.x_row_index != nullptr) r = p.x_row_index[r];
      return r < 0 ? 0 : r < p.x_rows ? r : p.x_rows - 1;
    };
    if (tid < here) source_of[tid] = static_cast<int32_t>(x_row(tid));
    __syncthreads();
    // Phase ph of x to LDS: chunk c of a row's block at place c ^ (row & 7), so that the 16 lanes that LDS serves at a time meet 16
    // places.  Past K stands something of the same row (W is zero there), and lanes whose row is not there read the last one:
    // their results are never stored.
    auto stage_x = [&](int ph) {
      const int first = ph * phase_blocks;
      if constexpr (X == kXFp8) {
        // eight blocks of a row a load, past the registers: a lane asks for the chunk that belongs at its place
        const int runs = (phase_blocks + 7) / 8;
        for (int c = wave; c < here * runs; c += kRowWaves) {
          const int m = __builtin_amdgcn_readfirstlane(c / runs), run = c - m * runs, at = run * 64 + lane;
          const int k = first * kFp8Block + (at & ~7) * 16 + (((at & 7) ^ (m & 7)) << 4);
          const uint8_t* from = static_cast<const uint8_t*>(p.x) + static_cast<int64_t>(source_of[m]) * p.x_pitch;
          if (run * 8 + (lane >> 3) < phase_blocks)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + (k < K ? k : 0)),
                                             (__attribute__((address_space(3))) void*)(x_lds + m * x_pitch + run * 1024), 16, 0, 0);
        }
        for (int c = tid; c < phase_blocks * here; c += 64 * kRowWaves) {
          const int b = c / here, m = c - b * here;
          xs[b * 16 + m] = first + b < groups ? p.xs[(first + b) * p.x_rows + source_of[m]] : 0.f;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      } else {
        // a group is 16 lanes of eight numbers, four groups a wave; U rows of them in flight
        constexpr int U = 2;
        for (int m0 = 0; m0 < here; m0 += U)
          for (int b = tid >> 4; b < phase_blocks; b += 4 * kRowWaves) {
            const int k = (first + b) * kFp8Block + 8 * (lane & 15);
            float f[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u)
              fp8_load8<X>(p.x, static_cast<int64_t>(source_of[m0 + u < here ? m0 + u : m0]) * K + (k < K ? k : 0), f[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
              for (int v = 0; v < 8; ++v) f[u][v] = k < K ? f[u][v] : 0.f;
              uint32_t bits;
              const uint2 out = fp8_group(f[u], &bits);
              const int m = m0 + u, chunk = (lane & 15) >> 1;
              if (m < here) {
                *reinterpret_cast<uint2*>(x_lds + m * x_pitch + b * kFp8Block + ((chunk ^ (m & 7)) << 4) + 8 * (lane & 1)) = out;
                if ((lane & 15) == 0) xs[b * 16 + m] = __builtin_bit_cast(float, bits);
              }
            }
          }
      }
    };
    const int x_at = col < here ? col : here - 1;  // this lane's row of x in LDS
    float4_t* const sums = reinterpret_cast<float4_t*>(x_lds + 16 * (x_pitch + phase_blocks * 4));  // [2][waves][64]
    if (phases == 1) {
      stage_x(0);
      __syncthreads();
    }

    for (int round = 0; round < rounds; ++round) {
      const int s = s_first + round * stride;
      float4_t acc[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) acc[i] = float4_t{};
      for (int ph = 0; ph < phases; ++ph) {
        if (phases > 1) {
          __syncthreads();  // (the phase before it has been read)
          stage_x(ph);
          __syncthreads();
        }
        for (int b0 = 0; b0 < nbw; b0 += D) {
          // what comes behind these D blocks: further ones, the next phase, the next step, or nothing
          const bool more = b0 + D < nbw, more_ph = ph + 1 < phases;
          const int b_next = more ? b0 + D : 0, ph_next = more ? ph : more_ph ? ph + 1 : 0;
          const int s_next = more || more_ph ? s : round + 1 < rounds ? s + stride : steps;
          uint32_t at[NR];
#pragma unroll
          for (int i = 0; i < NR; ++i) at[i] = row_at(s_next, i);
          float scale_now[NR];
#pragma unroll
          for (int i = 0; i < NR; ++i) scale_now[i] = wsc[i];
          load_scales(s_next, ph_next, b_next);
#pragma unroll
          for (int b = 0; b < D; ++b) {
            const int xb = kw * nbw + b0 + b;
            const uint8_t* const x = x_lds + x_at * x_pitch + xb * kFp8Block;
            const int4_t x0 = *reinterpret_cast<const int4_t*>(x + ((quad ^ (x_at & 7)) << 4));
            const int4_t x1 = *reinterpret_cast<const int4_t*>(x + (((quad + 4) ^ (x_at & 7)) << 4));
            const float x_scale = xs[xb * 16 + x_at];
            const bf16x8_t xw[4] = {fp8_widen(x0[0], x0[1]), fp8_widen(x0[2], x0[3]), fp8_widen(x1[0], x1[1]), fp8_widen(x1[2], x1[3])};
#pragma unroll
            for (int i = 0; i < NR; ++i) {
              bf16x8_t a[4];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                a[2 * h] = fp8_widen(wq[i][b][h][0], wq[i][b][h][1]);
                a[2 * h + 1] = fp8_widen(wq[i][b][h][2], wq[i][b][h][3]);
              }
              load_w(at[i], ph_next, i, b_next + b, b);
              const float scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale_now[i]), b)) * x_scale;
              float4_t part = {};
#pragma unroll
              for (int h = 0; h < 4; ++h) part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[h], xw[h], part, 0, 0, 0);
#pragma unroll
              for (int v = 0; v < 4; ++v) acc[i][v] = __builtin_fmaf(part[v], scale, acc[i][v]);
            }
            __builtin_amdgcn_sched_barrier(0);  // a block after the other: operands of two would not fit the registers
          }
        }
      }
      const int n = 16 * s + 4 * quad;
      const bool there = col < here && s < steps && n < N, vec = N % 4 == 0 && p.y_aligned;
      auto store = [&](const float4_t& v) {
        float o[4] = {v[0], v[1], v[2], v[3]};
        fp8_store<4>(p, r0 + pass + col, n, N, vec, o);
      };
      // the KW waves of a step add up, in LDS that the rounds take in turn: one barrier a round
      if (!SILU && KW > 1) {
        float4_t* const buf = sums + (round & 1) * kRowWaves * 64;
        buf[wave * 64 + lane] = acc[0];
        __syncthreads();
        if (kw == 0) {
          float4_t v = acc[0];
          for (int w = 1; w < KW; ++w) v += buf[(wave + w) * 64 + lane];
          if (there) store(v);
        }
      } else if (SILU) {
        // the workgroup's eight steps are one group of the activation: its top goes from wave to wave through LDS
        float* const tops = reinterpret_cast<float*>(sums);  // [waves][16]
        float h[4], top = 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          h[v] = silu_mul_f32(acc[0][v], acc[NR - 1][v]);
          top = fmaxf(top, fp8_magnitude(h[v]));
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (quad == 0) tops[wave * 16 + col] = top;
        __syncthreads();
        top = tops[col];
        for (int w = 1; w < kRowWaves; ++w) top = fmaxf(top, tops[w * 16 + col]);
        const uint32_t bits = fp8_scale_bits(top);
        const float inv = fp8_inverse(bits);
        if (col < here && s < steps) {
          const int64_t r = r0 + pass + col;
          *reinterpret_cast<uint32_t*>(p.q_out + r * half + 16 * s + 4 * quad) = fp8_quad(h[0] * inv, h[1] * inv, h[2] * inv, h[3] * inv);
          if (wave == 0 && quad == 0) p.scale_out[static_cast<int64_t>(s / 8) * p.rows + r] = __builtin_bit_cast(float, bits);
        }
        __syncthreads();
      } else {
        if (there) store(acc[0]);
      }
    }
    if (pass + 16 < rows) __syncthreads();  // (x, the slots and the sums of this pass have been read)
  }
}

// Work distribution.  KW: as few waves share K as keep about kRowTarget waves busy, and not fewer than D blocks a wave; phases of
// K where x would not fit LDS; as many workgroups as run at a time (two a CU where registers and LDS allow), four times that
// for segments, whose number and sizes vary, each with the same number of steps.
template <int X, bool SILU>
static hipError_t launch_rows(const Fp8RowsArgs& a, hipStream_t s) {
  constexpr int NR = SILU ? 2 : 1, D = kRowDepth / NR;
  const int64_t groups = (a.K + kFp8Block - 1) / kFp8Block;
  const int steps = static_cast<int>(((SILU ? a.N / 2 : a.N) + 15) / 16);
  const int64_t segments = a.indptr ? (a.rows < a.experts ? a.rows : a.experts) : 1;
  constexpr int64_t kBlockBytes = 16 * (kFp8Block + 4);
  static_assert(kRowLds / kBlockBytes >= D, "a wave's blocks fit");
  // blocks a wave and phase, as many as fit beside the sums
  const auto fit = [](int log2) {
    const int sums = log2 > 0 ? 2 * kRowWaves * 1024 : 0;
    return ((kRowLds - sums) / kBlockBytes >> log2) / D * D;
  };
  const auto share = [&](int log2) { return (((groups + (1 << log2) - 1) >> log2) + D - 1) / D * D; };
  int kw_log2 = 0;
  while (!SILU && kw_log2 < 3 && (steps * segments << kw_log2) < kRowTarget && (groups >> (kw_log2 + 1)) * 2 > D && fit(kw_log2 + 1) > 0 &&
         (fit(kw_log2 + 1) >= share(kw_log2 + 1) || fit(kw_log2) < share(kw_log2)))
    ++kw_log2;
  const int64_t phases = (share(kw_log2) + fit(kw_log2) - 1) / fit(kw_log2);
  const int64_t nbw = ((share(kw_log2) + phases - 1) / phases + D - 1) / D * D;
  const size_t lds = kRowHead + kBlockBytes * (nbw << kw_log2) + (kw_log2 > 0 ? 2 * kRowWaves * 1024 : kRowWaves * 16 * 4);
  const int64_t at_a_time = (segments > 1 ? 1024 : 256) * (lds <= 78 * 1024 ? 2 : 1);
  const int nw = kRowWaves >> kw_log2, sets = (steps + nw - 1) / nw;
  const int64_t want = (at_a_time + segments - 1) / segments, rounds = (sets + want - 1) / want;
  const dim3 grid(static_cast<unsigned>((sets + rounds - 1) / rounds), static_cast<unsigned>(segments));
  auto* kern = fp8_rows_kernel<X, SILU>;
  if (lds > 60 * 1024) {
    const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern));
    if (e != hipSuccess) return e;
  }
  note_kernel("fp8_rows %d blocks x %d waves, %d phases", static_cast<int>(nbw), 1 << kw_log2, static_cast<int>(phases));
  hipLaunchKernelGGL(kern, grid, dim3(64 * kRowWaves), lds, s, a, kw_log2, static_cast<int>(nbw), steps, static_cast<int>(phases));
  return hipGetLastError();
}

hipError_t launch_fp8_rows(const Fp8RowsArgs& a, hipStream_t s) {
  if (a.K % 16 != 0 || static_cast<uint64_t>(a.N) * a.w_pitch >= 0xffffffffull || (a.q_out != nullptr && !fp8_silu_takes(a.N, a.w_pitch)))
    return hipErrorNotSupported;
  if (a.q_out != nullptr) return launch_rows<kXFp8, true>(a, s);
  if (a.x_kind == kXFp8) return launch_rows<kXFp8, false>(a, s);
  if (a.x_kind == MODEL_BF16) return launch_rows<MODEL_BF16, false>(a, s);
  if (a.x_kind == MODEL_F16) return launch_rows<MODEL_F16, false>(a, s);
  return launch_rows<MODEL_F32, false>(a, s);
}

}  // namespace gq
