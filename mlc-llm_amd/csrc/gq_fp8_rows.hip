// e4m3 block-scaled products of few rows (up to 64 a segment): the weights stream through once, bound by HBM.
//
//   y[r, n] = sum over blocks g of 128 of  xs[g, r] ws[n / 128, g] sum_{k in g} xq[r, k] wq[n, k]
//
// A workgroup of eight waves takes rows of W sixteen at a time; KW of its waves share their K, SB blocks of 128 each, and the
// other 8 / KW factor works on further rows.  A wave keeps its part of x, all rows of it, in registers as e4m3 operands for
// the whole kernel, and the W it will need next is in flight while it computes: one load instruction covers 16 rows x 64 bytes.
// Sums are float32 on v_mfma_f32_16x16x32_bf16 (W is operand A, x operand B; a bfloat16 holds an e4m3 number exactly): at these
// sizes the conversion costs nothing that the memory would not cost anyway.  A lane of a result holds one row of x and four of W,
// so both scales of a block are one number; the waves' sums meet in LDS, where the epilogue runs.
//
// x may arrive quantised, or as numbers that each workgroup quantises itself (a launch less): a lane holds the 32 numbers
// of a row and block that its operand needs, and the row's maximum is two exchanges away.
#include "gq_fp8_common.hpp"
#include "gq_topk.hpp"

namespace gq {

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
typedef uint32_t uint4_vt __attribute__((ext_vector_type(4)));

constexpr int kRowWaves = 8;
constexpr int kRowBlocks = 512;  // workgroups of a launch: two a CU

// sixteen neighbouring numbers as float32, of which the first `count` are there (a multiple of 8, or ends of K % 16)
template <int DT>
__device__ __forceinline__ void load16(const void* p, int64_t i, bool there, float (&f)[16]) {
#pragma unroll
  for (int v = 0; v < 16; ++v) f[v] = 0.f;
  if (!there) return;
  if constexpr (DT == MODEL_F32) {
    const float4_t* q = reinterpret_cast<const float4_t*>(static_cast<const float*>(p) + i);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const float4_t a = q[h];
#pragma unroll
      for (int v = 0; v < 4; ++v) f[4 * h + v] = a[v];
    }
  } else {
    const uint4_vt* q = reinterpret_cast<const uint4_vt*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4_vt a = q[h];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        f[8 * h + 2 * v] = DT == MODEL_BF16 ? bf2f(a[v] & 0xffffu) : h2f(a[v] & 0xffffu);
        f[8 * h + 2 * v + 1] = DT == MODEL_BF16 ? bf2f(a[v] >> 16) : h2f(a[v] >> 16);
      }
    }
  }
}

// Four neighbouring results (SILU: of the gate and of the up rows) of row r.
template <bool SILU>
__device__ __forceinline__ void store_rows(const Fp8RowsArgs& p, int64_t r, int n, int N, const float4_t* v) {
  float o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = SILU ? silu_mul_f32(v[0][i], v[SILU ? 1 : 0][i]) : v[0][i];
  if (n < N) fp8_store<4>(p, r, n, N, N % 4 == 0 && p.y_aligned, o);
}

}  // namespace

// Sixteen rows of W a step (SILU: sixteen gate rows and their sixteen up rows), 16 MT rows of x a pass.
template <int MT, int SB, int X, bool SILU>
__global__ __launch_bounds__(64 * kRowWaves, 2) void fp8_rows_kernel(Fp8RowsArgs p, int kw_log2, int steps, int phases) {
  constexpr int NR = SILU ? 2 : 1;
  __shared__ float4_t sums[2][kRowWaves][NR][MT][64];
  __shared__ int32_t slot_of[16 * MT];
  __shared__ uint32_t used[16];
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KW = 1 << kw_log2, NW = kRowWaves >> kw_log2, kw = wave & (KW - 1), nw = wave >> kw_log2;
  const int K = static_cast<int>(p.K), N = static_cast<int>(p.N);
  const int groups = (K + kFp8Block - 1) / kFp8Block, n_blocks = (N + kFp8Block - 1) / kFp8Block;
  const int col = lane & 15, quad = lane >> 4;

  // the segment: expert e, `rows` rows, the first of them row r0 (indptr) or kept as a list of slots (ids)
  int e = 0, rows = static_cast<int>(p.rows), r0 = 0;
  if (p.ids != nullptr) {
    const int want = blockIdx.y;
    if (p.rows <= p.top_k) {  // one token: its slots are the segments
      e = p.ids[want];
      if (e < 0 || e >= p.experts) return;
      rows = 1;
      r0 = want;
    } else {
      if (tid < 16) used[tid] = 0u;
      __syncthreads();
      for (int s = tid; s < p.rows; s += 64 * kRowWaves) {
        const int id = p.ids[s];
        if (id >= 0 && id < p.experts) atomicOr(&used[id >> 5], 1u << (id & 31));
      }
      __syncthreads();
      int before = 0;
      e = -1;
#pragma unroll
      for (int w = 0; w < 16; ++w) {  // the want-th bit that is set
        uint32_t u = used[w];
        const int c = __builtin_popcount(u);
        if (e < 0 && want < before + c) {
          for (int i = before; i < want; ++i) u &= u - 1;
          e = 32 * w + __builtin_ctz(u);
        }
        before += c;
      }
      if (e < 0) return;
      e = __builtin_amdgcn_readfirstlane(e);
    }
  } else if (p.indptr != nullptr) {
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

  typedef const __attribute__((address_space(4))) float* scalar_floats;  // read through the scalar cache
  const uint32_t pitch = static_cast<uint32_t>(p.w_pitch);
  const rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w + static_cast<int64_t>(e) * N * p.w_pitch), 0,
                                                          static_cast<int>((N - 1) * pitch + K), 0x00027000);
  const scalar_floats ws = (scalar_floats)(p.ws + static_cast<int64_t>(e) * n_blocks * groups);
  // block b of this wave in phase ph of K
  auto block_of = [&](int ph, int b) { return (ph * KW + kw) * SB + b; };
  // row of W that this lane reads in step s, part i
  const int half = N >> 1;
  auto w_row = [&](int s, int i) {
    int n = 16 * s + col;
    if (SILU) return (n < half ? n : half - 1) + i * half;
    return n < N ? n : N - 1;
  };
  int4_t wq[NR][SB][2];
  // A chunk past K (16 bytes; K is a multiple of 16) is read from the row's start: x has zeros there.
  auto load_w = [&](int s, int ph, int i, int b) {
    const uint32_t at = static_cast<uint32_t>(w_row(s, i)) * pitch;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = block_of(ph, b) * kFp8Block + 64 * h + 16 * quad;
      wq[i][b][h] = __builtin_bit_cast(int4_t, __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, at + (k < K ? k : 0), 0, 0));
    }
  };
  const int stride = gridDim.x * NW, s_first = blockIdx.x * NW + nw, rounds = (steps + stride - 1) / stride;
  auto clamp_step = [&](int s) { return s < steps ? s : steps - 1; };

  for (int pass = 0; pass < rows; pass += 16 * MT) {
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int b = 0; b < SB; ++b) load_w(clamp_step(s_first), 0, i, b);

    if (p.ids != nullptr && p.rows > p.top_k) {  // the pass's slots, in order
      if (tid == 0) found = 0;
      __syncthreads();
      if (wave == 0) {
        int seen = 0;
        for (int s0 = 0; s0 < p.rows; s0 += 64) {
          const int s = s0 + lane;
          const unsigned long long m = __ballot(s < p.rows && p.ids[s < p.rows ? s : 0] == e);
          const int at = seen + __popcll(m & ((1ull << lane) - 1ull)) - pass;
          if (((m >> lane) & 1ull) && at >= 0 && at < 16 * MT) slot_of[at] = s;
          seen += __popcll(m);
        }
        if (lane == 0) found = seen;
      }
      __syncthreads();
      rows = found;
      if (pass >= rows) break;  // (uniform)
    }
    auto y_row = [&](int m) -> int64_t {  // row of y behind row m of the segment
      if (p.ids != nullptr) return p.rows <= p.top_k ? r0 : slot_of[m - pass];
      return r0 + m;
    };
    auto x_row = [&](int m) -> int64_t {
      int64_t r = y_row(m);
      if (p.ids != nullptr) return r / p.x_div;
      if (p.x_row_index != nullptr) {
        r = p.x_row_index[r];
        r = r < 0 ? 0 : r < p.x_rows ? r : p.x_rows - 1;
      }
      return r;
    };

    int4_t xq[SB][MT][2];
    float xs[SB][MT];
    auto load_x = [&](int ph) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int m = pass + 16 * t + col;
      const bool here = m < rows;
      const int64_t r = here ? x_row(m) : 0;
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        const int k = block_of(ph, b) * kFp8Block + 16 * quad;
        if constexpr (X == kXFp8) {
          const int4_t none = {0, 0, 0, 0};
          xq[b][t][0] = here && k < K ? *reinterpret_cast<const int4_t*>(static_cast<const uint8_t*>(p.x) + r * p.x_pitch + k) : none;
          xq[b][t][1] = here && k + 64 < K ? *reinterpret_cast<const int4_t*>(static_cast<const uint8_t*>(p.x) + r * p.x_pitch + k + 64) : none;
          xs[b][t] = here && block_of(ph, b) < groups ? p.xs[block_of(ph, b) * p.x_rows + r] : 0.f;
        } else {
          float lo[16], hi[16];
          load16<X>(p.x, r * K + k, here && k < K, lo);
          load16<X>(p.x, r * K + k + 64, here && k + 64 < K, hi);
          float top = 0.f;
#pragma unroll
          for (int v = 0; v < 16; ++v) top = fmaxf(top, fmaxf(fp8_magnitude(lo[v]), fp8_magnitude(hi[v])));
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const uint32_t bits = fp8_scale_bits(top);
          const float inv = fp8_inverse(bits);
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            xq[b][t][0][v] = fp8_quad(lo[4 * v] * inv, lo[4 * v + 1] * inv, lo[4 * v + 2] * inv, lo[4 * v + 3] * inv);
            xq[b][t][1][v] = fp8_quad(hi[4 * v] * inv, hi[4 * v + 1] * inv, hi[4 * v + 2] * inv, hi[4 * v + 3] * inv);
          }
          xs[b][t] = __builtin_bit_cast(float, bits);
        }
      }
    }

    };
    if (phases == 1) load_x(0);

    for (int round = 0; round < rounds; ++round) {
      const int s = s_first + round * stride, sc = clamp_step(s), s_after = clamp_step(s + stride);
      float4_t acc[NR][MT];
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[i][t] = float4_t{};
      for (int ph = 0; ph < phases; ++ph) {
      if (phases > 1) load_x(ph);
      const int ph_next = ph + 1 < phases ? ph + 1 : 0, s_next = ph + 1 < phases ? sc : s_after;
      scalar_floats wsr[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int wb = (16 * sc + i * half) / kFp8Block;  // (half is a multiple of 16: sixteen rows share a block)
        wsr[i] = ws + (wb < n_blocks ? wb : n_blocks - 1) * groups;
      }
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        bf16x8_t a[NR][4];
        float w_scale[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            a[i][2 * h] = fp8_widen(wq[i][b][h][0], wq[i][b][h][1]);
            a[i][2 * h + 1] = fp8_widen(wq[i][b][h][2], wq[i][b][h][3]);
          }
          load_w(s_next, ph_next, i, b);
          w_scale[i] = wsr[i][block_of(ph, b) < groups ? block_of(ph, b) : groups - 1];
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          int4_t x0 = xq[b][t][0], x1 = xq[b][t][1];
          if (MT * SB > 4) asm volatile("" : "+v"(x0), "+v"(x1));  // (widened anew each round: the registers would not hold all of it)
          const bf16x8_t xw[4] = {fp8_widen(x0[0], x0[1]), fp8_widen(x0[2], x0[3]), fp8_widen(x1[0], x1[1]), fp8_widen(x1[2], x1[3])};
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            float4_t part = {};
#pragma unroll
            for (int h = 0; h < 4; ++h) part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i][h], xw[h], part, 0, 0, 0);
            const float scale = w_scale[i] * xs[b][t];
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[i][t][v] = __builtin_fmaf(part[v], scale, acc[i][t][v]);
          }
        }
      }
      }
      // the KW waves of a step add up, in LDS that the rounds take in turn: one barrier a round
      if (KW > 1) {
        auto& buf = sums[round & 1];
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int t = 0; t < MT; ++t) buf[wave][i][t][lane] = acc[i][t];
        __syncthreads();
        for (int t = kw; t < MT; t += KW) {
          float4_t v[NR];
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            v[i] = buf[nw << kw_log2][i][t][lane];
            for (int w = 1; w < KW; ++w) v[i] += buf[(nw << kw_log2) + w][i][t][lane];
          }
          const int m = pass + 16 * t + col;
          if (m < rows && s < steps) store_rows<SILU>(p, y_row(m), 16 * s + 4 * quad, SILU ? half : N, v);
        }
      } else {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          float4_t v[NR];
#pragma unroll
          for (int i = 0; i < NR; ++i) v[i] = acc[i][t];
          const int m = pass + 16 * t + col;
          if (m < rows && s < steps) store_rows<SILU>(p, y_row(m), 16 * s + 4 * quad, SILU ? half : N, v);
        }
      }
    }
    if (pass + 16 * MT < rows) __syncthreads();
  }
}

// Work distribution: the waves that share K (as few as hold it in one phase), steps a workgroup, segments in grid.y.
template <int MT, int SB, int X, bool SILU>
static hipError_t launch_rows(const Fp8RowsArgs& a, hipStream_t s) {
  const int groups = static_cast<int>((a.K + kFp8Block - 1) / kFp8Block);
  int kw_log2 = 0;
  while (kw_log2 < 3 && (SB << kw_log2) < groups) ++kw_log2;
  const int phases = (groups + (SB << kw_log2) - 1) / (SB << kw_log2), nw = kRowWaves >> kw_log2;
  const int steps = static_cast<int>(((SILU ? a.N / 2 : a.N) + 15) / 16), sets = (steps + nw - 1) / nw;
  const int segments = a.ids ? (a.rows <= a.top_k ? static_cast<int>(a.rows) : static_cast<int>(a.rows < a.experts ? a.rows : a.experts))
                             : a.indptr ? static_cast<int>(a.rows < a.experts ? a.rows : a.experts) : 1;
  const int want = (kRowBlocks + segments - 1) / segments, rounds = (sets + want - 1) / want;
  const dim3 grid((sets + rounds - 1) / rounds, segments);
  note_kernel("fp8_rows %d rows, %d blocks x %d waves, %d phases", 16 * MT, SB, 1 << kw_log2, phases);
  hipLaunchKernelGGL((fp8_rows_kernel<MT, SB, X, SILU>), grid, dim3(64 * kRowWaves), 0, s, a, kw_log2, steps, phases);
  return hipGetLastError();
}

template <int MT, int X, bool SILU>
static hipError_t launch_rows_by_k(const Fp8RowsArgs& a, hipStream_t s) {
  if constexpr (MT == 4) return launch_rows<MT, 2, X, SILU>(a, s);
  else if (a.K <= 2048) return launch_rows<MT, 2, X, SILU>(a, s);
  else return launch_rows<MT, 4, X, SILU>(a, s);
}

template <int X, bool SILU>
static hipError_t launch_rows_by_rows(const Fp8RowsArgs& a, int rows_max, hipStream_t s) {
  if constexpr (X == kXFp8) {
    if (rows_max > 32) return launch_rows_by_k<4, X, SILU>(a, s);
    if (rows_max > 16) return launch_rows_by_k<2, X, SILU>(a, s);
  }
  return launch_rows_by_k<1, X, SILU>(a, s);
}

hipError_t launch_fp8_rows(const Fp8RowsArgs& a, int rows_max, hipStream_t s) {
  if (a.K % 16 != 0 || (a.silu && a.N % 32 != 0) || static_cast<uint64_t>(a.N) * a.w_pitch >= 0xffffffffull) return hipErrorNotSupported;
  if (a.silu) {
    if (a.x_kind == kXFp8) return launch_rows_by_rows<kXFp8, true>(a, rows_max, s);
    if (a.x_kind == MODEL_BF16) return launch_rows_by_rows<MODEL_BF16, true>(a, rows_max, s);
    if (a.x_kind == MODEL_F16) return launch_rows_by_rows<MODEL_F16, true>(a, rows_max, s);
    return launch_rows_by_rows<MODEL_F32, true>(a, rows_max, s);
  }
  if (a.x_kind == kXFp8) return launch_rows_by_rows<kXFp8, false>(a, rows_max, s);
  if (a.x_kind == MODEL_BF16) return launch_rows_by_rows<MODEL_BF16, false>(a, rows_max, s);
  if (a.x_kind == MODEL_F16) return launch_rows_by_rows<MODEL_F16, false>(a, rows_max, s);
  return launch_rows_by_rows<MODEL_F32, false>(a, rows_max, s);
}

}  // namespace gq
