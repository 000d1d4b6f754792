// Products of up to 32 rows with 16-bit weights: the weights stream through once, bound by HBM.
#include "gq_dense_stream.hpp"

namespace gq {

namespace {
constexpr int kWaves = 8;
constexpr double kTarget = 3000;  // waves that keep the memory busy
}

// Eight waves: KW of them share the K of an item, 16 NR rows of W (gated: 16 gate rows and their up rows), and their sums meet in LDS.
template <bool BF, bool GATED, int NR, int TT, int D>
__global__ __launch_bounds__(64 * kWaves, 4) void dense_rows_kernel(DenseArgs a, int kw_log2, int nb, int rounds) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int kTiles = NR * TT, kRows = GATED ? 16 : 16 * NR;
  float4_t* const sums = reinterpret_cast<float4_t*>(smem);  // [2][waves][kTiles][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int KW = 1 << kw_log2, kw = wave & (KW - 1), nw = wave >> kw_log2, stride = gridDim.x * (kWaves >> kw_log2);
  const int K = static_cast<int>(a.K), rows = static_cast<int>(a.rows), cols = static_cast<int>(GATED ? a.N / 2 : a.N);
  const int first = blockIdx.x * (kWaves >> kw_log2) + nw;
  const int64_t pitch = a.K * 2;
  auto place_of = [&](int round) {
    StreamPlace<NR, TT> p;
    const int64_t n0 = (static_cast<int64_t>(round) * stride + first) * kRows;
    const bool there = round < rounds && n0 < cols;
    p.end = there ? K : 0;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int64_t n = there ? n0 + (GATED ? 0 : 16 * i) : 0;
      const int64_t left = cols - n < 16 ? cols - n : 16;
      p.w[i] = dense_buffer(reinterpret_cast<const char*>(a.w) + (n + (GATED ? static_cast<int64_t>(i) * cols : 0)) * pitch, left > 0 ? left * pitch : 0);
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int r = 16 * t + (lane & 15);  // (a row that is not there reads the last one: its results are never stored)
      p.x_at[t] = static_cast<uint32_t>(r < rows ? r : rows - 1) * static_cast<uint32_t>(pitch);
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
    const int64_t n0 = (static_cast<int64_t>(round) * stride + first) * kRows + 4 * (lane >> 4);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int r = 16 * t + (lane & 15);
#pragma unroll
      for (int i = 0; i < (GATED ? 1 : NR); ++i) {
        const int64_t n = n0 + 16 * i;
        const float4_t g = acc[i][t], up = acc[GATED ? NR - 1 : i][t];
        float o[4] = {g[0], g[1], g[2], g[3]}, u[4] = {up[0], up[1], up[2], up[3]};
        if (r < rows && n < cols) dense_store<4, GATED>(a, r, static_cast<int>(n), o, u);
      }
    }
  };
  dense_stream<BF, NR, TT, D>(K, kw, KW, nb, rounds, dense_buffer(a.x, a.rows * pitch), place_of, done);
}

template <bool BF, bool GATED, int NR, int TT, int D>
static hipError_t launch(const DenseArgs& a, hipStream_t s) {
  const int64_t cols = GATED ? a.N / 2 : a.N, items = (cols + (GATED ? 16 : 16 * NR) - 1) / (GATED ? 16 : 16 * NR);
  const StreamPlan plan = stream_plan(static_cast<double>(items), a.K, D, kTarget);
  const int nw = kWaves >> plan.kw_log2;
  const int64_t sets = (items + nw - 1) / nw, rounds = (sets + 511) / 512;
  const size_t lds = plan.kw_log2 > 0 ? 2 * kWaves * NR * TT * 1024 : 0;
  note_kernel("dense_rows %d x %d tiles, %d waves share K", NR, TT, 1 << plan.kw_log2);
  hipLaunchKernelGGL((dense_rows_kernel<BF, GATED, NR, TT, D>), dim3(static_cast<unsigned>((sets + rounds - 1) / rounds)), dim3(64 * kWaves), lds, s, a,
                     plan.kw_log2, plan.nb, static_cast<int>(rounds));
  return hipGetLastError();
}

hipError_t launch_dense_rows(const DenseArgs& a, hipStream_t s) {
  auto go = [&](auto bf) {
    constexpr bool BF = decltype(bf)::value;
    if (a.gated) return a.rows <= 16 ? launch<BF, true, 2, 1, 2>(a, s) : launch<BF, true, 2, 2, 2>(a, s);
    return a.rows <= 16 ? launch<BF, false, 1, 1, 4>(a, s) : launch<BF, false, 2, 2, 2>(a, s);
  };
  if (a.rows > 32) return hipErrorNotSupported;
  return a.bf16 ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace gq
