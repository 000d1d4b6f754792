// Products of up to 16 rows with 16-bit weights: the weights stream through once, bound by HBM.
#include "gq_dense_stream.hpp"

namespace gq {

// Eight waves: KW of them share the K of an item, 16 rows of W (gated: 8 gate rows and their up rows), and their sums meet in LDS.
template <bool BF, bool GATED, int XG>
__global__ __launch_bounds__(64 * kStreamWaves, 4) void dense_rows_kernel(DenseArgs a, int kw_log2, int nb) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int TT = (XG + 1) / 2, kCols = GATED ? 8 : 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int KW = 1 << kw_log2, kw = wave & (KW - 1), nw = wave >> kw_log2;
  const int K = static_cast<int>(a.K), rows = static_cast<int>(a.rows);
  const int64_t pitch = a.K * 2, cols = GATED ? a.N / 2 : a.N, n0 = (static_cast<int64_t>(blockIdx.x) * (kStreamWaves >> kw_log2) + nw) * kCols;
  uint8_t* const ring = smem + wave * stream_ring<XG, 1>();
  auto place_of = [&](int round) {
    StreamPlace<XG, 1> p;
    p.k = kw * kStreamBlock;
    p.end = round == 0 && n0 < cols ? K : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t left = GATED ? cols - n0 : cols - n0 - 8 * i, count = left < 0 ? 0 : left < 8 ? left : 8;
      p.w[i] = dense_buffer(reinterpret_cast<const char*>(a.w) + (n0 + i * (GATED ? cols : 8)) * pitch, count * pitch);
    }
    p.x[0] = dense_buffer(a.x, a.rows * pitch);
#pragma unroll
    for (int g = 0; g < XG; ++g) {
      const int r = 8 * g + (lane >> 3);
      p.x_at[g] = r < rows ? static_cast<uint32_t>(r) * static_cast<uint32_t>(pitch) : kNowhere;
    }
    return p;
  };
  auto done = [&](int, float4_t (&acc)[TT]) {
    if (KW > 1) {
      stream_join(reinterpret_cast<float4_t*>(smem + kStreamWaves * stream_ring<XG, 1>()), wave, KW, acc);
      if (kw != 0) return;
    }
    const int64_t n = n0 + 4 * (lane >> 4);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int r = 16 * t + (lane & 15);
      const float4_t g = acc[t], up = GATED ? stream_up(g) : g;
      float o[4] = {g[0], g[1], g[2], g[3]}, u[4] = {up[0], up[1], up[2], up[3]};
      if (r < rows && n < cols && (!GATED || lane < 32)) dense_store<BF, 4, GATED>(a, r, static_cast<int>(n), o, u);
    }
  };
  dense_stream<BF, XG>(ring, static_cast<uint32_t>(pitch), KW * kStreamBlock, nb, 1, place_of, done);
}

template <bool BF, bool GATED, int XG>
static hipError_t launch(const DenseArgs& a, hipStream_t s) {
  const int64_t cols = GATED ? a.N / 2 : a.N, items = (cols + (GATED ? 7 : 15)) / (GATED ? 8 : 16);
  const StreamPlan plan = stream_plan(a.K);
  const int nw = kStreamWaves >> plan.kw_log2;
  const size_t lds = kStreamWaves * (stream_ring<XG, 1>() + (plan.kw_log2 > 0 ? (XG + 1) / 2 * 1024 : 0));
  auto* kern = dense_rows_kernel<BF, GATED, XG>;
  if (lds > 65536) {
    const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern));
    if (e != hipSuccess) return e;
  }
  note_kernel("dense_rows up to %d rows%s, %d waves share K", 8 * XG, GATED ? " gated" : "", 1 << plan.kw_log2);
  constexpr int64_t kMost = 0xffffffffll / (64 * kStreamWaves);  // workgroups a launch: 2^32 work items would wrap, without an error
  if ((items + nw - 1) / nw > kMost) return hipErrorNotSupported;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((items + nw - 1) / nw)), dim3(64 * kStreamWaves), lds, s, a, plan.kw_log2, plan.nb);
  return hipGetLastError();
}

hipError_t launch_dense_rows(const DenseArgs& a, hipStream_t s) {
  auto go = [&](auto bf) {
    constexpr bool BF = decltype(bf)::value;
    if (a.gated) return a.rows <= 8 ? launch<BF, true, 1>(a, s) : launch<BF, true, 2>(a, s);
    return a.rows <= 8 ? launch<BF, false, 1>(a, s) : launch<BF, false, 2>(a, s);
  };
  if (a.rows > 16) return hipErrorNotSupported;
  return a.bf16 ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace gq
