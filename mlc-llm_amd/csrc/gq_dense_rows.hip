// Products of up to 16 rows with 16-bit weights: the weights stream through once, bound by HBM.
//
// 256 workgroups of eight waves, one a unit: together 64 KiB of weights a unit are on their way, which keeps the memory busy over a load's 1 to 2 us, and
// a launch has no second round of workgroups to ramp up.  Measured, us (TB/s of weights): 128256 x 4096 of 5 rows 152 (6.9); 28672 x 4096, gated, of one
// row 37.0 (6.3); 4096 x 4096 of one row 7.2 (4.7, of which 2.3 us are the launch); 128 x 2048 of 16 rows 5.4 with its call.
#include "gq_dense_stream.hpp"

namespace gq {

namespace {
constexpr int kDepth = 4;  // blocks in flight a wave
}

// Eight waves: KW of them share the K of an item, 16 rows of W (gated: 8 gate rows and their up rows), and their sums meet in LDS.  The arguments
// that the first loads wait for come first: a launch brings them in scalar registers (4096 x 4096 of one row 7.5 -> 7.2 us).
template <bool BF, bool GATED, int XG, bool ANY>
__global__ __launch_bounds__(64 * kStreamWaves, 2) void dense_rows_kernel(
    const uint16_t* __restrict__ x, const uint16_t* __restrict__ w, int K, int rows, int cols_, int kw_log2, int nb, int rounds, DenseArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int TT = (XG + 1) / 2, kCols = GATED ? 8 : 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int KW = 1 << kw_log2, kw = wave & (KW - 1), nw = wave >> kw_log2;
  const int64_t pitch = static_cast<int64_t>(K) * 2, cols = cols_, stride = static_cast<int64_t>(gridDim.x) * (kStreamWaves >> kw_log2);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kStreamWaves >> kw_log2) + nw;
  uint8_t* const ring = smem + wave * stream_ring<XG, kDepth>();
  auto place_of = [&](int round) {
    StreamPlace<XG> p;
    p.k = kw * kStreamBlock;
    const int64_t n0 = (round * stride + first) * kCols;
    p.end = round < rounds && n0 < cols ? K : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t left = GATED ? cols - n0 : cols - n0 - 8 * i, count = p.end == 0 || left < 0 ? 0 : left < 8 ? left : 8;
      p.w[i] = dense_buffer(reinterpret_cast<const char*>(w) + (n0 + i * (GATED ? cols : 8)) * pitch, count * pitch);
    }
    p.x = dense_buffer(x, rows * pitch);
#pragma unroll
    for (int g = 0; g < XG; ++g) {
      const int r = 8 * g + (lane >> 3);
      p.x_at[g] = r < rows ? static_cast<uint32_t>(r) * static_cast<uint32_t>(pitch) : kNowhere;
    }
    return p;
  };
  auto done = [&](int round, float4_t (&acc)[TT]) {
    if (KW > 1) {
      // (two buffers in turn: one barrier a round)
      stream_join(reinterpret_cast<float4_t*>(smem + kStreamWaves * stream_ring<XG, kDepth>()) + (round & 1) * kStreamWaves * TT * 64, wave, KW, acc);
      if (kw != 0) return;
    }
    const int64_t n = (round * stride + first) * kCols + 4 * (lane >> 4);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int r = 16 * t + (lane & 15);
      const float4_t g = acc[t], up = GATED ? stream_up(g) : g;
      float o[4] = {g[0], g[1], g[2], g[3]}, u[4] = {up[0], up[1], up[2], up[3]};
      if (r < rows && n < cols && (!GATED || lane < 32)) dense_store<BF, 4, GATED>(a, r, static_cast<int>(n), o, u);
    }
  };
  dense_stream<BF, XG, kDepth, ANY>(ring, static_cast<uint32_t>(pitch), KW * kStreamBlock, nb, rounds, place_of, done);
}

template <bool BF, bool GATED, int XG>
static hipError_t launch(const DenseArgs& a, hipStream_t s) {
  const int64_t cols = GATED ? a.N / 2 : a.N, items = (cols + (GATED ? 7 : 15)) / (GATED ? 8 : 16);
  const StreamPlan plan = stream_plan(static_cast<double>(items), a.K, kDepth, true);
  const int nw = kStreamWaves >> plan.kw_log2;
  const int64_t sets = (items + nw - 1) / nw;
  constexpr size_t lds = kStreamWaves * (stream_ring<XG, kDepth>() + 2 * ((XG + 1) / 2) * 1024);
  static_assert(lds <= 160 * 1024, "LDS of a unit");
  auto* kern = plan.nb % kDepth == 0 ? dense_rows_kernel<BF, GATED, XG, false> : dense_rows_kernel<BF, GATED, XG, true>;
  const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern));
  if (e != hipSuccess) return e;
  note_kernel("dense_rows up to %d rows%s, %d waves share K", 8 * XG, GATED ? " gated" : "", 1 << plan.kw_log2);
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((sets + plan.rounds - 1) / plan.rounds)), dim3(64 * kStreamWaves), lds, s, a.x, a.w,
                     static_cast<int>(a.K), static_cast<int>(a.rows), static_cast<int>(cols), plan.kw_log2, plan.nb, plan.rounds, a);
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
