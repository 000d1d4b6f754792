// Products with 16-bit weights for any sizes and alignments: tiles of 64 x 64 through LDS, element by element.
//
// It serves what the others do not take: rows that do not start at 16 bytes (K no multiple of 8, or x or W in the middle of
// something), which models do not have.  Bound by its 2-byte loads.
#include "gq_dense_common.hpp"

namespace gq {

namespace {
constexpr int kTile = 64, kStep = 32, kRow = kStep + 8;  // (rows of 80 bytes: 16-byte reads of 16 rows meet all banks evenly)
}

// Four waves, each 16 rows of x by 64 rows of W; gated: 32 gate rows and the 32 up rows that belong to them.
template <bool BF, bool GATED>
__global__ __launch_bounds__(256) void dense_simple_kernel(DenseArgs a, int64_t n_tiles, int64_t tiles) {
  __shared__ __attribute__((aligned(16))) uint16_t xs[kTile * kRow], ws[kTile * kRow];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int P = GATED ? 2 : 1, kCols = kTile / P;
  const int64_t half = a.N / P;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t mt = tile / n_tiles, r0 = mt * kTile, n0 = (tile - mt * n_tiles) * kCols;
    float4_t acc[4] = {};
    for (int64_t k0 = 0; k0 < a.K; k0 += kStep) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kTile * kStep / 256; ++i) {
        const int at = i * 256 + tid, row = at / kStep, k = at % kStep;
        const int64_t n = n0 + row % kCols;
        const bool in = k0 + k < a.K;
        xs[row * kRow + k] = in && r0 + row < a.rows ? a.x[(r0 + row) * a.K + k0 + k] : 0;
        ws[row * kRow + k] = in && n < half ? a.w[(n + row / kCols * half) * a.K + k0 + k] : 0;
      }
      __syncthreads();
      const int4_t x = *reinterpret_cast<const int4_t*>(xs + (16 * wave + (lane & 15)) * kRow + 8 * (lane >> 4));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[i] = dense_mfma<BF>(*reinterpret_cast<const int4_t*>(ws + (16 * i + (lane & 15)) * kRow + 8 * (lane >> 4)), x, acc[i]);
    }
    const int64_t r = r0 + 16 * wave + (lane & 15);
#pragma unroll
    for (int i = 0; i < 4 / P; ++i) {
      const int64_t n = n0 + 16 * i + 4 * (lane >> 4);
      if (r < a.rows && n < half) {
        const float4_t g = acc[i], up = acc[GATED ? i + 2 : i];
        float o[4] = {g[0], g[1], g[2], g[3]}, u[4] = {up[0], up[1], up[2], up[3]};
        dense_store<BF, 4, GATED>(a, r, static_cast<int>(n), o, u);
      }
    }
  }
}

hipError_t launch_dense_simple(const DenseArgs& a, hipStream_t s) {
  const int64_t cols = a.gated ? kTile / 2 : kTile, n_tiles = ((a.gated ? a.N / 2 : a.N) + cols - 1) / cols;
  const int64_t tiles = n_tiles * ((a.rows + kTile - 1) / kTile);
  const dim3 grid(static_cast<unsigned>(tiles < 65536 ? tiles : 65536));
  note_kernel("dense_simple%s", a.gated ? " gated" : "");
  auto go = [&](auto* kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a, n_tiles, tiles); };
  if (a.bf16) a.gated ? go(dense_simple_kernel<true, true>) : go(dense_simple_kernel<true, false>);
  else a.gated ? go(dense_simple_kernel<false, true>) : go(dense_simple_kernel<false, false>);
  return hipGetLastError();
}

}  // namespace gq
