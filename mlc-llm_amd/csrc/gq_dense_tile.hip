// Products with 16-bit weights of more than a few rows: which tile form takes them, in how many shares of K, and the join of these.
#include "gq_dense_tile.hpp"

namespace gq {

// the sums of the shares of K, in their order, and the epilogue.  Four columns a thread.
template <bool BF, bool GATED>
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
  dense_store<BF, 4, GATED>(p, r, n, o[0], o[GATED ? 1 : 0]);
}

hipError_t launch_dense_join(const DenseArgs& a, int splits, hipStream_t s) {
  const int64_t items = a.rows * (((a.gated ? a.N / 2 : a.N) + 3) / 4);
  const dim3 grid(static_cast<unsigned>((items + 255) / 256));
  auto go = [&](auto* kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a, splits); };
  if (a.bf16) a.gated ? go(dense_join_kernel<true, true>) : go(dense_join_kernel<true, false>);
  else a.gated ? go(dense_join_kernel<false, true>) : go(dense_join_kernel<false, false>);
  return hipGetLastError();
}

namespace {

// A form's tile, the workgroups of it that a unit holds (one or two), what a block of K of its tiles takes in ns: alone_ns where few run, one_ns where
// a unit has one each, full_ns where the units are full (L2 and clocks are shared), and what a byte of W takes from memory, with loads of lines that
// are read once for up to once_rows rows of x (6.8 TB/s where all the others get 4.8).  Fitted to 20000 timings of 420 shapes, 9 to 4096 rows, all
// forms, 1 to 16 shares: the choice takes 1.4 % longer than the best one on average, 21 % at most.  (160 rows of x: 1.5 % on average over 130 to 2048
// rows, 10 % at 160, 320 and 800 of them.)
struct Form {
  int bn, bm, a_unit;
  float alone_ns, one_ns, full_ns;
  int once_rows;
  float once_ns;
};
constexpr int kForms = 11;
constexpr Form kForm[kForms] = {{256, 256, 1, 813.f, 1479.f, 1479.f, 0, 0.f},      {256, 192, 1, 794.f, 1298.f, 1298.f, 0, 0.f},
                                {256, 128, 1, 645.f, 920.f, 920.f, 0, 0.f},        {128, 192, 1, 642.f, 753.f, 753.f, 0, 0.f},
                                {128, 128, 1, 453.f, 561.f, 561.f, 128, 1.56e-4f}, {128, 128, 2, 530.f, 601.f, 925.f, 0, 0.f},
                                {64, 128, 1, 275.f, 326.f, 326.f, 128, 1.75e-4f},  {64, 64, 2, 205.f, 218.f, 654.f, 64, 1.48e-4f},
                                {64, 32, 2, 142.f, 216.f, 546.f, 32, 1.48e-4f},    {128, 160, 1, 569.f, 643.f, 643.f, 0, 0.f},
                                {256, 160, 1, 784.f, 1079.f, 1079.f, 0, 0.f}};
// a round's ends, the launch that joins, a number of a share, a byte of W from memory and how much more it takes with no unit busy, a second launch
// for the rest of the last round
constexpr float kRoundNs = 3325.f, kJoinNs = 2216.f, kShareNs = 1.94e-3f, kByteNs = 2.1e-4f, kIdle = 0.17f, kRestNs = 1500.f;
constexpr int64_t kUnits = 256;
// tiles, of `blocks` blocks each, that read w_bytes of W
float ns_of(const Form& f, int64_t rows, int64_t tiles, int64_t blocks, int64_t w_bytes) {
  const int64_t at_a_time = kUnits * f.a_unit, full = tiles / at_a_time, rest = tiles - full * at_a_time;
  float ns = full * (blocks * f.full_ns + kRoundNs);
  if (rest > kUnits) ns += blocks * f.full_ns + kRoundNs;
  else if (rest > 0) ns += blocks * (f.alone_ns + (f.one_ns - f.alone_ns) * rest / kUnits) + kRoundNs;
  const float from_memory = w_bytes * (rows <= f.once_rows ? f.once_ns : kByteNs) * (full > 0 ? 1.f : 1.f + kIdle * (at_a_time - tiles) / at_a_time);
  return ns > from_memory ? ns : from_memory;
}
bool may_take(int form) { return options().gemm_variant < 0 || options().gemm_variant >= kForms || options().gemm_variant == form; }
// N: rows of W
DensePlan plan_of(int64_t rows, int64_t N, int64_t K, bool only_whole = false) {
  const int64_t blocks = (K + kBlock - 1) / kBlock;
  DensePlan best;
  for (int f = 0; f < kForms; ++f) {
    if (!may_take(f) || (kForm[f].bm == 32 && rows > 32 && options().gemm_variant != f)) continue;
    const int64_t m_tiles = (rows + kForm[f].bm - 1) / kForm[f].bm, n_tiles = (N + kForm[f].bn - 1) / kForm[f].bn, tiles = m_tiles * n_tiles;
    for (int64_t want = 1; want <= 16 && want <= (only_whole || blocks < 4 ? 1 : blocks / 4); ++want) {
      if (options().gemm_split_k > 0 && options().gemm_split_k != want) continue;
      const int64_t per = (blocks + want - 1) / want, splits = (blocks + per - 1) / per;
      const float ns = ns_of(kForm[f], rows, tiles * splits, per, N * K * 2) + (splits > 1 ? kJoinNs + splits * rows * N * kShareNs : 0.f);
      if (best.per_split == 0 || ns < best.ns) {
        best = DensePlan{};
        best.form = f;
        best.splits = static_cast<int>(splits);
        best.per_split = static_cast<int>(per);
        best.ns = ns;
      }
    }
    // whole rounds of this form, and what is left of the last in a form that fills a round of its own
    const int64_t at_a_time = kUnits * kForm[f].a_unit, whole = tiles / at_a_time * at_a_time / m_tiles;
    if (!only_whole && options().gemm_split_k <= 1 && whole > 0 && whole < n_tiles) {
      const DensePlan rest = plan_of(rows, N - whole * kForm[f].bn, K, true);
      const float ns = ns_of(kForm[f], rows, whole * m_tiles, blocks, whole * kForm[f].bn * K * 2) + rest.ns + kRestNs;
      if (ns < best.ns) {
        best = DensePlan{};
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

// The plan of a call, made for its workspace and needed again for its launch right behind: 4 to 9 us of arithmetic, by sizes.
DensePlan plan_for(int64_t rows, int64_t N, int64_t K) {
  struct Last {
    int64_t rows = 0, N, K;
    int variant, split;
    DensePlan plan;
  };
  static thread_local Last last;
  const int variant = options().gemm_variant, split = options().gemm_split_k;
  if (last.rows != rows || last.N != N || last.K != K || last.variant != variant || last.split != split)
    last = {rows, N, K, variant, split, plan_of(rows, N, K)};
  return last.plan;
}

}  // namespace

int64_t dense_tile_workspace_bytes(int64_t rows, int64_t N, int64_t K) {
  const DensePlan p = plan_for(rows, N, K);
  return p.splits > 1 ? p.splits * rows * N * 4 : 0;
}

hipError_t launch_dense_tile(const DenseArgs& a, hipStream_t s) {
  const DensePlan plan = plan_for(a.rows, a.N, a.K);
  auto go = [&](int part) {
    return a.bf16 ? launch_dense_part_bf16(a, plan, part, s) : launch_dense_part_f16(a, plan, part, s);
  };
  const hipError_t e = go(0);
  return e != hipSuccess || plan.n_rest == 0 ? e : go(1);
}

}  // namespace gq
