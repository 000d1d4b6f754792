// e4m3 block-scaled matrix product y = x W^T with float32 sums, dense or by expert segments.
//
//   y[r, n] = sum over blocks g of 128 of  xs[g, r] ws[n / 128, g] sum_{k in g} xq[r, k] wq[n, k]
//
// The 8-bit matrix instructions do not sum in float32: they align a step's products to the largest one and drop what lies
// about 17 bits below it, 1e-5 of a typical result.  A bfloat16 holds an e4m3 number exactly and the bfloat16 instruction
// sums in float32, at half the rate and for a conversion in front (v_cvt_scalef32_pk_bf16_fp8, two numbers each).
//
// The weights are the instruction's A operand and the activations its B operand, so a lane of the result holds one row r of x
// and 16 rows n of W that share a block: the two scales of a block of K are one number per lane, and a block's sum joins
// the float32 accumulator with 16 multiply-adds.
#include "gq_fp8_common.hpp"
#include "gq_topk.hpp"

namespace gq {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// 16 bytes of a row at k, of which those at or past K count as zero; rows are 16-byte aligned and hold K rounded up to 16
__device__ __forceinline__ uint4 load_chunk(const uint8_t* row, int k, int K) {
  uint4 v = {0u, 0u, 0u, 0u};
  if (k < K) {
    v = *reinterpret_cast<const uint4*>(row + k);
    const int left = K - k;
    if (left < 16) {
      uint32_t* u = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int b = left - 4 * i;
        if (b <= 0) u[i] = 0u;
        else if (b < 4) u[i] &= (1u << (8 * b)) - 1u;
      }
    }
  }
  return v;
}

}  // namespace

// 64 rows of W by 64 rows of x, four waves of 32 x 32.
template <int OUT, int MODEL>
__global__ __launch_bounds__(256) void fp8_gemm_kernel(Fp8Args p, int m_tiles) {
  __shared__ __attribute__((aligned(16))) uint8_t sw[64 * 128], sx[64 * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n0 = blockIdx.x * 64;
  const int groups = static_cast<int>((p.K + kFp8Block - 1) / kFp8Block), n_blocks = static_cast<int>((p.N + kFp8Block - 1) / kFp8Block);
  int e = 0, r0 = blockIdx.y * 64, r_end = static_cast<int>(p.rows);
  if (p.indptr != nullptr) {
    // tiles of segment e are numbered from indptr[e] / 64 + e on: no two segments share a number, and some have no tile
    const int t = blockIdx.y;
    for (int i = 1; i < p.experts; ++i)
      if (p.indptr[i] / 64 + i <= t) e = i;
    const int begin = p.indptr[e];
    r0 = begin + (t - (begin / 64 + e)) * 64;
    r_end = p.indptr[e + 1] < r_end ? p.indptr[e + 1] : r_end;
  }
  if (r0 >= r_end || r0 < 0) return;
  const uint8_t* w = p.w + static_cast<int64_t>(e) * p.N * p.w_pitch;
  const float* ws = p.ws + static_cast<int64_t>(e) * n_blocks * groups;
  const int wn = (wave & 1) * 32, wm = (wave >> 1) * 32;
  auto source = [&](int r) -> int64_t {
    r = r < r_end ? r : r_end - 1;
    int64_t j = p.x_row_index ? p.x_row_index[r] : r;
    return j < 0 ? 0 : (j >= p.x_rows ? p.x_rows - 1 : j);
  };
  const int64_t my_x = source(r0 + wm + (lane & 31));
  float16_t acc = {};
  for (int g = 0; g < groups; ++g) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = (tid >> 3) + 32 * i, c = tid & 7, at = row * 128 + ((c ^ (row & 7)) << 4);
      const int64_t n = n0 + row < p.N ? n0 + row : p.N - 1;
      *reinterpret_cast<uint4*>(sw + at) = load_chunk(w + n * p.w_pitch, g * 128 + c * 16, static_cast<int>(p.K));
      *reinterpret_cast<uint4*>(sx + at) = load_chunk(p.x + source(r0 + row) * p.x_pitch, g * 128 + c * 16, static_cast<int>(p.K));
    }
    __syncthreads();
    const int bn = (n0 + wn) / kFp8Block < n_blocks ? (n0 + wn) / kFp8Block : n_blocks - 1;
    const float s = ws[static_cast<int64_t>(bn) * groups + g] * p.xs[g * p.x_rows + my_x];
    float16_t part = {};
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      auto frag = [&](const uint8_t* base, int row) {
        const uint2 v = *reinterpret_cast<const uint2*>(base + row * 128 + ((c ^ (row & 7)) << 4) + 8 * (lane >> 5));
        const bf16x2_dot_t a = __builtin_bit_cast(bf16x2_dot_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.x, 1.0f, false));
        const bf16x2_dot_t b = __builtin_bit_cast(bf16x2_dot_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.x, 1.0f, true));
        const bf16x2_dot_t d = __builtin_bit_cast(bf16x2_dot_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.y, 1.0f, false));
        const bf16x2_dot_t e = __builtin_bit_cast(bf16x2_dot_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.y, 1.0f, true));
        return bf16x8_t{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
      };
      part = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag(sw, wn + (lane & 31)), frag(sx, wm + (lane & 31)), part, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = __builtin_fmaf(part[i], s, acc[i]);
  }
  const int r = r0 + wm + (lane & 31);
  if (r >= r_end) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int n = n0 + wn + (i >> 2) * 8 + (lane >> 5) * 4 + (i & 3);
    if (n >= p.N) continue;
    float v = acc[i];
    if (p.bias) v += Elem<MODEL>::load(p.bias, n);
    if (p.residual) v += Elem<MODEL>::load(p.residual, r * p.N + n);
    Elem<OUT>::store(p.y, r * p.N + n, v);
  }
}

hipError_t launch_fp8_gemm(const Fp8Args& a, hipStream_t s) {
  const int64_t m_tiles = a.indptr ? a.rows / 64 + a.experts : (a.rows + 63) / 64;
  const dim3 grid(static_cast<unsigned>((a.N + 63) / 64), static_cast<unsigned>(m_tiles));
  auto go = [&](auto out, auto model) {
    hipLaunchKernelGGL((fp8_gemm_kernel<decltype(out)::value, decltype(model)::value>), grid, dim3(256), 0, s, a,
                       static_cast<int>(m_tiles));
  };
  auto by_model = [&](auto out) {
    if (a.model_dtype == MODEL_F32) go(out, std::integral_constant<int, MODEL_F32>{});
    else if (a.model_dtype == MODEL_BF16) go(out, std::integral_constant<int, MODEL_BF16>{});
    else go(out, std::integral_constant<int, MODEL_F16>{});
  };
  if (a.out_dtype == MODEL_F32) by_model(std::integral_constant<int, MODEL_F32>{});
  else if (a.out_dtype == MODEL_BF16) by_model(std::integral_constant<int, MODEL_BF16>{});
  else by_model(std::integral_constant<int, MODEL_F16>{});
  return hipGetLastError();
}

}  // namespace gq
