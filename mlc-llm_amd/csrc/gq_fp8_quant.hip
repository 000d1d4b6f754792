// e4m3 quantisers and the way back.  One read and one write of each number; bound by HBM.  Measured: 2048 x 14336 bfloat16 rows 15.1 us
// = 5.9 TB/s read and written (part of it stays in the last-level cache), 28672 x 4096 bfloat16 weights 71 us = 4.95 TB/s.
#include "gq_fp8_common.hpp"
#include "gq_topk.hpp"

namespace gq {

namespace {

// eight neighbouring numbers of a row, of which those past `cols` count as zero; ALIGNED: rows start at 16 bytes and cols is a multiple of 8
template <int DT, bool ALIGNED>
__device__ __forceinline__ void load8_row(const void* p, int64_t row0, int col, int cols, float (&f)[8]) {
  if constexpr (ALIGNED) {
    if (col < cols) {
      fp8_load8<DT>(p, row0 + col, f);
      return;
    }
#pragma unroll
    for (int v = 0; v < 8; ++v) f[v] = 0.f;
  } else {
#pragma unroll
    for (int v = 0; v < 8; ++v) f[v] = col + v < cols ? Elem<DT>::load(p, row0 + col + v) : 0.f;
  }
}

}  // namespace

// A launch of 2^32 or more work items loses all but the rest of that division, without an error: the row kernels, four rows a workgroup of 256,
// take this many at most.
constexpr int64_t kRowsALaunch = int64_t(1) << 25;

// A wave takes four groups of a row at a time: 16 lanes a group, eight numbers a lane, the group's maximum by four DPP steps.
template <int DT, bool SILU, bool ALIGNED>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const void* __restrict__ x, int64_t row0, int64_t rows, int cols,
                                                           uint8_t* __restrict__ q, int64_t q_pitch,
                                                           float* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t row = row0 + static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int col = blockIdx.y * 512 + lane * 8;
  float f[8];
  if constexpr (SILU) {
    float up[8];
    load8_row<DT, ALIGNED>(x, row * 2 * cols, col, cols, f);
    load8_row<DT, ALIGNED>(x, row * 2 * cols + cols, col, cols, up);
#pragma unroll
    for (int v = 0; v < 8; ++v) f[v] = silu_mul_f32(f[v], up[v]);
  } else {
    load8_row<DT, ALIGNED>(x, row * cols, col, cols, f);
  }
  uint32_t bits;
  const uint2 out = fp8_group(f, &bits);
  if (col >= cols) return;  // (what a row holds from the next multiple of 8 on may be somebody's)
  *reinterpret_cast<uint2*>(q + row * q_pitch + col) = out;
  if ((lane & 15) == 0) scale[static_cast<int64_t>(col / kFp8Block) * rows + row] = __builtin_bit_cast(float, bits);
}

hipError_t launch_fp8_quantize(const void* x, int64_t rows, int64_t cols, int model_dtype, bool silu_mul, uint8_t* q,
                               int64_t q_pitch, float* scale, hipStream_t s) {
  const bool aligned = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
  auto go = [&](auto dt, auto silu, auto al) {
    for (int64_t row0 = 0; row0 < rows; row0 += kRowsALaunch) {
      const int64_t here = rows - row0 < kRowsALaunch ? rows - row0 : kRowsALaunch;
      const dim3 grid(static_cast<unsigned>((here + 3) / 4), static_cast<unsigned>((cols + 511) / 512));
      hipLaunchKernelGGL((fp8_quantize_kernel<decltype(dt)::value, decltype(silu)::value, decltype(al)::value>), grid, dim3(256),
                         0, s, x, row0, rows, static_cast<int>(cols), q, q_pitch, scale);
    }
  };
  auto by_form = [&](auto dt) {
    if (silu_mul) {
      if (aligned) go(dt, std::true_type{}, std::true_type{});
      else go(dt, std::true_type{}, std::false_type{});
    } else {
      if (aligned) go(dt, std::false_type{}, std::true_type{});
      else go(dt, std::false_type{}, std::false_type{});
    }
  };
  if (model_dtype == MODEL_F32) by_form(std::integral_constant<int, MODEL_F32>{});
  else if (model_dtype == MODEL_BF16) by_form(std::integral_constant<int, MODEL_BF16>{});
  else by_form(std::integral_constant<int, MODEL_F16>{});
  return hipGetLastError();
}

// A workgroup a block of 128 x 128: 16 lanes a row of it, eight rows a thread, which stay in registers between the maximum
// and the conversion.
template <int DT, bool ALIGNED>
__global__ __launch_bounds__(256) void fp8_quantize_weight_kernel(const void* __restrict__ w, int N, int K, int n_blocks,
                                                                  uint8_t* __restrict__ q, int64_t q_pitch,
                                                                  float* __restrict__ scale) {
  __shared__ float tops[4];
  const int64_t mat = blockIdx.y / n_blocks;
  const int bn = blockIdx.y - static_cast<int>(mat) * n_blocks;
  const int col = blockIdx.x * kFp8Block + (threadIdx.x & 15) * 8, row0 = bn * kFp8Block + (threadIdx.x >> 4);
  float f[8][8];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + 16 * i;
    load8_row<DT, ALIGNED>(w, (mat * N + (row < N ? row : N - 1)) * K, col, K, f[i]);
#pragma unroll
    for (int v = 0; v < 8; ++v) top = fmaxf(top, fp8_magnitude(f[i][v]));
  }
  top = row_max16(top);
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const uint32_t bits = fp8_scale_bits(top);
  const float inv = fp8_inverse(bits);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + 16 * i;
    if (row < N && col < K) {
      uint2 out;
      out.x = fp8_quad(f[i][0] * inv, f[i][1] * inv, f[i][2] * inv, f[i][3] * inv);
      out.y = fp8_quad(f[i][4] * inv, f[i][5] * inv, f[i][6] * inv, f[i][7] * inv);
      *reinterpret_cast<uint2*>(q + (mat * N + row) * q_pitch + col) = out;
    }
  }
  if (threadIdx.x == 0) scale[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = __builtin_bit_cast(float, bits);
}

hipError_t launch_fp8_quantize_weight(const void* w, int64_t mats, int64_t N, int64_t K, int model_dtype, uint8_t* q,
                                      int64_t q_pitch, float* scale, hipStream_t s) {
  const bool aligned = K % 8 == 0 && (reinterpret_cast<uintptr_t>(w) & 15u) == 0;
  const int n_blocks = static_cast<int>((N + kFp8Block - 1) / kFp8Block);
  // blockIdx.y holds at most 65535 blocks: stacks with more go in parts
  const int64_t per = 65535 / n_blocks;
  const size_t size = model_dtype == MODEL_F32 ? 4 : 2;
  const int64_t k_blocks = (K + kFp8Block - 1) / kFp8Block;
  for (int64_t m0 = 0; m0 < mats; m0 += per) {
    const int64_t m = mats - m0 < per ? mats - m0 : per;
    const dim3 grid(static_cast<unsigned>(k_blocks), static_cast<unsigned>(m * n_blocks));
    auto go = [&](auto dt, auto al) {
      hipLaunchKernelGGL((fp8_quantize_weight_kernel<decltype(dt)::value, decltype(al)::value>), grid, dim3(256), 0, s,
                         static_cast<const char*>(w) + m0 * N * K * size, static_cast<int>(N), static_cast<int>(K), n_blocks,
                         q + m0 * N * q_pitch, q_pitch, scale + m0 * n_blocks * k_blocks);
    };
    auto by_form = [&](auto dt) {
      if (aligned) go(dt, std::true_type{});
      else go(dt, std::false_type{});
    };
    if (model_dtype == MODEL_F32) by_form(std::integral_constant<int, MODEL_F32>{});
    else if (model_dtype == MODEL_BF16) by_form(std::integral_constant<int, MODEL_BF16>{});
    else by_form(std::integral_constant<int, MODEL_F16>{});
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// q s in float32, rounded to the output type.  ROWS: scale [ceil(cols / 128), rows] (activations), else
// [mats, ceil(rows / 128), ceil(cols / 128)] (weights).
template <int DT, bool ROWS>
__global__ __launch_bounds__(256) void fp8_dequantize_kernel(const uint8_t* __restrict__ q, int64_t q_pitch,
                                                             const float* __restrict__ scale, int64_t row0, int64_t rows_all,
                                                             int64_t rows, int cols, void* __restrict__ out) {
  const int64_t row = row0 + static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int col = blockIdx.y * 512 + (threadIdx.x & 63) * 8;
  if (row >= rows_all || col >= cols) return;
  const int64_t mat = ROWS ? 0 : row / rows;
  const int groups = (cols + kFp8Block - 1) / kFp8Block;
  const float s = ROWS ? scale[static_cast<int64_t>(col / kFp8Block) * rows + row]
                       : scale[(mat * ((rows + kFp8Block - 1) / kFp8Block) + (row - mat * rows) / kFp8Block) * groups + col / kFp8Block];
  const uint2 b = *reinterpret_cast<const uint2*>(q + row * q_pitch + col);  // pitch is a multiple of 16: all eight are the row's own
  float f[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int u = static_cast<int>(h == 0 ? b.x : b.y);
    f[4 * h] = __builtin_amdgcn_cvt_f32_fp8(u, 0);
    f[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(u, 1);
    f[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(u, 2);
    f[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(u, 3);
  }
#pragma unroll
  for (int v = 0; v < 8; ++v)
    if (col + v < cols) Elem<DT>::store(out, row * cols + col + v, f[v] * s);
}

hipError_t launch_fp8_dequantize(const uint8_t* q, int64_t q_pitch, const float* scale, int64_t mats, int64_t rows,
                                 int64_t cols, bool row_groups, int out_dtype, void* out, hipStream_t s) {
  auto go = [&](auto dt, auto by_row) {
    for (int64_t row0 = 0; row0 < mats * rows; row0 += kRowsALaunch) {
      const int64_t here = mats * rows - row0 < kRowsALaunch ? mats * rows - row0 : kRowsALaunch;
      const dim3 grid(static_cast<unsigned>((here + 3) / 4), static_cast<unsigned>((cols + 511) / 512));
      hipLaunchKernelGGL((fp8_dequantize_kernel<decltype(dt)::value, decltype(by_row)::value>), grid, dim3(256), 0, s, q, q_pitch,
                         scale, row0, mats * rows, rows, static_cast<int>(cols), out);
    }
  };
  auto by_form = [&](auto dt) {
    if (row_groups) go(dt, std::true_type{});
    else go(dt, std::false_type{});
  };
  if (out_dtype == MODEL_F32) by_form(std::integral_constant<int, MODEL_F32>{});
  else if (out_dtype == MODEL_BF16) by_form(std::integral_constant<int, MODEL_BF16>{});
  else by_form(std::integral_constant<int, MODEL_F16>{});
  return hipGetLastError();
}

}  // namespace gq
