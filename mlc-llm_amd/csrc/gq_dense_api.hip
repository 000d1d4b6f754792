// C entry points of the operators on 16-bit weights: argument checks, workspaces, dispatch.  Declared, with what each computes, in
// include/mi355gq.h.
#include "../../include/mi355gq.h"
#include "gq_dense_common.hpp"

namespace {

using gq::set_error;

#define DENSE_REQUIRE(cond, ...) \
  do {                           \
    if (!(cond)) return set_error(MI355GQ_ERR_ARG, __VA_ARGS__); \
  } while (0)

constexpr int64_t kMaxDim = (int64_t(1) << 31) - 256;
// numbers of a row: 256 rows of a tile are to end below what is left of 2^32 bytes at any block of K
constexpr int64_t kMaxRow = (int64_t(1) << 23) - 128;

constexpr int64_t kMostRows = int64_t(1) << 20;  // in one launch

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool act_ok(int a) { return a >= MI355GQ_ACT_NONE && a <= MI355GQ_ACT_GELU_TANH; }
bool dim_ok(int64_t d) { return d >= 0 && d < kMaxDim; }

int hip_result(hipError_t e, const char* what) {
  return e == hipSuccess ? MI355GQ_OK : set_error(MI355GQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}
hipStream_t as_stream(mi355gq_stream_t s) { return static_cast<hipStream_t>(s); }

// Where the kernel that streams the weights past up to sixteen rows of x is faster than the tiles; N rows of W.  us, it / the tiles: 4096 x 4096 of 4
// rows 8.3 / 10.7, of 16 9.3 / 11.2; 6144 x 4096 of 8 rows 11.9 / 13.9, of 16 13.9 / 14.4; 11264 x 2048 of 8 rows 10.6 / 11.0, of 12 11.7 / 11.1; 5120 x 5120
// of 8 rows 14.3 / 13.6, of 12 16.0 / 13.9; 28672 x 4096 of 8 rows 37.5 / 37.9, of 12 39.4 / 38.2; 128256 x 4096 of 8 rows 157 / 154, of 16 186 / 160.
bool few_rows(int64_t M, int64_t N, int64_t K) { return gq::options().gemm_variant < 0 && (M <= 8 || (M <= 16 && N * K < 20000000)); }

// cols: of y
int product(const char* what, const void* x, const void* w, const void* bias, const void* residual, int64_t M, int64_t cols, int64_t K,
            bool gated, int activation, int model_dtype, int out_dtype, void* y, void* workspace, int64_t workspace_bytes, mi355gq_stream_t stream) {
  DENSE_REQUIRE(model_dtype == MI355GQ_F16 || model_dtype == MI355GQ_BF16, "%s: model_dtype=%d (MI355GQ_F16 or MI355GQ_BF16)", what, model_dtype);
  DENSE_REQUIRE(out_dtype == model_dtype || out_dtype == MI355GQ_F32, "%s: out_dtype=%d (model_dtype or MI355GQ_F32)", what, out_dtype);
  DENSE_REQUIRE(act_ok(activation), "%s: activation=%d", what, activation);
  DENSE_REQUIRE(dim_ok(M) && dim_ok(cols) && dim_ok(gated ? 2 * cols : cols) && K > 0 && dim_ok(K), "%s: bad shape M=%lld N=%lld K=%lld", what,
                (long long)M, (long long)cols, (long long)K);
  if (M == 0 || cols == 0) return MI355GQ_OK;
  if (K >= kMaxRow) return set_error(MI355GQ_ERR_UNSUPPORTED, "%s: K=%lld (below 2^23 - 128)", what, (long long)K);
  DENSE_REQUIRE(x && w && y, "%s: null pointer", what);
  DENSE_REQUIRE(aligned(x, 2) && aligned(w, 2) && aligned(bias, 2) && aligned(residual, 2) && aligned(y, out_dtype == MI355GQ_F32 ? 4 : 2),
                "%s: misaligned pointer", what);
  gq::DenseArgs a;
  a.x = static_cast<const uint16_t*>(x);
  a.w = static_cast<const uint16_t*>(w);
  a.bias = static_cast<const uint16_t*>(bias);
  a.residual = static_cast<const uint16_t*>(residual);
  a.y = y;
  a.rows = M;
  a.N = gated ? 2 * cols : cols;
  a.K = K;
  a.act = activation;
  a.gated = gated;
  a.bf16 = model_dtype == MI355GQ_BF16;
  a.out_f32 = out_dtype == MI355GQ_F32;
  a.vec = cols % 8 == 0 && aligned(y, 16) && aligned(bias, 16) && aligned(residual, 16);
  if (aligned(workspace, 16)) {
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
  }
  const hipStream_t s = as_stream(stream);
  const int64_t y_row = cols * (a.out_f32 ? 4 : 2);
  hipError_t e = hipSuccess;
  for (int64_t r = 0; r < M && e == hipSuccess; r += kMostRows) {  // (2^32 work items or more in a launch would wrap, without an error)
    a.rows = M - r < kMostRows ? M - r : kMostRows;
    e = hipErrorNotSupported;
    if (gq::dense_aligned(a)) {
      if (few_rows(a.rows, a.N, K)) e = gq::launch_dense_rows(a, s);
      if (e == hipErrorNotSupported) e = gq::launch_dense_tile(a, s);
    }
    if (e == hipErrorNotSupported) e = gq::launch_dense_simple(a, s);
    a.x += a.rows * K;
    if (a.residual != nullptr) a.residual += a.rows * cols;
    a.y = static_cast<char*>(a.y) + a.rows * y_row;
  }
  return hip_result(e, what);
}

bool moe_sizes_ok(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t top_k) {
  return T >= 0 && T < kMaxDim && hidden > 0 && hidden % 8 == 0 && hidden < kMaxRow && inter > 0 && inter % 8 == 0 && inter < kMaxRow && experts > 0 &&
         experts <= 512 && top_k > 0 && top_k <= 32 && top_k <= experts;
}
// (work items are counted in 32 bits)
bool moe_takes(int64_t T, int64_t inter, int64_t top_k) { return T <= gq::kMoeTokens && T * top_k * inter * 2 < 0xc0000000ll; }

}  // namespace

extern "C" {

int64_t mi355gq_dense_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated) {
  const int64_t rows_of_w = gated ? 2 * N : N;
  if (!dim_ok(M) || !dim_ok(N) || !dim_ok(rows_of_w) || !dim_ok(K) || M == 0 || N == 0 || K == 0 || few_rows(M, rows_of_w, K) || K % 8 != 0) return 0;
  return gq::dense_tile_workspace_bytes(M < kMostRows ? M : kMostRows, rows_of_w, K);
}

int mi355gq_dense_linear(const void* x, const void* w, const void* bias, const void* residual, int64_t M, int64_t N, int64_t K, int activation,
                         int model_dtype, int out_dtype, void* y, void* workspace, int64_t workspace_bytes, mi355gq_stream_t stream) {
  return product("dense_linear", x, w, bias, residual, M, N, K, false, activation, model_dtype, out_dtype, y, workspace, workspace_bytes, stream);
}

int mi355gq_dense_linear_gated(const void* x, const void* w, const void* bias, int64_t M, int64_t inter, int64_t K, int activation, int model_dtype,
                               int out_dtype, void* y, void* workspace, int64_t workspace_bytes, mi355gq_stream_t stream) {
  return product("dense_linear_gated", x, w, bias, nullptr, M, inter, K, true, activation, model_dtype, out_dtype, y, workspace, workspace_bytes,
                 stream);
}

int64_t mi355gq_dense_moe_workspace_bytes(int64_t T, int64_t hidden, int64_t inter, int64_t num_experts, int64_t top_k) {
  if (!moe_sizes_ok(T, hidden, inter, num_experts, top_k) || T == 0 || !moe_takes(T, inter, top_k)) return 0;
  return gq::dense_moe_workspace_bytes(T, hidden, inter, num_experts, top_k);
}

int mi355gq_dense_moe(const void* x, const void* logits, const void* score_bias, int64_t T, int64_t hidden, int64_t inter, int64_t num_experts,
                      int64_t top_k, int scoring, int64_t num_groups, int64_t top_groups, int renormalize, float scale, int logits_dtype,
                      const void* w13, const void* w2, int activation, int model_dtype, void* out, void* workspace, int64_t workspace_bytes,
                      mi355gq_stream_t stream) {
  DENSE_REQUIRE(model_dtype == MI355GQ_F16 || model_dtype == MI355GQ_BF16, "dense_moe: model_dtype=%d (MI355GQ_F16 or MI355GQ_BF16)", model_dtype);
  DENSE_REQUIRE(logits_dtype == MI355GQ_F16 || logits_dtype == MI355GQ_F32 || logits_dtype == MI355GQ_BF16, "dense_moe: logits_dtype=%d", logits_dtype);
  DENSE_REQUIRE(act_ok(activation), "dense_moe: activation=%d", activation);
  DENSE_REQUIRE(scoring == MI355GQ_SCORE_SOFTMAX || scoring == MI355GQ_SCORE_SIGMOID, "dense_moe: scoring=%d", scoring);
  DENSE_REQUIRE(moe_sizes_ok(T, hidden, inter, num_experts, top_k),
                "dense_moe: T=%lld, hidden=%lld and inter=%lld (multiples of 8 below 2^23 - 128), num_experts=%lld (1..512), top_k=%lld (1..32)", (long long)T,
                (long long)hidden, (long long)inter, (long long)num_experts, (long long)top_k);
  DENSE_REQUIRE(num_groups > 0 && num_groups <= 64 && num_experts % num_groups == 0 && top_groups > 0 && top_groups <= num_groups &&
                    top_groups * (num_experts / num_groups) >= top_k,
                "dense_moe: the %lld best of %lld groups of %lld experts cannot give %lld", (long long)top_groups, (long long)num_groups,
                (long long)num_experts, (long long)top_k);
  if (T == 0) return MI355GQ_OK;
  if (!moe_takes(T, inter, top_k))
    return set_error(MI355GQ_ERR_UNSUPPORTED, "dense_moe: %lld tokens of %lld experts of %lld (%d tokens at most, and 3 GiB of activations in 16 bits)", (long long)T,
                     (long long)top_k, (long long)inter, gq::kMoeTokens);
  DENSE_REQUIRE(x && logits && w13 && w2 && out, "dense_moe: null pointer");
  DENSE_REQUIRE(aligned(x, 16) && aligned(w13, 16) && aligned(w2, 16) && aligned(out, 16) && aligned(score_bias, 4) &&
                    aligned(logits, logits_dtype == MI355GQ_F32 ? 4 : 2), "dense_moe: misaligned pointer (x, out and weights: 16 bytes)");
  DENSE_REQUIRE(aligned(workspace, 16), "dense_moe: workspace must be 16-byte aligned");
  const int64_t need = gq::dense_moe_workspace_bytes(T, hidden, inter, num_experts, top_k);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(MI355GQ_ERR_WORKSPACE, "dense_moe: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  gq::DenseMoeArgs a;
  a.x = static_cast<const uint16_t*>(x);
  a.w13 = static_cast<const uint16_t*>(w13);
  a.w2 = static_cast<const uint16_t*>(w2);
  a.out = static_cast<uint16_t*>(out);
  a.logits = logits;
  a.score_bias = static_cast<const float*>(score_bias);
  a.T = static_cast<int>(T);
  a.experts = static_cast<int>(num_experts);
  a.k = static_cast<int>(top_k);
  a.hidden = static_cast<int>(hidden);
  a.inter = static_cast<int>(inter);
  a.act = activation;
  a.bf16 = model_dtype == MI355GQ_BF16;
  a.sigmoid = scoring == MI355GQ_SCORE_SIGMOID;
  a.groups = static_cast<int>(num_groups);
  a.top_groups = static_cast<int>(top_groups);
  a.renormalize = renormalize != 0;
  a.logits_dtype = logits_dtype;
  a.scale = scale;
  a.workspace = workspace;
  return hip_result(gq::launch_dense_moe(a, as_stream(stream)), "dense_moe launch");
}

}  // extern "C"
