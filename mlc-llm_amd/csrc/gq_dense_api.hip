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

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool act_ok(int a) { return a >= MI355GQ_ACT_NONE && a <= MI355GQ_ACT_GELU_TANH; }
bool dim_ok(int64_t d) { return d >= 0 && d < kMaxDim; }

int hip_result(hipError_t e, const char* what) {
  return e == hipSuccess ? MI355GQ_OK : set_error(MI355GQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}
hipStream_t as_stream(mi355gq_stream_t s) { return static_cast<hipStream_t>(s); }

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
  return hip_result(gq::launch_dense_simple(a, as_stream(stream)), what);
}

}  // namespace

extern "C" {

int64_t mi355gq_dense_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated) {
  (void)gated;
  if (!dim_ok(M) || !dim_ok(N) || !dim_ok(K) || M == 0 || N == 0 || K == 0) return 0;
  return 0;
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

}  // extern "C"
