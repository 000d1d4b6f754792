// C entry points of the 8-bit block-scaled operators: argument checks, workspaces, dispatch.  Declared, with what each
// computes, in include/mi355gq.h.
#include "../../include/mi355gq.h"
#include "gq_fp8_common.hpp"

namespace {

using gq::set_error;

#define FP8_REQUIRE(cond, ...) \
  do {                         \
    if (!(cond)) return set_error(MI355GQ_ERR_ARG, __VA_ARGS__); \
  } while (0)

constexpr int64_t kMaxDim = (int64_t(1) << 31) - 256;
constexpr int64_t kMaxTiles = 65535;
constexpr int64_t kMaxSlots = kMaxDim - 2048;  // (moe_plan_kernel's waves count up to 1342 past the last slot, in 32 bits)

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool dtype_ok(int d) { return d == MI355GQ_F16 || d == MI355GQ_F32 || d == MI355GQ_BF16; }
int64_t dtype_bytes(int d) { return d == MI355GQ_F32 ? 4 : 2; }
bool dtype_aligned(const void* p, int d) { return (reinterpret_cast<uintptr_t>(p) & (dtype_bytes(d) - 1)) == 0; }
bool dim_ok(int64_t d) { return d >= 0 && d < kMaxDim; }
bool pitch_ok(int64_t pitch, int64_t k) { return pitch % 16 == 0 && pitch >= k && pitch < kMaxDim; }
// rows of an operand of a product: 256 of them are to end below what is left of 2^32 at any block of K
constexpr int64_t kMaxRow = (int64_t(1) << 24) - 256;
bool rows_ok(int64_t pitch) { return pitch < kMaxRow; }
int64_t groups_of(int64_t k) { return (k + gq::kFp8Block - 1) / gq::kFp8Block; }
int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }

int hip_result(hipError_t e, const char* what) {
  return e == hipSuccess ? MI355GQ_OK : set_error(MI355GQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}
hipStream_t as_stream(mi355gq_stream_t s) { return static_cast<hipStream_t>(s); }

// the pieces of a caller's workspace, each at a multiple of 256 bytes
struct Carver {
  char* base;
  int64_t used = 0;
  template <class T>
  T* take(int64_t count) {
    T* p = reinterpret_cast<T*>(base + used);
    used += (count * static_cast<int64_t>(sizeof(T)) + 255) / 256 * 256;
    return p;
  }
};

int quantize(const void* x, int64_t rows, int64_t K, int model_dtype, bool silu, void* q, int64_t q_pitch, void* scale,
             mi355gq_stream_t stream, const char* what) {
  FP8_REQUIRE(dtype_ok(model_dtype), "%s: model_dtype=%d (MI355GQ_F16, MI355GQ_F32 or MI355GQ_BF16)", what, model_dtype);
  FP8_REQUIRE(dim_ok(rows) && dim_ok(K) && (K + 511) / 512 <= kMaxTiles, "%s: bad shape [%lld, %lld]", what, (long long)rows, (long long)K);
  FP8_REQUIRE(pitch_ok(q_pitch, K), "%s: q_pitch=%lld for K=%lld: a multiple of 16, at least K", what, (long long)q_pitch, (long long)K);
  if (rows == 0 || K == 0) return MI355GQ_OK;
  FP8_REQUIRE(x && q && scale, "%s: null pointer", what);
  FP8_REQUIRE(dtype_aligned(x, model_dtype) && aligned16(q) && aligned4(scale), "%s: misaligned pointer (q: 16 bytes)", what);
  return hip_result(gq::launch_fp8_quantize(x, rows, K, model_dtype, silu, static_cast<uint8_t*>(q), q_pitch,
                                            static_cast<float*>(scale), as_stream(stream)), what);
}

// the few-row kernel's view of a product on quantised x
gq::Fp8RowsArgs few_rows(const gq::Fp8Args& a) {
  gq::Fp8RowsArgs r;
  r.x = a.x;
  r.xs = a.xs;
  r.x_pitch = a.x_pitch;
  r.x_rows = a.x_rows;
  r.w = a.w;
  r.ws = a.ws;
  r.w_pitch = a.w_pitch;
  r.N = a.N;
  r.K = a.K;
  r.experts = a.experts;
  r.bias = a.bias;
  r.residual = a.residual;
  r.y = a.y;
  r.rows = a.rows;
  r.indptr = a.indptr;
  r.x_row_index = a.x_row_index;
  r.model_dtype = a.model_dtype;
  r.out_dtype = a.out_dtype;
  r.y_aligned = aligned16(a.y);
  return r;
}

// Where the kernel that streams the weights past up to sixteen rows of x is faster than the tiles.  Each of its workgroups brings all
// of x to LDS: 0.4 us a row of 2048, 2 us a row of 14336.  In a graph, against the tiles with the quantiser that they need: 4096 x 4096
// of 8 rows 12.1 / 14.6 us, of 12 13.8 / 14.4, of 16 16.2 / 15.1; 10240 x 8192 of 4 rows 26.4 / 25.6, of 6 28.6 / 25.7; 4096 x 14336
// of 2 18.9 / 23.6, of 6 27.0 / 23.9.  With segments, rows of one on average: expert layers of 128 x 2048 x 768 at 4 rows 128 / 139 us, at
// 8 138 / 143, at 10 159 / 145; of 8 x 4096 x 14336 at 5 rows 289 / 292, at 10 314 / 305.
bool few_rows_dense(int64_t rows, int64_t K) { return rows == 1 || (rows <= 12 && rows * K < 49152); }
constexpr int64_t kFewRowsEach = 8;

hipError_t product(const gq::Fp8Args& a, hipStream_t s) {
  const int64_t segments = a.indptr ? (a.rows < a.experts ? a.rows : a.experts) : 1;
  if (a.indptr ? a.rows <= kFewRowsEach * segments : few_rows_dense(a.rows, a.K)) {
    hipError_t e = a.rows == 1 && !a.indptr ? gq::launch_fp8_gemv(few_rows(a), s) : hipErrorNotSupported;
    if (e == hipErrorNotSupported) e = gq::launch_fp8_rows(few_rows(a), s);
    if (e != hipErrorNotSupported) return e;
  }
  return gq::launch_fp8_tile(a, s);
}

struct LinearWorkspace {
  uint8_t* q = nullptr;
  float* scale = nullptr;
  void* split = nullptr;  // sums of shares of K
  int64_t split_bytes = 0, bytes = 0;
};
LinearWorkspace linear_workspace(int64_t M, int64_t N, int64_t K, bool x_quantized, void* base) {
  LinearWorkspace w;
  Carver c{static_cast<char*>(base)};
  if (!x_quantized) {
    w.q = c.take<uint8_t>(M * up16(K));
    w.scale = c.take<float>(M * groups_of(K));
  }
  w.split_bytes = !few_rows_dense(M, K) || K % 16 != 0 ? gq::fp8_tile_workspace_bytes(M, N, K) : 0;
  w.split = c.take<char>(w.split_bytes);
  w.bytes = c.used;
  return w;
}

struct MoeWorkspace {
  uint8_t *xq, *hq;
  float *xs, *hs, *both;
  int32_t *row_token, *slot_row, *indptr;
  float* y;
  int64_t bytes;
};
// `both`, gate and up in float32, is the largest piece by far: it is there only where no kernel quantises the activation as it comes up
// (one token's is small; its first product leaves silu(gate) * up there).
MoeWorkspace moe_workspace(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t top_k, int64_t w13_pitch, void* base) {
  const int64_t slots = T * top_k;
  Carver c{static_cast<char*>(base)};
  MoeWorkspace w;
  w.xq = c.take<uint8_t>(T * hidden);
  w.xs = c.take<float>(T * groups_of(hidden));
  w.row_token = c.take<int32_t>(slots);
  w.slot_row = c.take<int32_t>(slots);
  w.indptr = c.take<int32_t>(experts + 1);
  w.both = c.take<float>(T == 1 || !gq::fp8_silu_takes(2 * inter, w13_pitch) ? slots * 2 * inter : 0);
  w.hq = c.take<uint8_t>(slots * inter);
  w.hs = c.take<float>(slots * groups_of(inter));
  w.y = c.take<float>(slots * hidden);
  w.bytes = c.used;
  return w;
}

}  // namespace

extern "C" {

int mi355gq_fp8_quantize(const void* x, int64_t rows, int64_t K, int model_dtype, void* q, int64_t q_pitch, void* scale,
                         mi355gq_stream_t stream) {
  return quantize(x, rows, K, model_dtype, false, q, q_pitch, scale, stream, "fp8_quantize");
}

int mi355gq_fp8_silu_mul_quantize(const void* x, int64_t rows, int64_t K, int model_dtype, void* q, int64_t q_pitch,
                                  void* scale, mi355gq_stream_t stream) {
  return quantize(x, rows, K, model_dtype, true, q, q_pitch, scale, stream, "fp8_silu_mul_quantize");
}

int mi355gq_fp8_quantize_weight(const void* w, int64_t mats, int64_t N, int64_t K, int model_dtype, void* q, int64_t q_pitch,
                                void* scale, mi355gq_stream_t stream) {
  FP8_REQUIRE(dtype_ok(model_dtype), "fp8_quantize_weight: model_dtype=%d", model_dtype);
  FP8_REQUIRE(dim_ok(mats) && dim_ok(N) && dim_ok(K) && groups_of(N) <= kMaxTiles, "fp8_quantize_weight: bad shape [%lld, %lld, %lld]",
              (long long)mats, (long long)N, (long long)K);
  FP8_REQUIRE(pitch_ok(q_pitch, K), "fp8_quantize_weight: q_pitch=%lld for K=%lld: a multiple of 16, at least K", (long long)q_pitch,
              (long long)K);
  if (mats == 0 || N == 0 || K == 0) return MI355GQ_OK;
  FP8_REQUIRE(w && q && scale, "fp8_quantize_weight: null pointer");
  FP8_REQUIRE(dtype_aligned(w, model_dtype) && aligned16(q) && aligned4(scale), "fp8_quantize_weight: misaligned pointer (q: 16 bytes)");
  return hip_result(gq::launch_fp8_quantize_weight(w, mats, N, K, model_dtype, static_cast<uint8_t*>(q), q_pitch,
                                                   static_cast<float*>(scale), as_stream(stream)), "fp8_quantize_weight launch");
}

int mi355gq_fp8_dequantize(const void* q, int64_t q_pitch, const void* scale, int64_t mats, int64_t rows, int64_t K,
                           int row_groups, int out_dtype, void* out, mi355gq_stream_t stream) {
  FP8_REQUIRE(dtype_ok(out_dtype), "fp8_dequantize: out_dtype=%d", out_dtype);
  FP8_REQUIRE(row_groups == 0 || (row_groups == 1 && mats == 1), "fp8_dequantize: row_groups=%d with %lld matrices", row_groups,
              (long long)mats);
  FP8_REQUIRE(dim_ok(mats) && dim_ok(rows) && dim_ok(K) && (K + 511) / 512 <= kMaxTiles && (rows == 0 || mats < kMaxDim / rows), "fp8_dequantize: bad shape [%lld, %lld, %lld]",
              (long long)mats, (long long)rows, (long long)K);
  FP8_REQUIRE(pitch_ok(q_pitch, K), "fp8_dequantize: q_pitch=%lld for K=%lld: a multiple of 16, at least K", (long long)q_pitch, (long long)K);
  if (mats == 0 || rows == 0 || K == 0) return MI355GQ_OK;
  FP8_REQUIRE(q && scale && out, "fp8_dequantize: null pointer");
  FP8_REQUIRE(aligned16(q) && aligned4(scale) && dtype_aligned(out, out_dtype), "fp8_dequantize: misaligned pointer (q: 16 bytes)");
  return hip_result(gq::launch_fp8_dequantize(static_cast<const uint8_t*>(q), q_pitch, static_cast<const float*>(scale), mats,
                                              rows, K, row_groups == 1, out_dtype, out, as_stream(stream)), "fp8_dequantize launch");
}

int64_t mi355gq_fp8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int x_quantized) {
  if (!dim_ok(M) || !dim_ok(N) || !dim_ok(K) || M == 0 || N == 0 || K == 0) return 0;
  return linear_workspace(M, N, K, x_quantized != 0, nullptr).bytes;
}

int mi355gq_fp8_linear(const void* x, int64_t x_pitch, const void* x_scale, const void* w, int64_t w_pitch,
                       const void* w_scale, const void* bias, const void* residual, int64_t M, int64_t N, int64_t K,
                       int model_dtype, int out_dtype, int precise, void* y, void* workspace, int64_t workspace_bytes,
                       mi355gq_stream_t stream) {
  FP8_REQUIRE(dtype_ok(model_dtype) && dtype_ok(out_dtype), "fp8_linear: model_dtype=%d, out_dtype=%d", model_dtype, out_dtype);
  FP8_REQUIRE(dim_ok(M) && dim_ok(N) && dim_ok(K) && K > 0, "fp8_linear: bad shape M=%lld N=%lld K=%lld", (long long)M, (long long)N,
              (long long)K);
  FP8_REQUIRE((M + 63) / 64 <= kMaxTiles, "fp8_linear: M=%lld rows in one call", (long long)M);
  FP8_REQUIRE(pitch_ok(w_pitch, K) && (!x_scale || pitch_ok(x_pitch, K)),
              "fp8_linear: x_pitch=%lld, w_pitch=%lld for K=%lld: multiples of 16, at least K", (long long)x_pitch, (long long)w_pitch,
              (long long)K);
  if (M == 0 || N == 0) return MI355GQ_OK;
  if (!rows_ok(w_pitch) || (x_scale && !rows_ok(x_pitch)) || K >= kMaxRow)
    return set_error(MI355GQ_ERR_UNSUPPORTED, "fp8_linear: rows of %lld bytes (below 2^24)", (long long)(w_pitch > x_pitch ? w_pitch : x_pitch));
  FP8_REQUIRE(x && w && w_scale && y, "fp8_linear: null pointer");
  FP8_REQUIRE(aligned16(w) && aligned4(w_scale) && aligned4(x_scale) && (x_scale ? aligned16(x) : dtype_aligned(x, model_dtype)) &&
                  dtype_aligned(bias, model_dtype) && dtype_aligned(residual, model_dtype) && dtype_aligned(y, out_dtype),
              "fp8_linear: misaligned pointer (e4m3 tensors: 16 bytes)");
  const LinearWorkspace ws = linear_workspace(M, N, K, x_scale != nullptr, workspace);
  if (ws.bytes > 0) {
    FP8_REQUIRE(workspace == nullptr || aligned16(workspace), "fp8_linear: workspace must be 16-byte aligned");
    if (workspace == nullptr || workspace_bytes < ws.bytes)
      return set_error(MI355GQ_ERR_WORKSPACE, "fp8_linear: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)ws.bytes);
  }
  gq::Fp8Args a;
  a.w = static_cast<const uint8_t*>(w);
  a.ws = static_cast<const float*>(w_scale);
  a.w_pitch = w_pitch;
  a.bias = bias;
  a.residual = residual;
  a.y = y;
  a.rows = a.x_rows = M;
  a.N = N;
  a.K = K;
  a.model_dtype = model_dtype;
  a.out_dtype = out_dtype;
  a.precise = precise != 0;
  a.workspace = ws.split;
  a.workspace_bytes = ws.split_bytes;
  if (x_scale == nullptr && few_rows_dense(M, K) && aligned16(x)) {  // the kernel quantises x itself
    gq::Fp8RowsArgs r = few_rows(a);
    r.x = x;
    r.x_kind = model_dtype;
    hipError_t e = M == 1 ? gq::launch_fp8_gemv(r, as_stream(stream)) : hipErrorNotSupported;
    if (e == hipErrorNotSupported) e = gq::launch_fp8_rows(r, as_stream(stream));
    if (e != hipErrorNotSupported) return hip_result(e, "fp8_linear launch");
  }
  if (x_scale == nullptr) {
    const hipError_t e = gq::launch_fp8_quantize(x, M, K, model_dtype, false, ws.q, up16(K), ws.scale, as_stream(stream));
    if (e != hipSuccess) return hip_result(e, "fp8_linear: quantize launch");
    a.x = ws.q;
    a.xs = ws.scale;
    a.x_pitch = up16(K);
  } else {
    a.x = static_cast<const uint8_t*>(x);
    a.xs = static_cast<const float*>(x_scale);
    a.x_pitch = x_pitch;
  }
  return hip_result(product(a, as_stream(stream)), "fp8_linear launch");
}

int mi355gq_fp8_group_gemm(const void* x, int64_t x_pitch, const void* x_scale, int64_t x_rows, const void* x_row_index,
                           int64_t rows, const void* w, int64_t w_pitch, const void* w_scale, const void* indptr,
                           int64_t num_experts, int64_t N, int64_t K, int out_dtype, int precise, void* y,
                           mi355gq_stream_t stream) {
  FP8_REQUIRE(dtype_ok(out_dtype), "fp8_group_gemm: out_dtype=%d", out_dtype);
  FP8_REQUIRE(dim_ok(rows) && dim_ok(x_rows) && dim_ok(N) && dim_ok(K) && K > 0 && num_experts > 0 && num_experts <= 512,
              "fp8_group_gemm: bad shape rows=%lld experts=%lld N=%lld K=%lld", (long long)rows, (long long)num_experts, (long long)N, (long long)K);
  FP8_REQUIRE(rows / 64 + num_experts <= kMaxTiles, "fp8_group_gemm: %lld rows in one call", (long long)rows);
  FP8_REQUIRE(pitch_ok(x_pitch, K) && pitch_ok(w_pitch, K), "fp8_group_gemm: x_pitch=%lld, w_pitch=%lld for K=%lld: multiples of 16, at least K",
              (long long)x_pitch, (long long)w_pitch, (long long)K);
  if (rows == 0 || N == 0) return MI355GQ_OK;
  if (!rows_ok(w_pitch) || !rows_ok(x_pitch))
    return set_error(MI355GQ_ERR_UNSUPPORTED, "fp8_group_gemm: rows of %lld bytes (below 2^24)", (long long)(w_pitch > x_pitch ? w_pitch : x_pitch));
  FP8_REQUIRE(x_row_index || x_rows == rows, "fp8_group_gemm: %lld rows of x for %lld rows without an index", (long long)x_rows, (long long)rows);
  FP8_REQUIRE(x_rows > 0 && x && x_scale && w && w_scale && indptr && y, "fp8_group_gemm: null pointer");
  FP8_REQUIRE(aligned16(x) && aligned16(w) && aligned4(x_scale) && aligned4(w_scale) && aligned4(indptr) && aligned4(x_row_index) &&
                  dtype_aligned(y, out_dtype), "fp8_group_gemm: misaligned pointer (e4m3 tensors: 16 bytes)");
  if (x_row_index != nullptr && x_rows >= (int64_t(1) << 32) / x_pitch)
    return set_error(MI355GQ_ERR_UNSUPPORTED, "fp8_group_gemm: x of %lld rows of %lld bytes with a row index (4 GiB at most)", (long long)x_rows,
                     (long long)x_pitch);
  gq::Fp8Args a;
  a.x = static_cast<const uint8_t*>(x);
  a.xs = static_cast<const float*>(x_scale);
  a.x_pitch = x_pitch;
  a.x_rows = x_rows;
  a.x_row_index = static_cast<const int32_t*>(x_row_index);
  a.w = static_cast<const uint8_t*>(w);
  a.ws = static_cast<const float*>(w_scale);
  a.w_pitch = w_pitch;
  a.indptr = static_cast<const int32_t*>(indptr);
  a.experts = num_experts;
  a.y = y;
  a.rows = rows;
  a.N = N;
  a.K = K;
  a.out_dtype = out_dtype;
  a.precise = precise != 0;
  return hip_result(product(a, as_stream(stream)), "fp8_group_gemm launch");
}

int mi355gq_moe_gating(const void* logits, const void* bias, int64_t T, int64_t num_experts, int64_t top_k, int scoring,
                       int64_t num_groups, int64_t top_groups, int renormalize, float scale, int model_dtype, void* weights,
                       void* ids, mi355gq_stream_t stream) {
  FP8_REQUIRE(dtype_ok(model_dtype), "moe_gating: model_dtype=%d", model_dtype);
  FP8_REQUIRE(scoring == MI355GQ_SCORE_SOFTMAX || scoring == MI355GQ_SCORE_SIGMOID, "moe_gating: scoring=%d", scoring);
  FP8_REQUIRE(T >= 0 && T < kMaxDim && num_experts > 0 && num_experts <= 512 && top_k > 0 && top_k <= 32 && top_k <= num_experts,
              "moe_gating: T=%lld, num_experts=%lld (1..512), top_k=%lld (1..32)", (long long)T, (long long)num_experts, (long long)top_k);
  FP8_REQUIRE(num_groups > 0 && num_groups <= 64 && num_experts % num_groups == 0 && top_groups > 0 && top_groups <= num_groups &&
                  top_groups * (num_experts / num_groups) >= top_k,
              "moe_gating: the %lld best of %lld groups of %lld experts cannot give %lld", (long long)top_groups, (long long)num_groups,
              (long long)num_experts, (long long)top_k);
  if (T == 0) return MI355GQ_OK;
  FP8_REQUIRE(logits && weights && ids, "moe_gating: null pointer");
  FP8_REQUIRE(dtype_aligned(logits, model_dtype) && aligned4(bias) && aligned4(weights) && aligned4(ids), "moe_gating: misaligned pointer");
  gq::GatingArgs a{logits, static_cast<const float*>(bias), T, static_cast<int>(num_experts), static_cast<int>(top_k),
                   scoring == MI355GQ_SCORE_SIGMOID, static_cast<int>(num_groups), static_cast<int>(top_groups), renormalize != 0,
                   model_dtype, scale, static_cast<float*>(weights), static_cast<int32_t*>(ids)};
  return hip_result(gq::launch_moe_gating(a, as_stream(stream)), "moe_gating launch");
}

int mi355gq_moe_plan(const void* ids, int64_t T, int64_t top_k, int64_t num_experts, void* row_token, void* slot_row, void* indptr,
                     mi355gq_stream_t stream) {
  FP8_REQUIRE(dim_ok(T) && top_k > 0 && top_k <= 512 && T <= kMaxSlots / top_k && num_experts > 0 && num_experts <= 512,
              "moe_plan: T=%lld, top_k=%lld, num_experts=%lld (1..512)", (long long)T, (long long)top_k, (long long)num_experts);
  FP8_REQUIRE(indptr && (T == 0 || (ids && row_token && slot_row)), "moe_plan: null pointer");
  FP8_REQUIRE(aligned4(ids) && aligned4(row_token) && aligned4(slot_row) && aligned4(indptr), "moe_plan: misaligned pointer");
  return hip_result(gq::launch_moe_plan(static_cast<const int32_t*>(ids), T * top_k, static_cast<int>(top_k), static_cast<int>(num_experts),
                                        static_cast<int32_t*>(row_token), static_cast<int32_t*>(slot_row), static_cast<int32_t*>(indptr),
                                        as_stream(stream)), "moe_plan launch");
}

static bool moe_sizes_ok(int64_t T, int64_t hidden, int64_t inter, int64_t experts, int64_t top_k) {
  return dim_ok(T) && T * hidden < (int64_t(1) << 32) && hidden > 0 && hidden % 16 == 0 && hidden < kMaxRow && inter > 0 && inter % 16 == 0 && inter < kMaxRow &&
         experts > 0 && experts <= 512 && top_k > 0 && top_k <= 32 && T * top_k / 64 + experts <= kMaxTiles;
}

int64_t mi355gq_fp8_moe_workspace_bytes(int64_t T, int64_t hidden, int64_t inter, int64_t num_experts, int64_t top_k) {
  if (!moe_sizes_ok(T, hidden, inter, num_experts, top_k) || T == 0) return 0;
  return moe_workspace(T, hidden, inter, num_experts, top_k, hidden, nullptr).bytes;
}

int mi355gq_fp8_moe(const void* x, int64_t T, int64_t hidden, int64_t inter, int64_t num_experts, int64_t top_k, const void* weights,
                    const void* ids, const void* w13, int64_t w13_pitch, const void* w13_scale, const void* w2, int64_t w2_pitch,
                    const void* w2_scale, int model_dtype, void* out, void* workspace, int64_t workspace_bytes,
                    mi355gq_stream_t stream) {
  FP8_REQUIRE(model_dtype == MI355GQ_F16 || model_dtype == MI355GQ_BF16, "fp8_moe: model_dtype=%d (MI355GQ_F16 or MI355GQ_BF16)", model_dtype);
  FP8_REQUIRE(moe_sizes_ok(T, hidden, inter, num_experts, top_k),
              "fp8_moe: T=%lld, hidden=%lld and inter=%lld (multiples of 16), num_experts=%lld (1..512), top_k=%lld (1..32)", (long long)T,
              (long long)hidden, (long long)inter, (long long)num_experts, (long long)top_k);
  FP8_REQUIRE(pitch_ok(w13_pitch, hidden) && pitch_ok(w2_pitch, inter) && rows_ok(w13_pitch) && rows_ok(w2_pitch), "fp8_moe: w13_pitch=%lld, w2_pitch=%lld: multiples of 16, at least a row",
              (long long)w13_pitch, (long long)w2_pitch);
  if (T == 0) return MI355GQ_OK;
  FP8_REQUIRE(x && weights && ids && w13 && w13_scale && w2 && w2_scale && out, "fp8_moe: null pointer");
  FP8_REQUIRE(aligned16(x) && aligned16(out) && aligned16(w13) && aligned16(w2) && aligned4(weights) && aligned4(ids) && aligned4(w13_scale) &&
                  aligned4(w2_scale), "fp8_moe: misaligned pointer (x, out and e4m3 tensors: 16 bytes)");
  const MoeWorkspace ws = moe_workspace(T, hidden, inter, num_experts, top_k, w13_pitch, workspace);
  FP8_REQUIRE(workspace == nullptr || aligned16(workspace), "fp8_moe: workspace must be 16-byte aligned");
  if (workspace == nullptr || workspace_bytes < ws.bytes)
    return set_error(MI355GQ_ERR_WORKSPACE, "fp8_moe: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)ws.bytes);
  const hipStream_t s = as_stream(stream);
  const int64_t slots = T * top_k;
  const int64_t segments = slots < num_experts ? slots : num_experts;
  hipError_t e;
  // One token: its slots are the segments, x and the activation are quantised where they are read.  Only where both products go this way: the
  // second one's refusal behind the first would have gate and up computed again (4096 x 14336, two of eight experts: 113 us, 81 without that).
  if (T == 1 && gq::fp8_gemv_takes(2 * inter, hidden, w13_pitch) && gq::fp8_gemv_takes(hidden, inter, w2_pitch)) {
    gq::Fp8RowsArgs r;
    r.x = x;
    r.x_rows = T;
    r.x_kind = model_dtype;
    r.w = static_cast<const uint8_t*>(w13);
    r.ws = static_cast<const float*>(w13_scale);
    r.w_pitch = w13_pitch;
    r.N = 2 * inter;
    r.K = hidden;
    r.experts = num_experts;
    r.y = ws.both;
    r.rows = slots;
    r.ids = static_cast<const int32_t*>(ids);
    r.x_div = static_cast<int>(top_k);
    r.silu = 1;
    r.out_dtype = MI355GQ_F32;
    r.y_aligned = 1;
    e = gq::launch_fp8_gemv(r, s);
    if (e == hipSuccess) {
      r.x = ws.both;
      r.x_rows = slots;
      r.x_kind = MI355GQ_F32;
      r.w = static_cast<const uint8_t*>(w2);
      r.ws = static_cast<const float*>(w2_scale);
      r.w_pitch = w2_pitch;
      r.N = hidden;
      r.K = inter;
      r.y = out;
      r.x_div = 1;
      r.silu = 0;
      r.out_dtype = model_dtype;
      e = gq::launch_fp8_gemv_sum(r, static_cast<const float*>(weights), static_cast<int>(top_k), s);
    }
    return hip_result(e, "fp8_moe launch");
  }
  e = gq::launch_moe_plan_quantize(static_cast<const int32_t*>(ids), slots, static_cast<int>(top_k), static_cast<int>(num_experts),
                                   ws.row_token, ws.slot_row, ws.indptr, x, T, hidden, model_dtype, ws.xq, ws.xs, s);
  gq::Fp8Args a;
  a.x = ws.xq;
  a.xs = ws.xs;
  a.x_pitch = hidden;
  a.x_rows = T;
  a.x_row_index = ws.row_token;
  a.w = static_cast<const uint8_t*>(w13);
  a.ws = static_cast<const float*>(w13_scale);
  a.w_pitch = w13_pitch;
  a.indptr = ws.indptr;
  a.experts = num_experts;
  a.rows = slots;
  a.N = 2 * inter;
  a.K = hidden;
  a.y = ws.both;
  a.out_dtype = MI355GQ_F32;
  a.precise = true;  // sums that are rounded to e4m3 again: an error of 2e-5 would move one in thousands by a sixteenth
  const bool by_rows = slots <= kFewRowsEach * segments;
  if (e == hipSuccess) {
    if (!gq::fp8_silu_takes(a.N, a.w_pitch)) {  // inter is no multiple of 128, mostly: product and activation apart
      e = product(a, s);
      if (e == hipSuccess) e = gq::launch_fp8_quantize(ws.both, slots, inter, MI355GQ_F32, true, ws.hq, inter, ws.hs, s);
    } else if (by_rows) {
      gq::Fp8RowsArgs r = few_rows(a);
      r.q_out = ws.hq;
      r.scale_out = ws.hs;
      e = gq::launch_fp8_rows(r, s);
    } else {
      a.q_out = ws.hq;
      a.scale_out = ws.hs;
      e = gq::launch_fp8_tile(a, s);
      a.q_out = nullptr;
      a.scale_out = nullptr;
    }
  }
  a.precise = false;  // the layer's output has 16 bits: as a linear's (4096 rows of 8 x 4096 x 14336 297 us, with float32 sums throughout 466)
  a.x = ws.hq;
  a.xs = ws.hs;
  a.x_pitch = inter;
  a.x_rows = slots;
  a.x_row_index = nullptr;
  a.w = static_cast<const uint8_t*>(w2);
  a.ws = static_cast<const float*>(w2_scale);
  a.w_pitch = w2_pitch;
  a.N = hidden;
  a.K = inter;
  a.y = ws.y;  // float32: one rounding, behind the weighted sum, where two made the error 1.4 times as large (4 of 159 us for 509 tokens)
  a.out_dtype = MI355GQ_F32;
  if (e == hipSuccess) e = product(a, s);
  if (e == hipSuccess)
    e = gq::launch_moe_weighted_sum(ws.y, ws.slot_row, static_cast<const float*>(weights), T, static_cast<int>(top_k), hidden,
                                    model_dtype, out, s);
  return hip_result(e, "fp8_moe launch");
}

}  // extern "C"
