// The dense operators' way from a Python call to a kernel launch, in native code: argument checks, the output and scratch
// allocation, the current stream and the C ABI call of linear / linear_silu_mul / embedding_take and of the operators on 8-bit and 16-bit weights, one
// Python call each.
//
// What it replaces took 13 us of interpreter time per projection (a torch.cuda.Stream object, three Python checks per tensor, two
// ctypes calls), which is more than a decode projection takes on the GPU: a one-row 4096 x 4096 linear took 14.0 us per call for
// a 4.3 us kernel (7.3 us this way), and every decode step of one to a few rows was bound by it (34 linears of an 8-layer step with
// one row: 455 -> 332 us, with 3-bit weights 449 -> 277).
//
// A function returns the output tensor, or the C ABI's (negative) code as an int, or None where the arguments are not what it
// expects: plain strided tensors on the GPU of the types and shapes that the operator takes, no torch function mode.  The caller
// then runs the Python route, which accepts or refuses them in its own words; nothing is accepted here that is refused there.
#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include "../../include/mi355gq.h"

namespace {

using at::ScalarType;
using at::Tensor;

// A plain tensor in GPU memory; a subclass may mean anything by its methods and goes to the Python route.
const Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.is_contiguous() ? &t : nullptr;
}

// the model dtypes -> the C ABI's codes, -1 for anything else
int model_code(ScalarType t) {
  switch (t) {
    case ScalarType::Half: return MI355GQ_F16;
    case ScalarType::Float: return MI355GQ_F32;
    case ScalarType::BFloat16: return MI355GQ_BF16;
    default: return -1;
  }
}

bool small_int(PyObject* o, int* out) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long v = PyLong_AsLongAndOverflow(o, &overflow);
  if (overflow || v < 1 || v > 1 << 20) return false;
  *out = static_cast<int>(v);
  return true;
}

struct Packed {
  const Tensor *words, *scales;
  int bits, group;
};

// q_weight [N, words(K)] and q_scale [N, groups(K)] of `dtype`
bool packed_fits(const Packed& p, int64_t n, int64_t k, ScalarType dtype) {
  if (p.bits > 32 || p.words->dim() != 2 || p.scales->dim() != 2 || p.scales->scalar_type() != dtype) return false;
  const ScalarType w = p.words->scalar_type();
  if (w != ScalarType::Int && w != ScalarType::UInt32) return false;
  const int64_t groups = (k + p.group - 1) / p.group, words = (p.group / (32 / p.bits)) * groups;
  return p.words->size(0) == n && p.words->size(1) == words && p.scales->size(0) == n && p.scales->size(1) == groups;
}

bool packed_args(PyObject* const* a, Packed* p) {
  p->words = plain(a[0]);
  p->scales = plain(a[1]);
  return p->words && p->scales && small_int(a[2], &p->bits) && small_int(a[3], &p->group);
}

void* current_stream() { return c10::hip::getCurrentHIPStream().stream(); }

// leading sizes of x, then `last`
c10::SmallVector<int64_t, 6> with_last(const Tensor& x, int64_t last) {
  c10::SmallVector<int64_t, 6> s(x.sizes().begin(), x.sizes().end());
  s.back() = last;
  return s;
}

int64_t leading_rows(const Tensor& x) {
  int64_t m = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) m *= x.size(d);
  return m;
}

// scratch for one call, given back to the allocator when it goes (the kernels that use it are on the same stream)
struct Scratch {
  Tensor t;
  void* ptr = nullptr;
  Scratch(const Tensor& like, int64_t bytes) {
    if (bytes == 0) return;
    t = at::empty({bytes}, like.options().dtype(at::kByte));
    ptr = t.mutable_data_ptr();
  }
};

PyObject* result(int rc, const Tensor& out) { return rc == MI355GQ_OK ? THPVariable_Wrap(out) : PyLong_FromLong(rc); }

// linear(x, q_weight, q_scale, bits, group_size, bias | None, out_dtype, out | None, residual | None)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Packed p;
  if (nargs != 9 || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const Tensor* x = plain(a[0]);
  if (!x || x->dim() < 1 || !packed_args(a + 1, &p) || !THPDtype_Check(a[6])) Py_RETURN_NONE;
  const ScalarType dtype = x->scalar_type();
  const int code = model_code(dtype);
  const int64_t k = x->size(-1), n = p.words->dim() ? p.words->size(0) : -1, m = leading_rows(*x);
  if (code < 0 || !packed_fits(p, n, k, dtype)) Py_RETURN_NONE;
  ScalarType out_dtype = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  if (out_dtype == ScalarType::Half) out_dtype = dtype;  // the signature's default: a model's own dtype
  if (out_dtype != dtype && out_dtype != ScalarType::Float) Py_RETURN_NONE;
  const Tensor *bias = nullptr, *given = nullptr, *residual = nullptr;
  if (a[5] != Py_None) {
    bias = plain(a[5]);
    if (!bias || bias->scalar_type() != dtype || bias->dim() != 1 || bias->size(0) != n) Py_RETURN_NONE;
  }
  const auto shape = with_last(*x, n);
  if (a[7] != Py_None) {
    given = plain(a[7]);
    if (!given || given->scalar_type() != out_dtype || given->sizes() != at::IntArrayRef(shape)) Py_RETURN_NONE;
  }
  if (a[8] != Py_None) {
    residual = plain(a[8]);
    if (!residual || residual->scalar_type() != dtype || residual->sizes() != at::IntArrayRef(shape)) Py_RETURN_NONE;
  }
  Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release release;
    out = given ? *given : at::empty(shape, x->options().dtype(out_dtype));
    const int64_t bytes = mi355gq_linear_dt_workspace_bytes(m, n, k, p.bits, p.group, code);
    Scratch ws(*x, bytes);
    const void *xp = x->const_data_ptr(), *wp = p.words->const_data_ptr(), *sp = p.scales->const_data_ptr(),
               *bp = bias ? bias->const_data_ptr() : nullptr;
    void* yp = out.mutable_data_ptr();
    const int oc = model_code(out_dtype);
    if (residual)
      rc = mi355gq_linear_residual_dt(xp, wp, sp, bp, residual->const_data_ptr(), m, n, k, p.bits, p.group, code, oc, yp, ws.ptr,
                                      bytes, current_stream());
    else
      rc = mi355gq_linear_dt(xp, wp, sp, bp, m, n, k, p.bits, p.group, code, oc, yp, ws.ptr, bytes, current_stream());
  }
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// linear_silu_mul(x, q_weight, q_scale, bits, group_size)
PyObject* linear_silu_mul(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Packed p;
  if (nargs != 5 || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const Tensor* x = plain(a[0]);
  if (!x || x->dim() < 1 || !packed_args(a + 1, &p)) Py_RETURN_NONE;
  const ScalarType dtype = x->scalar_type();
  const int code = model_code(dtype);
  const int64_t k = x->size(-1), n = p.words->dim() ? p.words->size(0) : -1, m = leading_rows(*x);
  if (code < 0 || !packed_fits(p, n, k, dtype) || n % 2) Py_RETURN_NONE;
  Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release release;
    out = at::empty(with_last(*x, n / 2), x->options());
    const int64_t bytes = mi355gq_linear_silu_mul_dt_workspace_bytes(m, n, k, p.bits, p.group, code);
    Scratch ws(*x, bytes);
    rc = mi355gq_linear_silu_mul_dt(x->const_data_ptr(), p.words->const_data_ptr(), p.scales->const_data_ptr(), m, n, k, p.bits,
                                    p.group, code, out.mutable_data_ptr(), ws.ptr, bytes, current_stream());
  }
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// embedding_take(ids, q_weight, q_scale, k, bits, group_size)
PyObject* embedding_take(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Packed p;
  PyObject* packed[4];
  int k = 0;
  if (nargs != 6 || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  packed[0] = a[1], packed[1] = a[2], packed[2] = a[4], packed[3] = a[5];
  const Tensor* ids = plain(a[0]);
  if (!ids || ids->scalar_type() != ScalarType::Int || !packed_args(packed, &p) || !small_int(a[3], &k)) Py_RETURN_NONE;
  const ScalarType dtype = p.scales->scalar_type();
  const int code = model_code(dtype);
  const int64_t rows = p.words->dim() ? p.words->size(0) : -1;
  if (code < 0 || !packed_fits(p, rows, k, dtype)) Py_RETURN_NONE;
  Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release release;
    c10::SmallVector<int64_t, 6> shape(ids->sizes().begin(), ids->sizes().end());
    shape.push_back(k);
    out = at::empty(shape, p.scales->options());
    rc = mi355gq_embedding_take_dt(ids->const_data_ptr(), ids->numel(), p.words->const_data_ptr(), p.scales->const_data_ptr(), rows,
                                   k, p.bits, p.group, code, out.mutable_data_ptr(), current_stream());
  }
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// ---- 8-bit block-scaled operators (no weights in integers: e4m3 tensors, whose rows may lie further apart than they are long) ----

constexpr int64_t kBlock = 128;
int64_t blocks(int64_t k) { return (k + kBlock - 1) / kBlock; }

// An e4m3 tensor of `dims` dimensions with contiguous rows of K, a multiple of 16 here; its pitch, or -1.
int64_t e4m3_pitch(PyObject* o, int64_t dims, const Tensor** out) {
  if (!THPVariable_CheckExact(o)) return -1;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.scalar_type() != ScalarType::Float8_e4m3fn || t.dim() != dims || t.numel() == 0)
    return -1;
  const int64_t k = t.size(-1), pitch = t.size(-2) > 1 ? t.stride(-2) : k;
  if (k % 16 || t.stride(-1) != 1 || pitch < k || pitch % 16 || (dims == 3 && t.size(0) > 1 && t.stride(0) != t.size(1) * pitch)) return -1;
  *out = &t;
  return pitch;
}

bool floats(const Tensor* t, at::IntArrayRef sizes) { return t && t->scalar_type() == ScalarType::Float && t->sizes() == sizes; }

bool truth(PyObject* o, bool* out) {
  if (!PyBool_Check(o)) return false;
  *out = o == Py_True;
  return true;
}

// fp8_quantize(x): (q, scale)
PyObject* fp8_quantize(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 1 || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const Tensor* x = plain(a[0]);
  if (!x || x->dim() != 2 || x->numel() == 0 || x->size(1) % 16) Py_RETURN_NONE;
  const int code = model_code(x->scalar_type());
  if (code < 0) Py_RETURN_NONE;
  Tensor q, scale;
  int rc;
  {
    pybind11::gil_scoped_release release;
    const int64_t rows = x->size(0), k = x->size(1);
    q = at::empty({rows, k}, x->options().dtype(ScalarType::Float8_e4m3fn));
    scale = at::empty({blocks(k), rows}, x->options().dtype(ScalarType::Float));
    rc = mi355gq_fp8_quantize(x->const_data_ptr(), rows, k, code, q.mutable_data_ptr(), k, scale.mutable_data_ptr(), current_stream());
  }
  if (rc != MI355GQ_OK) return PyLong_FromLong(rc);
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(q));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(scale));
  return pair;
  END_HANDLE_TH_ERRORS
}

// fp8_linear(x, weight, weight_scale, bias | None, out_dtype | None, residual | None, precise | None), x a tensor of numbers
PyObject* fp8_linear(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7 || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const Tensor *x = plain(a[0]), *w = nullptr, *ws = plain(a[2]), *bias = nullptr, *residual = nullptr;
  const int64_t pitch = e4m3_pitch(a[1], 2, &w);
  if (!x || x->dim() < 1 || pitch < 0) Py_RETURN_NONE;
  const ScalarType dtype = x->scalar_type();
  const int code = model_code(dtype);
  const int64_t n = w->size(0), k = w->size(1), m = leading_rows(*x);
  if (code < 0 || x->size(-1) != k || !floats(ws, {blocks(n), blocks(k)})) Py_RETURN_NONE;
  const auto shape = with_last(*x, n);
  ScalarType out_dtype = dtype;
  if (a[4] != Py_None) {
    if (!THPDtype_Check(a[4])) Py_RETURN_NONE;
    out_dtype = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  }
  const int out_code = model_code(out_dtype);
  bool precise = out_dtype == ScalarType::Float;
  if (out_code < 0 || (a[6] != Py_None && !truth(a[6], &precise))) Py_RETURN_NONE;
  if (a[3] != Py_None) {
    bias = plain(a[3]);
    if (!bias || bias->scalar_type() != dtype || bias->dim() != 1 || bias->size(0) != n) Py_RETURN_NONE;
  }
  if (a[5] != Py_None) {
    residual = plain(a[5]);
    if (!residual || residual->scalar_type() != dtype || residual->sizes() != at::IntArrayRef(shape)) Py_RETURN_NONE;
  }
  Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release release;
    out = at::empty(shape, x->options().dtype(out_dtype));
    const int64_t bytes = mi355gq_fp8_linear_workspace_bytes(m, n, k, 0);
    Scratch scratch(*x, bytes);
    rc = mi355gq_fp8_linear(x->const_data_ptr(), 0, nullptr, w->const_data_ptr(), pitch, ws->const_data_ptr(),
                            bias ? bias->const_data_ptr() : nullptr, residual ? residual->const_data_ptr() : nullptr, m, n, k, code, out_code,
                            precise ? 1 : 0, out.mutable_data_ptr(), scratch.ptr, bytes, current_stream());
  }
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

struct Gating {
  const Tensor *logits, *bias = nullptr;
  int code, k, scoring, groups, top_groups;
  bool renormalize;
  float scale;
};
// logits, top_k, scoring, bias | None, num_groups, top_groups, renormalize, scale
bool gating_args(PyObject* const* a, Gating* g) {
  g->logits = plain(a[0]);
  if (!g->logits || g->logits->dim() != 2 || !small_int(a[1], &g->k) || !PyUnicode_CheckExact(a[2]) || !small_int(a[4], &g->groups) ||
      !small_int(a[5], &g->top_groups) || !truth(a[6], &g->renormalize) || !PyFloat_CheckExact(a[7]))
    return false;
  g->code = model_code(g->logits->scalar_type());
  if (PyUnicode_CompareWithASCIIString(a[2], "softmax") == 0) g->scoring = MI355GQ_SCORE_SOFTMAX;
  else if (PyUnicode_CompareWithASCIIString(a[2], "sigmoid") == 0) g->scoring = MI355GQ_SCORE_SIGMOID;
  else return false;
  if (a[3] != Py_None) {
    g->bias = plain(a[3]);
    if (!floats(g->bias, {g->logits->size(1)})) return false;
  }
  g->scale = static_cast<float>(PyFloat_AS_DOUBLE(a[7]));
  return g->code >= 0;
}
int run_gating(const Gating& g, Tensor* weights, Tensor* ids) {
  const int64_t t = g.logits->size(0);
  *weights = at::empty({t, g.k}, g.logits->options().dtype(ScalarType::Float));
  *ids = at::empty({t, g.k}, g.logits->options().dtype(ScalarType::Int));
  return mi355gq_moe_gating(g.logits->const_data_ptr(), g.bias ? g.bias->const_data_ptr() : nullptr, t, g.logits->size(1), g.k, g.scoring,
                            g.groups, g.top_groups, g.renormalize ? 1 : 0, g.scale, g.code, weights->mutable_data_ptr(),
                            ids->mutable_data_ptr(), current_stream());
}

// moe_gating(logits, top_k, scoring, bias | None, num_groups, top_groups, renormalize, scale): (weights, ids)
PyObject* moe_gating(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Gating g;
  if (nargs != 8 || at::impl::torch_function_mode_enabled() || !gating_args(a, &g)) Py_RETURN_NONE;
  Tensor weights, ids;
  int rc;
  {
    pybind11::gil_scoped_release release;
    rc = run_gating(g, &weights, &ids);
  }
  if (rc != MI355GQ_OK) return PyLong_FromLong(rc);
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(weights));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(ids));
  return pair;
  END_HANDLE_TH_ERRORS
}

// fp8_moe(x, w13, w13_scale, w2, w2_scale, then moe_gating's arguments)
PyObject* fp8_moe(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Gating g;
  if (nargs != 13 || at::impl::torch_function_mode_enabled() || !gating_args(a + 5, &g)) Py_RETURN_NONE;
  const Tensor *x = plain(a[0]), *w13 = nullptr, *w2 = nullptr, *s13 = plain(a[2]), *s2 = plain(a[4]);
  const int64_t p13 = e4m3_pitch(a[1], 3, &w13), p2 = e4m3_pitch(a[3], 3, &w2);
  if (!x || x->dim() != 2 || p13 < 0 || p2 < 0) Py_RETURN_NONE;
  const int code = model_code(x->scalar_type());
  const int64_t t = x->size(0), experts = w2->size(0), hidden = w2->size(1), inter = w2->size(2);
  if ((code != MI355GQ_F16 && code != MI355GQ_BF16) || t == 0 || x->size(1) != hidden || w13->sizes() != at::IntArrayRef({experts, 2 * inter, hidden}) ||
      g.logits->size(0) != t || g.logits->size(1) != experts || !floats(s13, {experts, blocks(2 * inter), blocks(hidden)}) ||
      !floats(s2, {experts, blocks(hidden), blocks(inter)}))
    Py_RETURN_NONE;
  Tensor out, weights, ids;
  int rc;
  {
    pybind11::gil_scoped_release release;
    rc = run_gating(g, &weights, &ids);
    if (rc == MI355GQ_OK) {
      out = at::empty(x->sizes(), x->options());
      int64_t bytes = mi355gq_fp8_moe_workspace_bytes(t, hidden, inter, experts, g.k);
      if (2 * inter * p13 >= 0xffffffffll) bytes += 8 * t * g.k * inter + 256;
      Scratch scratch(*x, bytes);
      rc = mi355gq_fp8_moe(x->const_data_ptr(), t, hidden, inter, experts, g.k, weights.const_data_ptr(), ids.const_data_ptr(),
                           w13->const_data_ptr(), p13, s13->const_data_ptr(), w2->const_data_ptr(), p2, s2->const_data_ptr(), code,
                           out.mutable_data_ptr(), scratch.ptr, bytes, current_stream());
    }
  }
  if (rc != MI355GQ_OK) Py_RETURN_NONE;  // the Python route names the call that failed
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ---- operators on 16-bit weights: on x's GPU, whichever is current, and its current stream ----

bool activation(PyObject* o, int* act) {
  static const char* const names[] = {"relu", "silu", "gelu", "gelu_tanh"};
  if (o == Py_None) {
    *act = MI355GQ_ACT_NONE;
    return true;
  }
  if (!PyUnicode_CheckExact(o)) return false;
  for (int i = 0; i < 4; ++i)
    if (PyUnicode_CompareWithASCIIString(o, names[i]) == 0) {
      *act = MI355GQ_ACT_RELU + i;
      return true;
    }
  return false;
}

bool half_code(ScalarType t, int* code) {
  *code = model_code(t);
  return *code == MI355GQ_F16 || *code == MI355GQ_BF16;
}

// a tensor of x's type and GPU with these sizes
const Tensor* beside(PyObject* o, const Tensor& x, at::IntArrayRef sizes) {
  const Tensor* t = plain(o);
  return t && t->scalar_type() == x.scalar_type() && t->device() == x.device() && t->sizes() == sizes ? t : nullptr;
}

void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.device().index()).stream(); }

bool overlap(const Tensor& a, const Tensor& b) {
  const char *a0 = static_cast<const char*>(a.const_data_ptr()), *b0 = static_cast<const char*>(b.const_data_ptr());
  return a0 < b0 + b.nbytes() && b0 < a0 + a.nbytes();
}

// dense(x, weight, bias | None, activation | None, out_dtype | None, residual | None, out | None): GATED without the last two
template <bool GATED>
PyObject* dense(PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != (GATED ? 5 : 7) || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const Tensor *x = plain(a[0]), *w = plain(a[1]), *bias = nullptr, *residual = nullptr;
  int act = 0, code = 0;
  if (!x || !w || x->dim() < 1 || w->dim() != 2 || !half_code(x->scalar_type(), &code) || w->scalar_type() != x->scalar_type() || w->device() != x->device() ||
      !activation(a[3], &act))
    Py_RETURN_NONE;
  const int64_t k = x->size(-1), rows_of_w = w->size(0), n = GATED ? rows_of_w / 2 : rows_of_w, m = leading_rows(*x);
  if (w->size(1) != k || k == 0 || m == 0 || n == 0 || (GATED && rows_of_w % 2)) Py_RETURN_NONE;
  if (a[2] != Py_None && !(bias = beside(a[2], *x, {rows_of_w}))) Py_RETURN_NONE;
  ScalarType out_dtype = x->scalar_type();
  if (a[4] != Py_None) {
    if (!THPDtype_Check(a[4])) Py_RETURN_NONE;
    out_dtype = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    if (out_dtype != x->scalar_type() && out_dtype != ScalarType::Float) Py_RETURN_NONE;
  }
  const auto shape = with_last(*x, n);
  const Tensor* given = nullptr;
  if constexpr (!GATED) {
    if (a[5] != Py_None && !(residual = beside(a[5], *x, shape))) Py_RETURN_NONE;
    if (a[6] != Py_None) {
      given = plain(a[6]);
      if (!given || given->scalar_type() != out_dtype || given->device() != x->device() || given->sizes() != at::IntArrayRef(shape) || overlap(*given, *x) ||
          overlap(*given, *w) || (bias && overlap(*given, *bias)) ||
          (residual && overlap(*given, *residual) && (given->const_data_ptr() != residual->const_data_ptr() || out_dtype != residual->scalar_type())))
        Py_RETURN_NONE;
    }
  }
  Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release release;
    const c10::DeviceGuard guard(x->device());
    out = given ? *given : at::empty(shape, x->options().dtype(out_dtype));
    const int64_t bytes = mi355gq_dense_linear_workspace_bytes(m, n, k, GATED);
    Scratch ws(*x, bytes);
    const void *xp = x->const_data_ptr(), *wp = w->const_data_ptr(), *bp = bias ? bias->const_data_ptr() : nullptr;
    if constexpr (GATED)
      rc = mi355gq_dense_linear_gated(xp, wp, bp, m, n, k, act, code, model_code(out_dtype), out.mutable_data_ptr(), ws.ptr, bytes, stream_of(*x));
    else
      rc = mi355gq_dense_linear(xp, wp, bp, residual ? residual->const_data_ptr() : nullptr, m, n, k, act, code, model_code(out_dtype),
                                out.mutable_data_ptr(), ws.ptr, bytes, stream_of(*x));
  }
  return result(rc, out);
}
PyObject* dense_linear(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  return dense<false>(a, nargs);
  END_HANDLE_TH_ERRORS
}
PyObject* dense_linear_gated(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  return dense<true>(a, nargs);
  END_HANDLE_TH_ERRORS
}

// dense_moe(x, w13, w2, activation | None, then moe_gating's arguments)
PyObject* dense_moe(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Gating g;
  int act = 0, code = 0;
  if (nargs != 12 || at::impl::torch_function_mode_enabled() || !gating_args(a + 4, &g) || !activation(a[3], &act)) Py_RETURN_NONE;
  const Tensor *x = plain(a[0]), *w2 = plain(a[2]);
  if (!x || !w2 || x->dim() != 2 || w2->dim() != 3 || !half_code(x->scalar_type(), &code) || w2->scalar_type() != x->scalar_type()) Py_RETURN_NONE;
  const int64_t t = x->size(0), experts = w2->size(0), hidden = w2->size(1), inter = w2->size(2);
  const Tensor* w13 = beside(a[1], *x, {experts, 2 * inter, hidden});
  if (!w13 || t == 0 || x->size(1) != hidden || w2->device() != x->device() || g.logits->device() != x->device() || g.logits->size(0) != t ||
      g.logits->size(1) != experts || (g.bias && g.bias->device() != x->device()) || reinterpret_cast<uintptr_t>(x->const_data_ptr()) % 16)
    Py_RETURN_NONE;
  Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release release;
    const c10::DeviceGuard guard(x->device());
    out = at::empty(x->sizes(), x->options());
    const int64_t bytes = mi355gq_dense_moe_workspace_bytes(t, hidden, inter, experts, g.k);
    Scratch ws(*x, bytes);
    rc = mi355gq_dense_moe(x->const_data_ptr(), g.logits->const_data_ptr(), g.bias ? g.bias->const_data_ptr() : nullptr, t, hidden, inter, experts, g.k,
                           g.scoring, g.groups, g.top_groups, g.renormalize ? 1 : 0, g.scale, g.code, w13->const_data_ptr(), w2->const_data_ptr(), act,
                           code, out.mutable_data_ptr(), ws.ptr, bytes, stream_of(*x));
  }
  return result(rc, out);
  END_HANDLE_TH_ERRORS
}

// the current HIP stream of the current device, as a number
PyObject* stream(PyObject*, PyObject*) {
  HANDLE_TH_ERRORS
  return PyLong_FromVoidPtr(current_stream());
  END_HANDLE_TH_ERRORS
}

#define GQ_FAST(fn) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL
PyMethodDef kMethods[] = {
    {"linear", GQ_FAST(linear), nullptr},
    {"linear_silu_mul", GQ_FAST(linear_silu_mul), nullptr},
    {"embedding_take", GQ_FAST(embedding_take), nullptr},
    {"fp8_quantize", GQ_FAST(fp8_quantize), nullptr},
    {"fp8_linear", GQ_FAST(fp8_linear), nullptr},
    {"moe_gating", GQ_FAST(moe_gating), nullptr},
    {"fp8_moe", GQ_FAST(fp8_moe), nullptr},
    {"dense_linear", GQ_FAST(dense_linear), nullptr},
    {"dense_linear_gated", GQ_FAST(dense_linear_gated), nullptr},
    {"dense_moe", GQ_FAST(dense_moe), nullptr},
    {"stream", stream, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_mi355gq_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mi355gq_torch() { return PyModule_Create(&kModule); }
