// Python binding of the operators (module tila_b200._ops): reads torch tensors,
// checks the arguments and calls the C ABI.  A call of a small operator costs the
// host about as much as the GPU; in Python the checks alone took 15 to 30 us.
//
// Every refusal is a ValueError (TypeError for what is no tensor) raised before
// anything is launched or allocated.  That the tensors are on a GPU is the last
// check, so that the others can be tested without one.

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <optional>
#include <string>
#include <vector>

#include "../../../include/tila_b200.h"

namespace {

using at::Tensor;

// ---------------------------------------------------------------------------
// errors
// ---------------------------------------------------------------------------

struct Refused : std::exception {
  PyObject *kind;
  std::string text;
  Refused(PyObject *k, std::string t) : kind(k), text(std::move(t)) {}
};
struct Raised : std::exception {};   // a Python exception is set

[[noreturn]] void refuse_as(PyObject *kind, const char *fmt, va_list ap) {
  char buf[512];
  vsnprintf(buf, sizeof(buf), fmt, ap);
  throw Refused(kind, buf);
}
[[noreturn]] void refuse(const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  refuse_as(PyExc_ValueError, fmt, ap);
}
[[noreturn]] void mistyped(const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  refuse_as(PyExc_TypeError, fmt, ap);
}

std::string text(at::IntArrayRef sizes) {
  std::string s = "(";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + (sizes.size() == 1 ? ",)" : ")");
}

// ---------------------------------------------------------------------------
// device state: error blocks, made by the Python side on first use
// ---------------------------------------------------------------------------

constexpr int kMaxDevices = 64;
struct ErrorBlock {
  uint64_t address = 0;
  const volatile uint32_t *word = nullptr;
};
ErrorBlock g_blocks[kMaxDevices];
PyObject *g_prepare = nullptr;   // prepare(index): set_error_block(index, ...)
PyObject *g_check = nullptr;     // check(index): raises for a recorded error
PyObject *g_native_error = nullptr;

void call(PyObject *f, int index) {
  PyObject *r = f == nullptr ? nullptr : PyObject_CallFunction(f, "i", index);
  if (r == nullptr) throw Raised();
  Py_DECREF(r);
}

uint64_t error_block(int index) {
  if (index < 0 || index >= kMaxDevices) refuse("device index %d is out of range", index);
  if (g_blocks[index].address == 0) call(g_prepare, index);
  if (*g_blocks[index].word != 0) call(g_check, index);
  return g_blocks[index].address;
}

void check_status(int status, const char *entry, const char *log) {
  if (status == TILA_OK) return;
  if (status == TILA_ERR_ARGUMENT) refuse("%s", log);
  const std::string message = std::string(entry) + ": " + tila_status_string(status);
  PyObject *e = PyObject_CallFunction(g_native_error, "iss", status, message.c_str(), log);
  if (e != nullptr) {
    PyErr_SetObject(g_native_error, e);
    Py_DECREF(e);
  }
  throw Raised();
}

// ---------------------------------------------------------------------------
// arguments
// ---------------------------------------------------------------------------

const Tensor &tensor(const char *fn, const char *what, PyObject *o) {
  if (!THPVariable_Check(o)) mistyped("%s: %s must be a tensor, not %s", fn, what, Py_TYPE(o)->tp_name);
  const Tensor &t = THPVariable_Unpack(o);
  // (its memory holds the values with their signs turned)
  if (t.is_neg()) refuse("%s: %s is a view that negates (of a conjugate's imaginary part): resolve_neg() it", fn, what);
  return t;
}

void on_device_of(const char *fn, const char *what, const Tensor &t, const Tensor &like) {
  if (t.device() != like.device())
    refuse("%s: %s is on %s, the other tensors on %s", fn, what, t.device().str().c_str(), like.device().str().c_str());
}

void on_gpu(const char *fn, const char *what, const Tensor &t) {
  if (!t.is_cuda()) refuse("%s: %s must be a CUDA tensor", fn, what);
}

void of_dtype(const char *fn, const char *what, const Tensor &t, at::ScalarType dtype) {
  if (t.scalar_type() != dtype)
    refuse("%s: %s must be %s, not %s", fn, what, c10::toString(dtype), c10::toString(t.scalar_type()));
}

void of_rank(const char *fn, const char *what, const Tensor &t, int rank) {
  if (t.dim() != rank) refuse("%s: %s must have %d dimensions, not %d", fn, what, rank, static_cast<int>(t.dim()));
}

void unit_last(const char *fn, const char *what, const Tensor &t) {
  if (t.stride(-1) != 1 && t.size(-1) > 1 && t.numel() > 0)
    refuse("%s: the last dimension of %s must be contiguous", fn, what);
}

int element_type(at::ScalarType t) {
  return t == at::kFloat ? TILA_F32 : t == at::kHalf ? TILA_F16 : t == at::kBFloat16 ? TILA_BF16 : -1;
}

uint64_t address(const Tensor &t) { return reinterpret_cast<uint64_t>(t.data_ptr()); }

double number(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}
int64_t whole(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}

// ---- overlap ----

int64_t extent(at::IntArrayRef sizes, at::IntArrayRef strides) {
  int64_t n = 1;
  for (size_t i = 0; i < sizes.size(); ++i) n += (sizes[i] - 1) * strides[i];
  return n;
}

// Refuses a result whose elements share memory (an expanded tensor).
void writable(const char *fn, const char *what, const Tensor &t) {
  if (t.is_contiguous()) return;
  std::vector<std::pair<int64_t, int64_t>> d;
  for (int i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) d.emplace_back(t.stride(i), t.size(i));
  std::sort(d.begin(), d.end());
  int64_t span = 1;
  for (auto [stride, size] : d) {
    if (stride < span) refuse("%s: elements of %s share memory", fn, what);
    span += (size - 1) * stride;
  }
}

// Refuses a result `a` that overlaps `b`.  It may lie between the rows or pages of
// `b` (two parts of one tensor) and, with `same`, be exactly the elements of `b` (a
// result in the place of its source).
void apart(const char *fn, const char *what, const Tensor &a, const char *other, const Tensor &b, bool same = false) {
  if (a.numel() == 0 || b.numel() == 0) return;
  const int64_t pa = static_cast<int64_t>(address(a)), pb = static_cast<int64_t>(address(b));
  const int64_t size = a.element_size();
  if (pa >= pb + extent(b.sizes(), b.strides()) * b.element_size() || pb >= pa + extent(a.sizes(), a.strides()) * size)
    return;
  if (a.scalar_type() == b.scalar_type()) {
    if (same && pa == pb && a.sizes() == b.sizes() && a.strides() == b.strides()) return;
    // equal steps in the outer dimensions: both lie in windows of one period
    for (int outer = 1; outer < a.dim(); ++outer) {
      const int64_t period = a.stride(outer - 1);
      if (b.dim() != a.dim() || a.size(outer - 1) != b.size(outer - 1) || period != b.stride(outer - 1) || period <= 0 ||
          (pb - pa) % size != 0)
        break;
      const int64_t shift = (((pb - pa) / size) % period + period) % period;
      bool whole_periods = true;
      for (int i = 0; i < outer; ++i) whole_periods = whole_periods && a.stride(i) % period == 0;
      if (whole_periods && shift >= extent(a.sizes().slice(outer), a.strides().slice(outer)) &&
          period - shift >= extent(b.sizes().slice(outer), b.strides().slice(outer)))
        return;
    }
  }
  refuse("%s: %s overlaps %s", fn, what, other);
}

struct Named {
  const char *what;
  const Tensor *t;
};

// Refuses a call that autograd would have to record: its result would pass for a
// constant, and gradients upstream of it would silently be zero.
void unrecorded(const char *fn, std::initializer_list<Named> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const Named &n : tensors)
    if (n.t->requires_grad())
      refuse("%s: %s requires a gradient, which autograd does not record here: call it under torch.no_grad(), or in a "
             "torch.autograd.Function", fn, n.what);
}

// The caller's result after its checks (None: one is made once everything else is
// checked).
std::optional<Tensor> result(const char *fn, const char *what, PyObject *o, const Tensor &like,
                             std::initializer_list<Named> own, std::initializer_list<Named> others) {
  if (o == Py_None) return std::nullopt;
  const Tensor &out = tensor(fn, what, o);
  unrecorded(fn, {{what, &out}});
  on_device_of(fn, what, out, like);
  of_dtype(fn, what, out, like.scalar_type());
  if (out.sizes() != like.sizes())
    refuse("%s: %s must have the shape %s, not %s", fn, what, text(like.sizes()).c_str(), text(out.sizes()).c_str());
  unit_last(fn, what, out);
  writable(fn, what, out);
  for (const Named &n : own) apart(fn, what, out, n.what, *n.t, true);
  for (const Named &n : others) apart(fn, what, out, n.what, *n.t);
  return out;
}

// Tells autograd that a tensor of the caller's was written: a backward pass that had
// saved it finds out.
void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor &like) {
  return Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt));
}

// ---------------------------------------------------------------------------
// rotary
// ---------------------------------------------------------------------------

void rows_shape(const char *fn, const char *what, const Tensor &x) {
  if (element_type(x.scalar_type()) < 0)
    refuse("%s: %s must be float32, float16 or bfloat16, not %s", fn, what, c10::toString(x.scalar_type()));
  if (x.dim() != 3 && x.dim() != 4)
    refuse("%s: %s must be (tokens, heads, dim) or (batch, tokens, heads, dim)", fn, what);
  if (x.size(-1) < 1 || x.size(-1) > 512)
    refuse("%s: %s must have heads of 1 to 512 elements, not %lld", fn, what, static_cast<long long>(x.size(-1)));
  if (x.size(-2) > (1 << 20))
    refuse("%s: %s must have at most 2^20 heads, not %lld", fn, what, static_cast<long long>(x.size(-2)));
  unit_last(fn, what, x);
}

// Fills the part of the arguments that says where each token is turned to.
void positions(const char *fn, PyObject *pos_o, PyObject *freq_o, const Tensor &x, tila_rotary_args &a) {
  const Tensor &pos = tensor(fn, "positions", pos_o);
  on_device_of(fn, "positions", pos, x);
  if (pos.scalar_type() != at::kLong && pos.scalar_type() != at::kInt)
    refuse("%s: positions must be int32 or int64, not %s", fn, c10::toString(pos.scalar_type()));
  const at::IntArrayRef tokens = x.sizes().slice(0, x.dim() - 2);
  if (pos.sizes() == tokens) {
    a.position_stride[0] = tokens.size() == 2 ? pos.stride(0) : 0;
    a.position_stride[1] = pos.stride(-1);
  } else if (tokens.size() == 2 && pos.sizes() == tokens.slice(1)) {
    a.position_stride[0] = 0;
    a.position_stride[1] = pos.stride(0);
  } else {
    refuse("%s: positions must have one position per token, %s, not %s", fn, text(tokens).c_str(),
           text(pos.sizes()).c_str());
  }
  const Tensor &freq = tensor(fn, "inv_freq", freq_o);
  on_device_of(fn, "inv_freq", freq, x);
  of_dtype(fn, "inv_freq", freq, at::kDouble);
  of_rank(fn, "inv_freq", freq, 1);
  if (2 * freq.size(0) > x.size(-1))
    refuse("%s: inv_freq rotates %lld elements, the heads have %lld", fn, static_cast<long long>(2 * freq.size(0)),
           static_cast<long long>(x.size(-1)));
  if (freq.size(0) > 1 && freq.stride(0) != 1) refuse("%s: inv_freq must be contiguous", fn);
  unrecorded(fn, {{"inv_freq", &freq}});
  a.rotary = static_cast<int32_t>(2 * freq.size(0));
  a.positions = address(pos);
  a.inv_freq = address(freq);
  a.index64 |= pos.scalar_type() == at::kLong ? 1 : 0;
}

void layout(const char *fn, PyObject *o, tila_rotary_args &a) {
  if (PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, "half") == 0) {
    a.interleaved = 0;
  } else if (PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, "interleaved") == 0) {
    a.interleaved = 1;
  } else {
    refuse("%s: layout must be 'half' or 'interleaved'", fn);
  }
}

// A stride of tokens or heads, which the kernels take in 32 bits; that of a single one
// is never used and may be any.
int64_t inner_stride(const char *fn, const char *what, const Tensor &t, int d) {
  if (t.stride(d) <= int64_t{0xffffffff}) return t.stride(d);
  if (t.size(d) > 1)
    refuse("%s: strides of %s's tokens and heads must be below 2^32 elements, not %lld", fn, what,
           static_cast<long long>(t.stride(d)));
  return 0;
}

void strides3(const char *fn, const char *what, const Tensor &t, int64_t (&s)[3]) {
  const bool batch = t.dim() == 4;
  s[0] = batch ? t.stride(0) : 0;
  s[1] = inner_stride(fn, what, t, batch ? 1 : 0);
  s[2] = inner_stride(fn, what, t, batch ? 2 : 1);
}

uint32_t weight(const char *fn, const char *what, const Tensor &w, const Tensor &x, tila_op_rows &r) {
  on_device_of(fn, what, w, x);
  of_rank(fn, what, w, 1);
  if (w.scalar_type() != at::kFloat && w.scalar_type() != x.scalar_type())
    refuse("%s: %s must be float32 or %s, not %s", fn, what, c10::toString(x.scalar_type()),
           c10::toString(w.scalar_type()));
  if (w.size(0) != x.size(-1) || (w.size(0) > 1 && w.stride(0) != 1))
    refuse("%s: %s must be a contiguous vector of %lld elements", fn, what, static_cast<long long>(x.size(-1)));
  r.weight = address(w);
  r.flags |= TILA_ROWS_NORM | (w.scalar_type() == at::kFloat ? TILA_ROWS_WEIGHT_F32 : 0);
  return r.flags;
}

tila_rotary_args rotary_args(const Tensor &x) {
  tila_rotary_args a{};
  a.size = sizeof(a);
  a.dtype = element_type(x.scalar_type());
  a.batch = x.dim() == 4 ? x.size(0) : 1;
  a.tokens = x.size(x.dim() == 4 ? 1 : 0);
  a.dim = static_cast<int32_t>(x.size(-1));
  a.amplitude = 1.f;
  return a;
}

void source(const char *fn, const char *what, const Tensor &x, tila_op_rows &r) {
  r.src = address(x);
  strides3(fn, what, x, r.src_stride);
  r.heads = static_cast<int32_t>(x.size(-2));
}
// The caller's result, whose strides are checked with the other arguments, or one made
// for it.
void destination(const char *fn, const char *what, const std::optional<Tensor> &given, tila_op_rows &r) {
  if (given) strides3(fn, what, *given, r.dst_stride);
}
Tensor result_of(const std::optional<Tensor> &given, const Tensor &like, tila_op_rows &r) {
  Tensor out = given ? *given : empty(like.sizes(), like.scalar_type(), like);
  if (!given) strides3("", "", out, r.dst_stride);
  r.dst = address(out);
  return out;
}

// Launches on x's device and its current stream.
void run(int (*entry)(const tila_rotary_args *, char *, size_t), const char *name, const Tensor &x, tila_rotary_args &a,
         Tensor *workspace) {
  const int index = x.get_device();
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != index) guard.set_index(index);
  a.err = error_block(index);
  a.stream = reinterpret_cast<uint64_t>(c10::cuda::getCurrentCUDAStream(index).stream());
  if (workspace != nullptr) {
    a.workspace_bytes = tila_rotary_workspace(&a);
    *workspace = empty({static_cast<int64_t>(a.workspace_bytes)}, at::kByte, x);
    a.workspace = address(*workspace);
  }
  char log[512] = "";
  check_status(entry(&a, log, sizeof(log)), name, log);
}

// rotate(name, x, positions, inv_freq, layout, amplitude, out, inverse)
PyObject *rotate(PyObject *const *o) {
  const bool inverse = o[6] == Py_True;
  const char *fn = inverse ? "rotate_backward" : "rotate", *what = inverse ? "grad" : "x";
  const Tensor &x = tensor(fn, what, o[0]);
  rows_shape(fn, what, x);
  tila_rotary_args a = rotary_args(x);
  layout(fn, o[3], a);
  positions(fn, o[1], o[2], x, a);
  a.amplitude = static_cast<float>(number(o[4]));
  a.inverse = inverse;
  std::optional<Tensor> given = result(fn, "out", o[5], x, {{what, &x}}, {});
  unrecorded(fn, {{what, &x}});
  source(fn, what, x, a.rows[0]);
  destination(fn, "out", given, a.rows[0]);
  on_gpu(fn, what, x);
  Tensor out = result_of(given, x, a.rows[0]);
  a.num_rows = 1;
  a.rows[0].flags = TILA_ROWS_ROTATE;
  run(tila_rotary_rows, "tila_rotary_rows", x, a, nullptr);
  if (!given) return THPVariable_Wrap(std::move(out));
  written(out);
  return Py_NewRef(o[5]);
}

PyObject *pair_of(PyObject *a, PyObject *b) {
  PyObject *r = a != nullptr && b != nullptr ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return r;
}

void query_key(const char *fn, const Tensor &q, const Tensor &k) {
  rows_shape(fn, "q", q);
  rows_shape(fn, "k", k);
  if (k.device() != q.device() || k.scalar_type() != q.scalar_type())
    refuse("%s: q and k must have one device and one dtype", fn);
  if (k.dim() != q.dim() || k.sizes().slice(0, k.dim() - 2) != q.sizes().slice(0, q.dim() - 2) ||
      k.size(-1) != q.size(-1))
    refuse("%s: q and k must have the same tokens and dim: %s and %s", fn, text(q.sizes()).c_str(),
           text(k.sizes()).c_str());
}

// norm_rotate(q, k, q_weight, k_weight, positions, inv_freq, layout, amplitude, eps, q_out, k_out)
PyObject *norm_rotate(PyObject *const *o) {
  const char *fn = "norm_rotate";
  const Tensor &q = tensor(fn, "q", o[0]), &k = tensor(fn, "k", o[1]);
  query_key(fn, q, k);
  tila_rotary_args a = rotary_args(q);
  const Tensor &q_weight = tensor(fn, "q_weight", o[2]), &k_weight = tensor(fn, "k_weight", o[3]);
  weight(fn, "q_weight", q_weight, q, a.rows[0]);
  weight(fn, "k_weight", k_weight, k, a.rows[1]);
  layout(fn, o[6], a);
  positions(fn, o[4], o[5], q, a);
  a.amplitude = static_cast<float>(number(o[7]));
  a.eps = static_cast<float>(number(o[8]));
  std::optional<Tensor> q_given = result(fn, "q_out", o[9], q, {{"q", &q}}, {{"k", &k}});
  std::optional<Tensor> k_given = result(fn, "k_out", o[10], k, {{"k", &k}}, {{"q", &q}});
  if (q_given && k_given) apart(fn, "k_out", *k_given, "q_out", *q_given);
  unrecorded(fn, {{"q", &q}, {"k", &k}, {"q_weight", &q_weight}, {"k_weight", &k_weight}});
  source(fn, "q", q, a.rows[0]);
  source(fn, "k", k, a.rows[1]);
  destination(fn, "q_out", q_given, a.rows[0]);
  destination(fn, "k_out", k_given, a.rows[1]);
  on_gpu(fn, "q", q);
  Tensor q_out = result_of(q_given, q, a.rows[0]), k_out = result_of(k_given, k, a.rows[1]);
  a.num_rows = 2;
  a.rows[0].flags |= TILA_ROWS_ROTATE;
  a.rows[1].flags |= TILA_ROWS_ROTATE;
  run(tila_rotary_rows, "tila_rotary_rows", q, a, nullptr);
  if (q_given) written(q_out);
  if (k_given) written(k_out);
  return pair_of(q_given ? Py_NewRef(o[9]) : THPVariable_Wrap(std::move(q_out)),
                 k_given ? Py_NewRef(o[10]) : THPVariable_Wrap(std::move(k_out)));
}

// norm_rotate_backward(q_grad, k_grad, q, k, q_weight, k_weight, positions, inv_freq, layout, amplitude, eps, dq, dk)
PyObject *norm_rotate_backward(PyObject *const *o) {
  const char *fn = "norm_rotate_backward";
  const Tensor &q = tensor(fn, "q", o[2]), &k = tensor(fn, "k", o[3]);
  query_key(fn, q, k);
  tila_rotary_args a = rotary_args(q);
  const Tensor &q_weight = tensor(fn, "q_weight", o[4]), &k_weight = tensor(fn, "k_weight", o[5]);
  weight(fn, "q_weight", q_weight, q, a.rows[0]);
  weight(fn, "k_weight", k_weight, k, a.rows[1]);
  layout(fn, o[8], a);
  positions(fn, o[6], o[7], q, a);
  a.amplitude = static_cast<float>(number(o[9]));
  a.eps = static_cast<float>(number(o[10]));
  const char *names[2] = {"q_grad", "k_grad"};
  const Tensor *like[2] = {&q, &k}, *grads[2];
  for (int i = 0; i < 2; ++i) {
    const Tensor &g = tensor(fn, names[i], o[i]);
    on_device_of(fn, names[i], g, q);
    of_dtype(fn, names[i], g, q.scalar_type());
    if (g.sizes() != like[i]->sizes())
      refuse("%s: %s must have the shape %s, not %s", fn, names[i], text(like[i]->sizes()).c_str(),
             text(g.sizes()).c_str());
    unit_last(fn, names[i], g);
    a.rows[i].grad = address(g);
    strides3(fn, names[i], g, a.rows[i].grad_stride);
    grads[i] = &g;
  }
  std::optional<Tensor> q_given =
      result(fn, "dq", o[11], q, {{"q", &q}, {"q_grad", grads[0]}}, {{"k", &k}, {"k_grad", grads[1]}});
  std::optional<Tensor> k_given =
      result(fn, "dk", o[12], k, {{"k", &k}, {"k_grad", grads[1]}}, {{"q", &q}, {"q_grad", grads[0]}});
  if (q_given && k_given) apart(fn, "dk", *k_given, "dq", *q_given);
  unrecorded(fn, {{"q_grad", grads[0]}, {"k_grad", grads[1]}, {"q", &q}, {"k", &k}, {"q_weight", &q_weight},
                  {"k_weight", &k_weight}});
  source(fn, "q", q, a.rows[0]);
  source(fn, "k", k, a.rows[1]);
  destination(fn, "dq", q_given, a.rows[0]);
  destination(fn, "dk", k_given, a.rows[1]);
  on_gpu(fn, "q", q);
  Tensor dq = result_of(q_given, q, a.rows[0]), dk = result_of(k_given, k, a.rows[1]);
  Tensor dqw = empty({q.size(-1)}, at::kFloat, q), dkw = empty({q.size(-1)}, at::kFloat, q);
  a.num_rows = 2;
  a.rows[0].flags |= TILA_ROWS_ROTATE;
  a.rows[1].flags |= TILA_ROWS_ROTATE;
  a.weight_grad[0] = address(dqw);
  a.weight_grad[1] = address(dkw);
  Tensor workspace;
  run(tila_rotary_norm_backward, "tila_rotary_norm_backward", q, a, &workspace);
  if (q_given) written(dq);
  if (k_given) written(dk);
  PyObject *r = PyTuple_New(4);
  if (r == nullptr) throw Raised();
  PyTuple_SET_ITEM(r, 0, q_given ? Py_NewRef(o[11]) : THPVariable_Wrap(std::move(dq)));
  PyTuple_SET_ITEM(r, 1, k_given ? Py_NewRef(o[12]) : THPVariable_Wrap(std::move(dk)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(dqw)));
  PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(std::move(dkw)));
  return r;
}

// append_paged(k, v, k_cache, v_cache, slots, positions, inv_freq, layout, amplitude, k_weight, q, q_weight, q_out, eps)
PyObject *append_paged(PyObject *const *o) {
  const char *fn = "append_paged";
  const Tensor &k = tensor(fn, "k", o[0]), &v = tensor(fn, "v", o[1]);
  rows_shape(fn, "k", k);
  if (k.dim() != 3) refuse("%s: k must be (tokens, kv_heads, dim)", fn);
  on_device_of(fn, "v", v, k);
  of_dtype(fn, "v", v, k.scalar_type());
  if (v.sizes() != k.sizes())
    refuse("%s: v must have the shape of k, %s, not %s", fn, text(k.sizes()).c_str(), text(v.sizes()).c_str());
  unit_last(fn, "v", v);
  tila_rotary_args a = rotary_args(k);
  tila_op_rows &rk = a.rows[0], &rv = a.rows[1], &rq = a.rows[2];
  if ((o[5] == Py_None) != (o[6] == Py_None)) refuse("%s: positions and inv_freq go together", fn);
  layout(fn, o[7], a);
  uint32_t turned = 0;
  if (o[5] != Py_None) {
    positions(fn, o[5], o[6], k, a);
    turned = TILA_ROWS_ROTATE;
  }
  a.amplitude = static_cast<float>(number(o[8]));
  a.eps = static_cast<float>(number(o[13]));
  const Tensor &slots = tensor(fn, "slots", o[4]);
  on_device_of(fn, "slots", slots, k);
  of_rank(fn, "slots", slots, 1);
  if (slots.scalar_type() != at::kLong && slots.scalar_type() != at::kInt)
    refuse("%s: slots must be int32 or int64, not %s", fn, c10::toString(slots.scalar_type()));
  if (slots.size(0) != k.size(0))
    refuse("%s: slots must have one slot per token, %lld, not %lld", fn, static_cast<long long>(k.size(0)),
           static_cast<long long>(slots.size(0)));
  const char *names[2] = {"k_cache", "v_cache"};
  const Tensor *caches[2];
  for (int i = 0; i < 2; ++i) {
    const Tensor &c = tensor(fn, names[i], o[2 + i]);
    on_device_of(fn, names[i], c, k);
    of_dtype(fn, names[i], c, k.scalar_type());
    of_rank(fn, names[i], c, 4);
    caches[i] = &c;
    if (c.size(2) != k.size(1) || c.size(3) != k.size(2) || c.size(0) != caches[0]->size(0) ||
        c.size(1) != caches[0]->size(1) || c.size(1) < 1 || c.size(0) > INT32_MAX || c.size(1) > INT32_MAX)
      refuse("%s: %s must be (pages, page_size, %lld, %lld), not %s", fn, names[i], static_cast<long long>(k.size(1)),
             static_cast<long long>(k.size(2)), text(c.sizes()).c_str());
    unit_last(fn, names[i], c);
    writable(fn, names[i], c);
    apart(fn, names[i], c, "k", k);
    apart(fn, names[i], c, "v", v);
    tila_op_rows &r = a.rows[i];
    r.dst = address(c);
    strides3(fn, names[i], c, r.dst_stride);
    r.flags = TILA_ROWS_PAGED;
  }
  apart(fn, "k_cache", *caches[0], "v_cache", *caches[1]);
  rk.flags |= turned;
  unrecorded(fn, {{"k", &k}, {"v", &v}, {names[0], caches[0]}, {names[1], caches[1]}});
  if (o[9] != Py_None) {
    const Tensor &w = tensor(fn, "k_weight", o[9]);
    weight(fn, "k_weight", w, k, rk);
    unrecorded(fn, {{"k_weight", &w}});
  }
  source(fn, "k", k, rk);
  source(fn, "v", v, rv);
  a.num_rows = 2;
  std::optional<Tensor> given;
  const Tensor *q = nullptr;
  if (o[10] == Py_None) {
    if (o[11] != Py_None || o[12] != Py_None) refuse("%s: q_weight and q_out need q", fn);
  } else {
    q = &tensor(fn, "q", o[10]);
    rows_shape(fn, "q", *q);
    if (q->dim() != 3 || q->device() != k.device() || q->scalar_type() != k.scalar_type() || q->size(0) != k.size(0) ||
        q->size(2) != k.size(2))
      refuse("%s: q must be (%lld, heads, %lld) of k's device and dtype", fn, static_cast<long long>(k.size(0)),
             static_cast<long long>(k.size(2)));
    unrecorded(fn, {{"q", q}});
    if (o[11] != Py_None) {
      const Tensor &w = tensor(fn, "q_weight", o[11]);
      weight(fn, "q_weight", w, *q, rq);
      unrecorded(fn, {{"q_weight", &w}});
    }
    given = result(fn, "q_out", o[12], *q, {{"q", q}},
                   {{"k", &k}, {"v", &v}, {"k_cache", caches[0]}, {"v_cache", caches[1]}});
    apart(fn, "k_cache", *caches[0], "q", *q);
    apart(fn, "v_cache", *caches[1], "q", *q);
  }
  if (q != nullptr) {
    source(fn, "q", *q, rq);
    destination(fn, "q_out", given, rq);
  }
  on_gpu(fn, "k", k);
  Tensor q_out;
  if (q != nullptr) {
    q_out = result_of(given, *q, rq);
    rq.flags |= turned;
    a.num_rows = 3;
  }
  a.slots = address(slots);
  a.slot_stride = slots.stride(0);
  a.num_slots = caches[0]->size(0) * caches[0]->size(1);
  a.page_size = static_cast<int32_t>(caches[0]->size(1));
  a.index64 |= slots.scalar_type() == at::kLong ? 2 : 0;
  run(tila_rotary_rows, "tila_rotary_rows", k, a, nullptr);
  for (const Tensor *c : caches) written(*c);
  if (given) written(q_out);
  if (q == nullptr) return Py_NewRef(Py_None);
  return given ? Py_NewRef(o[12]) : THPVariable_Wrap(std::move(q_out));
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

uint64_t indexes(const char *fn, const char *what, const Tensor &t, const Tensor &like, int rank, int64_t length) {
  on_device_of(fn, what, t, like);
  of_dtype(fn, what, t, at::kInt);
  of_rank(fn, what, t, rank);
  if (t.numel() > 1 && t.stride(-1) != 1 && t.size(-1) > 1)
    refuse("%s: the last dimension of %s must be contiguous", fn, what);
  if (length >= 0 && t.size(0) != length)
    refuse("%s: %s must have %lld entries, not %lld", fn, what, static_cast<long long>(length),
           static_cast<long long>(t.size(0)));
  return address(t);
}

// attend_shared_prefix(q, k_cache, v_cache, page_table, lengths, prefix_pages, prefix_length, query_offsets,
//                      max_queries, scale, out, return_lse, max_length)
PyObject *attend_shared_prefix(PyObject *const *o) {
  const char *fn = "attend_shared_prefix";
  const Tensor &q = tensor(fn, "q", o[0]);
  of_rank(fn, "q", q, 3);
  if (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16)
    refuse("%s: q must be float16 or bfloat16, not %s", fn, c10::toString(q.scalar_type()));
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
  if (dim % 8 != 0 || dim < 8 || dim > 256)
    refuse("%s: dim must be a multiple of 8 up to 256, not %lld", fn, static_cast<long long>(dim));
  unit_last(fn, "q", q);
  tila_attend_args a{};
  const char *names[2] = {"k_cache", "v_cache"};
  const Tensor *caches[2];
  for (int i = 0; i < 2; ++i) {
    const Tensor &c = tensor(fn, names[i], o[1 + i]);
    on_device_of(fn, names[i], c, q);
    of_dtype(fn, names[i], c, q.scalar_type());
    of_rank(fn, names[i], c, 4);
    caches[i] = &c;
    if (c.sizes() != caches[0]->sizes() || c.size(3) != dim || c.size(1) < 1 || c.size(0) > INT32_MAX ||
        c.size(1) > INT32_MAX)
      refuse("%s: %s must be (pages, page_size, kv_heads, %lld), both alike, not %s", fn, names[i],
             static_cast<long long>(dim), text(c.sizes()).c_str());
    unit_last(fn, names[i], c);
    if (address(c) % 16 != 0 || c.stride(0) % 8 != 0 || c.stride(1) % 8 != 0 || c.stride(2) % 8 != 0)
      refuse("%s: rows of %s must start on 16-byte boundaries", fn, names[i]);
    for (int d = 0; d < 3; ++d) (i == 0 ? a.k_stride : a.v_stride)[d] = c.stride(d);
  }
  const int64_t kv_heads = caches[0]->size(2), page_size = caches[0]->size(1);
  if (kv_heads < 1 || heads < 1 || heads % kv_heads != 0 || heads > INT32_MAX)
    refuse("%s: heads (%lld) must be a multiple of kv_heads (%lld)", fn, static_cast<long long>(heads),
           static_cast<long long>(kv_heads));
  const Tensor &table = tensor(fn, "page_table", o[3]);
  a.page_table = indexes(fn, "page_table", table, q, 2, -1);
  const int64_t batch = table.size(0);
  a.lengths = indexes(fn, "lengths", tensor(fn, "lengths", o[4]), q, 1, batch);
  int64_t most = 1;
  if (o[7] == Py_None) {
    if (tokens != batch)
      refuse("%s: q must have one row per sequence, %lld, not %lld (or query_offsets is needed)", fn,
             static_cast<long long>(batch), static_cast<long long>(tokens));
    if (o[8] != Py_None && whole(o[8]) != 1) refuse("%s: max_queries needs query_offsets", fn);
  } else {
    a.query_offsets = indexes(fn, "query_offsets", tensor(fn, "query_offsets", o[7]), q, 1, batch + 1);
    most = o[8] == Py_None ? tokens : whole(o[8]);
    if (o[8] != Py_None && most < 1)
      refuse("%s: max_queries must be at least 1, not %lld", fn, static_cast<long long>(most));
    most = std::max<int64_t>(1, std::min(most, tokens));
  }
  a.prefix_length = whole(o[6]);
  if (a.prefix_length < 0)
    refuse("%s: prefix_length must not be negative, is %lld", fn, static_cast<long long>(a.prefix_length));
  if (a.prefix_length > 0) {
    if (o[5] == Py_None) refuse("%s: prefix_length needs prefix_pages", fn);
    const Tensor &pages = tensor(fn, "prefix_pages", o[5]);
    a.prefix_pages = indexes(fn, "prefix_pages", pages, q, 1, -1);
    if (pages.size(0) * page_size < a.prefix_length)
      refuse("%s: prefix_pages holds %lld tokens, fewer than %lld", fn, static_cast<long long>(pages.size(0) * page_size),
             static_cast<long long>(a.prefix_length));
  }
  if (o[12] != Py_None) {
    const int64_t longest = whole(o[12]);
    if (longest < 1) refuse("%s: max_length must be at least 1, not %lld", fn, static_cast<long long>(longest));
    a.max_length = static_cast<int32_t>(std::min<int64_t>(longest, INT32_MAX));
  }
  constexpr int64_t limit = int64_t{1} << 30;
  if (tokens > limit / heads || batch > limit || table.size(1) > limit / page_size || most > limit / heads ||
      a.prefix_length > limit)
    refuse("%s: more than 2^30 rows of queries, sequences, or tokens of one sequence or of the prefix", fn);
  a.scale = o[9] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim))) : static_cast<float>(number(o[9]));
  // (base 2 in the kernels; a score times an infinite or missing scale is no number, but the wide form would have
  // taken the latter for 0)
  if (!std::isfinite(a.scale * 1.4426950408889634f))
    refuse("%s: scale must be finite, also times log2(e) in 32 bits, is %g", fn, static_cast<double>(a.scale));
  std::optional<Tensor> given =
      result(fn, "out", o[10], q, {}, {{"q", &q}, {"k_cache", caches[0]}, {"v_cache", caches[1]}});
  unrecorded(fn, {{"q", &q}, {"k_cache", caches[0]}, {"v_cache", caches[1]}});
  on_gpu(fn, "q", q);
  Tensor out = given ? *given : empty(q.sizes(), q.scalar_type(), q);
  const bool want_lse = o[11] == Py_True;
  Tensor lse;
  if (want_lse) lse = empty({tokens, heads}, at::kFloat, q);
  a.size = sizeof(a);
  a.dtype = element_type(q.scalar_type());
  a.tokens = tokens;
  a.batch = static_cast<int32_t>(batch);
  a.heads = static_cast<int32_t>(heads);
  a.kv_heads = static_cast<int32_t>(kv_heads);
  a.dim = static_cast<int32_t>(dim);
  a.page_size = static_cast<int32_t>(page_size);
  a.table_width = static_cast<int32_t>(table.size(1));
  a.max_queries = static_cast<int32_t>(most);
  a.num_pages = caches[0]->size(0);
  a.q = address(q);
  a.k_cache = address(*caches[0]);
  a.v_cache = address(*caches[1]);
  a.out = address(out);
  a.lse = want_lse ? address(lse) : 0;
  for (int d = 0; d < 2; ++d) {
    a.q_stride[d] = q.stride(d);
    a.out_stride[d] = out.stride(d);
  }
  a.table_stride = table.stride(0);
  const int index = q.get_device();
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != index) guard.set_index(index);
  a.err = error_block(index);
  a.stream = reinterpret_cast<uint64_t>(c10::cuda::getCurrentCUDAStream(index).stream());
  Tensor workspace;
  a.workspace_bytes = tila_attend_workspace(&a);
  if (a.workspace_bytes > 0) {
    workspace = empty({static_cast<int64_t>(a.workspace_bytes)}, at::kByte, q);
    a.workspace = address(workspace);
  }
  char log[512] = "";
  check_status(tila_attend_shared_prefix(&a, log, sizeof(log)), "tila_attend_shared_prefix", log);
  if (given) written(out);
  PyObject *out_o = given ? Py_NewRef(o[10]) : THPVariable_Wrap(std::move(out));
  return want_lse ? pair_of(out_o, THPVariable_Wrap(std::move(lse))) : out_o;
}

// ---------------------------------------------------------------------------
// module
// ---------------------------------------------------------------------------

// apart(name, what, a, other, b, same)
PyObject *check_apart(PyObject *const *o) {
  const char *names[3];
  for (int i = 0, at = 0; i < 3; ++i, at += i == 1 ? 1 : 2) {
    names[i] = PyUnicode_AsUTF8(o[at]);
    if (names[i] == nullptr) throw Raised();
  }
  apart(names[0], names[1], tensor(names[0], names[1], o[2]), names[2], tensor(names[0], names[2], o[4]), o[5] == Py_True);
  return Py_NewRef(Py_None);
}

// setup(prepare, check, native_error)
PyObject *setup(PyObject *const *o) {
  g_prepare = Py_NewRef(o[0]);
  g_check = Py_NewRef(o[1]);
  g_native_error = Py_NewRef(o[2]);
  return Py_NewRef(Py_None);
}

// set_error_block(index, device address, host address of the word)
PyObject *set_error_block(PyObject *const *o) {
  const int64_t index = whole(o[0]);
  if (index < 0 || index >= kMaxDevices) refuse("device index out of range");
  g_blocks[index].word = reinterpret_cast<const volatile uint32_t *>(whole(o[2]));
  g_blocks[index].address = static_cast<uint64_t>(whole(o[1]));
  return Py_NewRef(Py_None);
}

template <PyObject *(*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments are needed, not %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused &r) {
    PyErr_SetString(r.kind, r.text.c_str());
    return nullptr;
  } catch (const Raised &) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define TILA_ENTRY(F, N) \
  {#F, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr}

PyMethodDef g_methods[] = {
    TILA_ENTRY(rotate, 7),      TILA_ENTRY(norm_rotate, 11),          TILA_ENTRY(norm_rotate_backward, 13),
    TILA_ENTRY(append_paged, 14), TILA_ENTRY(attend_shared_prefix, 13), TILA_ENTRY(check_apart, 6),
    TILA_ENTRY(setup, 3),       TILA_ENTRY(set_error_block, 3),       {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ops", "Binding of tila_b200's operators.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&g_module); }
