// torch_calls.cc — the int8 layer's calls on torch tensors, without an interpreter between
// their checks.
//
// A call of one row takes less time on the GPU than its checks, allocations and argument
// conversions take in Python. Every function here looks whether its arguments are what
// such a call has (plain tensors of one CUDA device, rows that the kernels can read as they
// are), makes the outputs, calls the C ABI on torch's current stream and returns the
// outputs. Of anything else, and of a call that the C ABI refuses, it returns None: the Python
// form then converts what it can and names the reason where it cannot.
//
// Host time of a call of one row, in us, with the Python forms' in brackets: norm with
// residual 5.8 (12.7), product 4.4 (9.5), back to values 4.5 (7.8), rotation of queries and
// keys 5.1 (11.5), SiLU product 4.3 (9.8), as it is 4.4 (8.7); 2.7 of it is the launch.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/mlb200.h"

namespace {

constexpr long long kMostInt = 0x7fffffff;

struct Rows {  // [rows, n], or [rows, heads, dim] with n = heads * dim
  void* p = nullptr;
  long long stride = 0;
  int rows = 0, n = 0;
};

bool tensor(PyObject* o, const at::Tensor** t) {
  if (!THPVariable_CheckExact(o)) return false;
  *t = &THPVariable_Unpack(o);
  // a negated view's memory holds the values' negatives
  return (*t)->is_cuda() && (*t)->layout() == at::kStrided && !(*t)->is_neg();
}

bool on(const at::Tensor& t, int device) { return t.get_device() == device; }

// MLB_ACT_* of a tensor's type, or -1.
int act_type(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? MLB_ACT_F32
                                       : t.scalar_type() == at::kBFloat16 ? MLB_ACT_BF16 : -1;
}

// Rows of consecutive elements; the innermost dimensions of a third one together.
bool rows_of(const at::Tensor& t, int dims, Rows* r) {
  if (t.dim() != dims) return false;
  const auto size = t.sizes(), stride = t.strides();
  long long n = size[1];
  if (dims == 3) n *= size[2];
  if (size[0] <= 0 || n <= 0 || size[0] > kMostInt || n > kMostInt) return false;
  if (size[dims - 1] > 1 && stride[dims - 1] != 1) return false;
  if (dims == 3 && size[1] > 1 && stride[1] != size[2]) return false;
  if (size[0] > 1 && stride[0] < n) return false;
  *r = {t.data_ptr(), size[0] > 1 ? (long long)stride[0] : n, (int)size[0], (int)n};
  return true;
}

// Rows of codes that start at 16-byte boundaries.
bool codes_of(const at::Tensor& t, int device, Rows* r) {
  if (t.scalar_type() != at::kChar || !on(t, device) || !rows_of(t, 2, r)) return false;
  if (r->rows == 1) r->stride = ((long long)r->n + 15) / 16 * 16;
  return r->stride % 16 == 0 && reinterpret_cast<uintptr_t>(r->p) % 16 == 0;
}

bool floats_of(const at::Tensor& t, int device, int n, float** p) {
  if (t.scalar_type() != at::kFloat || !on(t, device) || t.dim() != 1 || t.sizes()[0] != n ||
      !t.is_contiguous())
    return false;
  *p = static_cast<float*>(t.data_ptr());
  return true;
}

at::Tensor new_rows(const at::Tensor& like, int rows, long long n, at::ScalarType type) {
  return at::empty({rows, n}, like.options().dtype(type));
}
at::Tensor new_codes(const at::Tensor& like, int rows, int n, long long* width) {
  *width = ((long long)n + 15) / 16 * 16;
  const auto options = like.options().dtype(at::kChar);
  return *width == n ? at::empty({rows, n}, options)
                     : at::empty_strided({rows, n}, {*width, 1}, options);
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

PyObject* none() { Py_RETURN_NONE; }

PyObject* wrapped(const at::Tensor& t) { return THPVariable_Wrap(t); }
template <class... T>
PyObject* wrapped(const at::Tensor& first, const at::Tensor& second, const T&... more) {
  PyObject* items[] = {THPVariable_Wrap(first), THPVariable_Wrap(second),
                       THPVariable_Wrap(more)...};
  constexpr Py_ssize_t n = 2 + sizeof...(T);
  bool whole = true;
  for (PyObject* o : items) whole = whole && o;
  PyObject* r = whole ? PyTuple_New(n) : nullptr;
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (r)
      PyTuple_SET_ITEM(r, i, items[i]);
    else
      Py_XDECREF(items[i]);
  }
  return r;
}

// Runs a call without the interpreter's lock, as a launch may wait for the device and the
// device for another thread's work: f checks, allocates and launches, and returns whether
// it did. What torch throws (no memory) is the Python form's to meet again. Returns the
// outputs, one alone or a tuple.
template <class F, class... T>
PyObject* attempt(F&& f, const T&... outputs) {
  PyThreadState* thread = PyEval_SaveThread();
  bool done;
  try {
    done = f();
  } catch (...) {
    done = false;
  }
  PyEval_RestoreThread(thread);
  if (!done) Py_RETURN_NONE;
  return wrapped(outputs...);
}

bool whole_number(PyObject* o, int* v) {
  const long long wide = PyLong_AsLongLong(o);
  *v = (int)wide;
  if (!PyErr_Occurred()) return *v == wide;
  PyErr_Clear();
  return false;
}
bool real_number(PyObject* o, double* v) {
  *v = PyFloat_AsDouble(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}

// int8_linear(x, x_scale, w, w_scale, bias or None, MLB_ACT_*) -> out
PyObject* int8_linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  const at::Tensor *x, *xs, *w, *ws, *b = nullptr;
  int act;
  if (n_args != 6 || !tensor(a[0], &x) || !tensor(a[1], &xs) || !tensor(a[2], &w) ||
      !tensor(a[3], &ws) || (a[4] != Py_None && !tensor(a[4], &b)) || !whole_number(a[5], &act))
    return none();
  at::Tensor out;
  const auto call = [&] {
    const int device = x->get_device();
    Rows xr, wr;
    float *xp, *wp, *bp = nullptr;
    if (!codes_of(*x, device, &xr) || !codes_of(*w, device, &wr) || xr.n != wr.n ||
        !floats_of(*xs, device, xr.rows, &xp) || !floats_of(*ws, device, wr.rows, &wp) ||
        (b && !floats_of(*b, device, wr.rows, &bp)))
      return false;
    out = new_rows(*xs, xr.rows, wr.rows, act == MLB_ACT_BF16 ? at::kBFloat16 : at::kFloat);
    if (mlb_int8_linear(static_cast<const int8_t*>(xr.p), xr.stride, xp, xr.rows, xr.n,
                        static_cast<const int8_t*>(wr.p), wr.stride, wp, wr.rows, bp, act,
                        out.data_ptr(), wr.rows, device, stream_of(device)) != MLB_OK)
      return false;
    return true;
  };
  return attempt(call, out);
}

// int8_dequantize(codes, scales, MLB_ACT_*) -> values
PyObject* int8_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  const at::Tensor *c, *s;
  int act;
  if (n_args != 3 || !tensor(a[0], &c) || !tensor(a[1], &s) || !whole_number(a[2], &act))
    return none();
  at::Tensor out;
  const auto call = [&] {
    const int device = c->get_device();
    Rows r;
    float* sp;
    if (!codes_of(*c, device, &r) || !floats_of(*s, device, r.rows, &sp)) return false;
    out = new_rows(*s, r.rows, r.n, act == MLB_ACT_BF16 ? at::kBFloat16 : at::kFloat);
    if (mlb_int8_dequantize(static_cast<const int8_t*>(r.p), r.stride, sp, r.rows, r.n, act,
                            out.data_ptr(), r.n, device, stream_of(device)) != MLB_OK)
      return false;
    return true;
  };
  return attempt(call, out);
}

// int8_quantize(x) -> (codes, scales)
PyObject* int8_quantize(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  const at::Tensor* x;
  if (n_args != 1 || !tensor(a[0], &x)) return none();
  at::Tensor codes, scales;
  const auto call = [&] {
    const int device = x->get_device(), act = act_type(*x);
    Rows r;
    if (act < 0 || !rows_of(*x, 2, &r)) return false;
    long long width;
    codes = new_codes(*x, r.rows, r.n, &width);
    scales = at::empty({r.rows}, x->options().dtype(at::kFloat));
    if (mlb_int8_quantize(act, r.p, r.stride, r.rows, r.n, static_cast<int8_t*>(codes.data_ptr()),
                          width, static_cast<float*>(scales.data_ptr()), device,
                          stream_of(device)) != MLB_OK)
      return false;
    return true;
  };
  return attempt(call, codes, scales);
}

// silu_mul_int8(gate, up) -> (codes, scales)
PyObject* silu_mul_int8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  const at::Tensor *g, *u;
  if (n_args != 2 || !tensor(a[0], &g) || !tensor(a[1], &u)) return none();
  at::Tensor codes, scales;
  const auto call = [&] {
    const int device = g->get_device(), act = act_type(*g);
    Rows gr, ur;
    if (act < 0 || act_type(*u) != act || !on(*u, device) || !rows_of(*g, 2, &gr) ||
        !rows_of(*u, 2, &ur) || gr.rows != ur.rows || gr.n != ur.n)
      return false;
    long long width;
    codes = new_codes(*g, gr.rows, gr.n, &width);
    scales = at::empty({gr.rows}, g->options().dtype(at::kFloat));
    if (mlb_silu_mul_int8(act, gr.p, gr.stride, ur.p, ur.stride, gr.rows, gr.n,
                          static_cast<int8_t*>(codes.data_ptr()), width,
                          static_cast<float*>(scales.data_ptr()), device,
                          stream_of(device)) != MLB_OK)
      return false;
    return true;
  };
  return attempt(call, codes, scales);
}

// rmsnorm_int8(x, w, eps, residual or None) -> (codes, scales) or (codes, scales, sum)
PyObject* rmsnorm_int8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  const at::Tensor *x, *w, *res = nullptr;
  double eps;
  if (n_args != 4 || !tensor(a[0], &x) || !tensor(a[1], &w) || !real_number(a[2], &eps) ||
      (a[3] != Py_None && !tensor(a[3], &res)))
    return none();
  at::Tensor codes, scales, sum;
  const auto call = [&] {
    const int device = x->get_device(), act = act_type(*x);
    Rows xr, rr;
    float* wp;
    if (act < 0 || !rows_of(*x, 2, &xr) || !floats_of(*w, device, xr.n, &wp)) return false;
    if (res && (act_type(*res) != act || !on(*res, device) || !rows_of(*res, 2, &rr) ||
                rr.rows != xr.rows || rr.n != xr.n))
      return false;
    long long width;
    codes = new_codes(*x, xr.rows, xr.n, &width);
    scales = at::empty({xr.rows}, x->options().dtype(at::kFloat));
    if (res) sum = new_rows(*x, xr.rows, xr.n, x->scalar_type());
    if (mlb_rmsnorm_int8(act, xr.p, xr.stride, rr.p, rr.stride, wp, xr.rows, xr.n, (float)eps,
                         res ? sum.data_ptr() : nullptr, xr.n,
                         static_cast<int8_t*>(codes.data_ptr()), width,
                         static_cast<float*>(scales.data_ptr()), device,
                         stream_of(device)) != MLB_OK)
      return false;
    return true;
  };
  return res ? attempt(call, codes, scales, sum) : attempt(call, codes, scales);
}

// rope_rows(q, k, positions, frequencies, amplitude, rope_type) -> (q_out, k_out)
PyObject* rope_rows(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  const at::Tensor *q, *k, *pos, *f;
  double amplitude;
  int type;
  if (n_args != 6 || !tensor(a[0], &q) || !tensor(a[1], &k) || !tensor(a[2], &pos) ||
      !tensor(a[3], &f) || !real_number(a[4], &amplitude) || !whole_number(a[5], &type))
    return none();
  at::Tensor q_out, k_out;
  const auto call = [&] {
    const int device = f->get_device(), act = act_type(*q);
    Rows qr, kr;
    if (f->scalar_type() != at::kDouble || f->dim() != 1 || f->sizes()[0] > kMostInt / 2 ||
        !f->is_contiguous())
      return false;
    if (act < 0 || act_type(*k) != act || !on(*q, device) || !on(*k, device) ||
        !on(*pos, device) || !rows_of(*q, 3, &qr) || !rows_of(*k, 3, &kr) || qr.rows != kr.rows ||
        q->sizes()[2] != k->sizes()[2] || pos->scalar_type() != at::kInt || pos->dim() != 1 ||
        pos->sizes()[0] != qr.rows || !pos->is_contiguous())
      return false;
    q_out = at::empty(q->sizes(), q->options());
    k_out = at::empty(k->sizes(), k->options());
    if (mlb_rope_rows(act, qr.p, qr.stride, (int)q->sizes()[1], kr.p, kr.stride,
                      (int)k->sizes()[1], (int)q->sizes()[2], 2 * (int)f->sizes()[0],
                      static_cast<const int*>(pos->data_ptr()),
                      static_cast<const double*>(f->data_ptr()), (float)amplitude, type, qr.rows,
                      q_out.data_ptr(), qr.n, k_out.data_ptr(), kr.n, device,
                      stream_of(device)) != MLB_OK)
      return false;
    return true;
  };
  return attempt(call, q_out, k_out);
}

#define CALL(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CALL(int8_linear), CALL(int8_dequantize), CALL(int8_quantize),
                         CALL(silu_mul_int8), CALL(rmsnorm_int8), CALL(rope_rows),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr,
                      nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
