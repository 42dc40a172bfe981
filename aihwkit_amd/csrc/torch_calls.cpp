// The compute calls of the Python tiles on torch tensors, natively: operand checks, the output tensor, the current stream
// and the C entry point in one call.  A training step on a small tile is three such calls of a few kernels each, and
// through ctypes the Python around a call took 7 us (a third of a whole step of a 129 x 10 tile at batch 64), for the 38
// tiles of a split layer group 3 us per tile.
//
// Every function handles the plain case -- contiguous float32 tensors of the right sizes on the GPU -- and returns None
// for everything else without having done anything: the caller (rpu_base/tiles.py) then takes its general path, which
// converts what can be converted and words the errors (for the digital operators, digital/: any of their types, and matrices
// whose rows are apart).  A failing C entry point raises RuntimeError with its message, and
// so does a C++ exception on the way to it.  Pointers and streams are taken before the GIL is released: nothing between
// the two can throw.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <vector>

#include "../../include/rpu_amd.h"

namespace {

// Tensors of a function transform (torch.vmap, torch.func) or of a tracer have no storage of their own to point into.
const at::Tensor *stored(PyObject *o) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  return t.defined() && t.has_storage() && !at::isTensorSubclassLike(t) ? &t : nullptr;
}

const at::Tensor *plain(PyObject *o) {
  const at::Tensor *p = stored(o);
  if (!p) return nullptr;
  const at::Tensor &t = *p;
  if (t.scalar_type() != at::kFloat || !t.is_cuda() || !t.is_contiguous() || t.dim() < 1) return nullptr;
  return &t;
}

// a matrix with unit column stride (dense, or a column slice of a larger one)
const at::Tensor *rows(PyObject *o) {
  const at::Tensor *p = stored(o);
  if (!p) return nullptr;
  const at::Tensor &t = *p;
  if (t.scalar_type() != at::kFloat || !t.is_cuda() || t.dim() != 2) return nullptr;
  if (t.size(1) > 1 && t.stride(1) != 1) return nullptr;
  return &t;
}

const float *data(const at::Tensor &t) { return static_cast<const float *>(t.const_data_ptr()); }
float *out_data(const at::Tensor &t) { return static_cast<float *>(t.data_ptr()); }

hipStream_t stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// an entry point of the module: a C++ exception becomes a Python one, and an error of a flag without a truth value is raised
template <typename F> PyObject *guarded(F &&f) {
  try {
    PyObject *result = f();
    if (result && PyErr_Occurred()) Py_CLEAR(result);
    return result;
  } catch (const c10::Error &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// runs a C call, which does not throw (and, for a blocking call, waits for the stream), without the GIL; false: a Python
// error is set
template <typename F> bool call(F &&f, hipStream_t s, bool non_blocking) {
  int rc = 0;
  hipError_t err = hipSuccess;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  if (rc == 0 && !non_blocking) err = hipStreamSynchronize(s);
  Py_END_ALLOW_THREADS
  if (rc != 0) {
    PyErr_SetString(PyExc_RuntimeError, rpu_last_error());
    return false;
  }
  if (err != hipSuccess) {
    PyErr_SetString(PyExc_RuntimeError, hipGetErrorString(err));
    return false;
  }
  return true;
}

long integer(PyObject *o) { return PyLong_AsLong(o); }
void *pointer(PyObject *o) { return PyLong_AsVoidPtr(o); }
bool truth(PyObject *o) { return PyObject_IsTrue(o) == 1; }

// batch of a call whose vectors are the last dimension (or the first, trans); < 0: not of `expected` elements each
int64_t batch_of(const at::Tensor &t, bool trans, int64_t expected) {
  const int64_t n = trans ? t.size(0) : t.size(-1);
  if (n != expected || n <= 0) return -1;
  return t.numel() / n;
}

// matrix-vector product: (handle, input, in size, out size, bias, in_trans, out_trans, is_test, non_blocking); the sizes are
// those of the tensors (without the bias column)
template <bool FORWARD> PyObject *product(PyObject *const *a, Py_ssize_t n) {
  if (n != 9) return PyErr_Format(PyExc_TypeError, "9 arguments expected"), nullptr;
  const at::Tensor *in = plain(a[1]);
  if (!in) Py_RETURN_NONE;
  const int64_t in_size = integer(a[2]), out_size = integer(a[3]);
  const bool bias = truth(a[4]), in_trans = truth(a[5]), out_trans = truth(a[6]), is_test = truth(a[7]);
  const int64_t batch = batch_of(*in, in_trans, in_size);
  if (batch < 0 || batch > 0x7fffffff) Py_RETURN_NONE;
  at::Tensor out;
  try {
    // the input's shape with its vector dimension replaced; with mixed layouts the plain matrix
    if (in_trans == out_trans) {
      c10::SmallVector<int64_t, 6> dims(in->sizes().begin(), in->sizes().end());
      dims[out_trans ? 0 : dims.size() - 1] = out_size;
      out = at::empty(dims, in->options());
    } else {
      out = out_trans ? at::empty({out_size, batch}, in->options()) : at::empty({batch, out_size}, in->options());
    }
  } catch (...) {
    Py_RETURN_NONE; // the general path meets (and words) the same failure
  }
  rpu_tile_t *h = static_cast<rpu_tile_t *>(pointer(a[0]));
  const hipStream_t s = stream_of(*in);
  const float *src = data(*in);
  float *dst = out_data(out);
  const bool ok = call(
      [&] {
        return FORWARD ? rpu_tile_forward(h, src, dst, (int)batch, bias, in_trans, out_trans, is_test, s)
                       : rpu_tile_backward(h, src, dst, (int)batch, bias, in_trans, out_trans, s);
      },
      s, truth(a[8]));
  return ok ? THPVariable_Wrap(std::move(out)) : nullptr;
}

PyObject *forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return product<true>(a, n); });
}
PyObject *backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return product<false>(a, n); });
}

// (handle, x, d, x size, d size, bias, x_trans, d_trans, without_allocation, non_blocking) -> True, or None
PyObject *update_checked(PyObject *const *a, Py_ssize_t n) {
  if (n != 10) return PyErr_Format(PyExc_TypeError, "10 arguments expected"), nullptr;
  rpu_tile_t *h = static_cast<rpu_tile_t *>(pointer(a[0]));
  if (rpu_tile_get_learning_rate(h) == 0.0f) Py_RETURN_TRUE;
  const at::Tensor *x = plain(a[1]), *d = plain(a[2]);
  if (!x || !d) Py_RETURN_NONE;
  const bool bias = truth(a[5]), x_trans = truth(a[6]), d_trans = truth(a[7]), noalloc = truth(a[8]);
  const int64_t batch = batch_of(*x, x_trans, integer(a[3]));
  if (batch < 0 || batch > 0x7fffffff || batch_of(*d, d_trans, integer(a[4])) != batch) Py_RETURN_NONE;
  const hipStream_t s = stream_of(*x);
  const float *xp = data(*x), *dp = data(*d);
  const bool ok = call(
      [&] { return (noalloc ? rpu_tile_update_noalloc : rpu_tile_update)(h, xp, dp, (int)batch, bias, x_trans, d_trans, s); }, s,
      truth(a[9]));
  if (!ok) return nullptr;
  Py_RETURN_TRUE;
}
PyObject *update(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return update_checked(a, n); });
}

// Grouped calls.  `sizes`: bytes of int32 pairs (x_size, d_size), one per tile.
struct GroupSizes {
  const int32_t *p;
  Py_ssize_t n;
  explicit GroupSizes(PyObject *o) : p(reinterpret_cast<const int32_t *>(PyBytes_AS_STRING(o))), n(PyBytes_GET_SIZE(o) / 8) {}
  int x(Py_ssize_t i) const { return p[2 * i]; }
  int d(Py_ssize_t i) const { return p[2 * i + 1]; }
};

struct Operands {
  std::vector<at::Tensor> tensors; // kept: the caller's list may change once the GIL is released
  std::vector<const float *> ptr;
  std::vector<long> ld;
  int64_t batch = -1;
};

// pointers and row strides of a list of matrices [batch][size of tile i] (WRITTEN: a pointer to write through, for which a
// copy-on-write tensor makes its copy); false: not the plain case
template <bool WRITTEN, typename Size> bool operands(PyObject *list, Py_ssize_t n, int64_t batch, Size size, Operands &o) {
  if (!PyList_Check(list) || PyList_GET_SIZE(list) != n) return false;
  o.tensors.reserve(n);
  o.ptr.reserve(n);
  o.ld.reserve(n);
  o.batch = batch;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor *t = rows(PyList_GET_ITEM(list, i));
    if (!t) return false;
    if (o.batch < 0) o.batch = t->size(0);
    if (t->size(0) != o.batch || t->size(1) != size(i)) return false;
    o.tensors.push_back(*t);
    o.ptr.push_back(WRITTEN ? out_data(*t) : data(*t));
    o.ld.push_back(o.batch > 1 ? (long)t->stride(0) : (long)size(i));
  }
  return n > 0 && o.batch >= 0 && o.batch <= 0x7fffffff;
}

// (group, sizes, inputs, outs or None, is_test, non_blocking) -> list of outputs, or None
template <bool FORWARD> PyObject *group_product(PyObject *const *a, Py_ssize_t nargs) {
  if (nargs != 6) return PyErr_Format(PyExc_TypeError, "6 arguments expected"), nullptr;
  const GroupSizes sz(a[1]);
  Operands in, out;
  if (!operands<false>(a[2], sz.n, -1, [&](Py_ssize_t i) { return FORWARD ? sz.x(i) : sz.d(i); }, in)) Py_RETURN_NONE;
  const auto out_size = [&](Py_ssize_t i) { return FORWARD ? sz.d(i) : sz.x(i); };
  THPObjectPtr result;
  if (a[3] == Py_None) {
    result = PyList_New(sz.n);
    if (!result) return nullptr;
    for (Py_ssize_t i = 0; i < sz.n; ++i) {
      PyObject *item = nullptr;
      try {
        item = THPVariable_Wrap(at::empty({in.batch, (int64_t)out_size(i)}, in.tensors[0].options()));
      } catch (...) {
      }
      if (!item) {
        PyErr_Clear();
        Py_RETURN_NONE; // the general path meets the same failure
      }
      PyList_SET_ITEM(result.get(), i, item);
    }
  } else if (PyList_Check(a[3])) {
    result = PyList_GetSlice(a[3], 0, PyList_GET_SIZE(a[3]));
    if (!result) return nullptr;
  } else {
    Py_RETURN_NONE;
  }
  if (!operands<true>(result.get(), sz.n, in.batch, out_size, out)) Py_RETURN_NONE;
  rpu_group_t *g = static_cast<rpu_group_t *>(pointer(a[0]));
  const hipStream_t s = stream_of(in.tensors[0]);
  const bool is_test = truth(a[4]);
  const bool ok = call(
      [&] {
        float *const *o = const_cast<float *const *>(reinterpret_cast<const float *const *>(out.ptr.data()));
        return FORWARD ? rpu_group_forward_strided(g, in.ptr.data(), in.ld.data(), o, out.ld.data(), (int)in.batch, is_test, s)
                       : rpu_group_backward_strided(g, in.ptr.data(), in.ld.data(), o, out.ld.data(), (int)in.batch, s);
      },
      s, truth(a[5]));
  return ok ? result.release() : nullptr;
}

PyObject *group_forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return group_product<true>(a, n); });
}
PyObject *group_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return group_product<false>(a, n); });
}

// (group, sizes, x inputs, d inputs, non_blocking) -> True, or None
PyObject *group_update_checked(PyObject *const *a, Py_ssize_t n) {
  if (n != 5) return PyErr_Format(PyExc_TypeError, "5 arguments expected"), nullptr;
  const GroupSizes sz(a[1]);
  Operands x, d;
  if (!operands<false>(a[2], sz.n, -1, [&](Py_ssize_t i) { return sz.x(i); }, x)) Py_RETURN_NONE;
  if (!operands<false>(a[3], sz.n, x.batch, [&](Py_ssize_t i) { return sz.d(i); }, d)) Py_RETURN_NONE;
  rpu_group_t *g = static_cast<rpu_group_t *>(pointer(a[0]));
  const hipStream_t s = stream_of(x.tensors[0]);
  const bool ok = call(
      [&] { return rpu_group_update_strided(g, x.ptr.data(), x.ld.data(), d.ptr.data(), d.ld.data(), (int)x.batch, s); }, s,
      truth(a[4]));
  if (!ok) return nullptr;
  Py_RETURN_TRUE;
}
PyObject *group_update(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return group_update_checked(a, n); });
}

// ---- digital operators beside the tiles ------------------------------------------------------------------------------

int rpu_type(const at::Tensor &t) {
  switch (t.scalar_type()) {
  case at::kFloat: return RPU_F32;
  case at::kHalf: return RPU_F16;
  case at::kBFloat16: return RPU_BF16;
  default: return -1;
  }
}

// a tensor whose last dimension holds the columns and the others together the rows
struct Rows {
  const at::Tensor *t = nullptr;
  int type = -1;
  int64_t rows = 0, cols = 0;
  long ld = 0;
  bool take(PyObject *o) {
    t = stored(o);
    if (!t || !t->is_cuda() || t->dim() < 1 || (type = rpu_type(*t)) < 0) return false;
    cols = t->size(-1);
    if (cols < 1 || cols > 0x7fffffff) return false;
    rows = t->numel() / cols;
    if (rows > 0x7fffffff) return false;
    ld = (long)cols;
    if (t->dim() == 2 && t->size(0) > 1) {
      ld = (long)t->stride(0);
      return (cols == 1 || t->stride(1) == 1) && ld >= cols;
    }
    return t->is_contiguous();
  }
  bool like(const Rows &o) const { return type == o.type && t->device() == o.t->device(); }
  const void *in() const { return t ? t->const_data_ptr() : nullptr; }
  void *out() const { return t->data_ptr(); }
};

// an operand that may be None, beside `x` and of the given shape
bool take_beside(PyObject *o, const Rows &x, at::IntArrayRef shape, Rows &r) {
  if (o == Py_None) return true;
  return r.take(o) && r.like(x) && r.t->sizes() == shape;
}

// the given output, or a new tensor; false: not the plain case
bool take_out(PyObject *o, const Rows &x, at::IntArrayRef shape, at::Tensor &keep, Rows &r) {
  if (o != Py_None) {
    if (!take_beside(o, x, shape, r)) return false;
    keep = *r.t;
    return true;
  }
  keep = at::empty(shape, x.t->options().requires_grad(false));
  r.t = &keep;
  r.type = x.type;
  r.cols = keep.size(-1);
  r.rows = keep.numel() / std::max<int64_t>(r.cols, 1);
  r.ld = (long)r.cols;
  return true;
}

// a dense vector of `count` values (None: null); types: bit t allows rpu_dtype t
bool take_vector(PyObject *o, const Rows &x, int64_t count, int types, const at::Tensor *&t) {
  t = nullptr;
  if (o == Py_None) return true;
  t = stored(o);
  if (!t || !t->is_cuda() || t->device() != x.t->device() || t->numel() != count || !t->is_contiguous()) return false;
  const int type = rpu_type(*t);
  return type >= 0 && ((types >> type) & 1);
}

// (p, seed, call) given as plain numbers
bool take_drop(PyObject *p, PyObject *seed, PyObject *call, rpu_dropout_params &d) {
  if (!PyFloat_CheckExact(p) || !PyLong_CheckExact(seed) || !PyLong_CheckExact(call)) return false;
  d = {};
  d.p = PyFloat_AS_DOUBLE(p);
  const unsigned long long s = PyLong_AsUnsignedLongLong(seed), c = PyLong_AsUnsignedLongLong(call);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  if (c > 0xffffffffull || !(d.p >= 0.0 && d.p <= 1.0)) return false;
  d.seed = s;
  d.call = (uint32_t)c;
  return true;
}

PyObject *tuple_of(at::Tensor a, at::Tensor b, at::Tensor c, int n) { // an undefined tensor becomes None
  THPObjectPtr result(PyTuple_New(n));
  if (!result) return nullptr;
  at::Tensor *all[3] = {&a, &b, &c};
  for (int i = 0; i < n; ++i) {
    PyObject *item = THPVariable_Wrap(std::move(*all[i]));
    if (!item) return nullptr;
    PyTuple_SET_ITEM(result.get(), i, item);
  }
  return result.release();
}

// (x, p, seed, call, base, out, non_blocking) -> out, or None
PyObject *dropout_checked(PyObject *const *a, Py_ssize_t n) {
  if (n != 7) return PyErr_Format(PyExc_TypeError, "7 arguments expected"), nullptr;
  Rows x, base, out;
  rpu_dropout_params d;
  at::Tensor y;
  if (!x.take(a[0]) || !take_drop(a[1], a[2], a[3], d) || !take_beside(a[4], x, x.t->sizes(), base) ||
      !take_out(a[5], x, x.t->sizes(), y, out))
    Py_RETURN_NONE;
  const hipStream_t s = stream_of(*x.t);
  void *yp = out.out(); // before the pointers of operands, which it may be one of
  const void *xp = x.in(), *bp = base.in();
  const int device = x.t->device().index();
  const bool ok = call([&] { return rpu_dropout(xp, x.ld, bp, base.ld, yp, out.ld, x.type, (int)x.rows, (int)x.cols, &d, device, s); }, s, truth(a[6]));
  return ok ? THPVariable_Wrap(std::move(y)) : nullptr;
}
PyObject *dropout(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return dropout_checked(a, n); });
}

at::Tensor per_row(const Rows &x, int64_t values) { // float, of the leading dimensions of x (values < 0: those alone)
  c10::SmallVector<int64_t, 6> dims(x.t->sizes().begin(), x.t->sizes().end() - 1);
  if (values >= 0) dims.push_back(values);
  return at::empty(dims, x.t->options().dtype(at::kFloat).requires_grad(false));
}

// (x, weight, bias, eps, out, non_blocking) -> (y, mean, rstd), or None
PyObject *layer_norm_checked(PyObject *const *a, Py_ssize_t n) {
  if (n != 6) return PyErr_Format(PyExc_TypeError, "6 arguments expected"), nullptr;
  Rows x, out;
  at::Tensor y;
  const at::Tensor *w, *b;
  if (!x.take(a[0]) || !PyFloat_CheckExact(a[3])) Py_RETURN_NONE;
  const int types = 1 << RPU_F32 | 1 << x.type;
  if (!take_vector(a[1], x, x.cols, types, w) || !take_vector(a[2], x, x.cols, types, b) || (w && b && w->scalar_type() != b->scalar_type()) ||
      !take_out(a[4], x, x.t->sizes(), y, out))
    Py_RETURN_NONE;
  at::Tensor mean = per_row(x, -1), rstd = per_row(x, -1);
  const hipStream_t s = stream_of(*x.t);
  const float eps = (float)PyFloat_AS_DOUBLE(a[3]);
  const int w_type = w ? rpu_type(*w) : b ? rpu_type(*b) : RPU_F32, device = x.t->device().index();
  void *yp = out.out();
  const void *xp = x.in(), *wp = w ? w->const_data_ptr() : nullptr, *bp = b ? b->const_data_ptr() : nullptr;
  float *mp = out_data(mean), *rp = out_data(rstd);
  const bool ok = call(
      [&] { return rpu_layer_norm(xp, x.ld, wp, bp, w_type, yp, out.ld, mp, rp, x.type, (int)x.rows, (int)x.cols, eps, device, s); }, s, truth(a[5]));
  return ok ? tuple_of(std::move(y), std::move(mean), std::move(rstd), 3) : nullptr;
}
PyObject *layer_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return layer_norm_checked(a, n); });
}

at::Tensor scratch_of(const Rows &x, size_t bytes) { return at::empty({(int64_t)bytes}, x.t->options().dtype(at::kByte).requires_grad(false)); }

// (d, x, mean, rstd, weight, base, out, non_blocking) -> (dx, dweight, dbias), or None
PyObject *layer_norm_backward_checked(PyObject *const *a, Py_ssize_t n) {
  if (n != 8) return PyErr_Format(PyExc_TypeError, "8 arguments expected"), nullptr;
  Rows d, x, base, out;
  at::Tensor dx, dw, db, scratch;
  const at::Tensor *mean, *rstd, *w;
  if (!x.take(a[1]) || !d.take(a[0]) || !d.like(x) || d.t->sizes() != x.t->sizes()) Py_RETURN_NONE;
  if (!take_vector(a[2], x, x.rows, 1 << RPU_F32, mean) || !take_vector(a[3], x, x.rows, 1 << RPU_F32, rstd) || !mean || !rstd ||
      !take_vector(a[4], x, x.cols, 1 << RPU_F32 | 1 << x.type, w) || !take_beside(a[5], x, x.t->sizes(), base) ||
      !take_out(a[6], x, x.t->sizes(), dx, out))
    Py_RETURN_NONE;
  size_t bytes = 0;
  if (w) {
    dw = at::empty(w->sizes(), w->options().requires_grad(false));
    db = at::empty(w->sizes(), w->options().requires_grad(false));
    bytes = rpu_layer_norm_backward_scratch((int)x.rows, (int)x.cols);
    scratch = scratch_of(x, bytes);
  }
  const hipStream_t s = stream_of(*x.t);
  const int device = x.t->device().index(), w_type = w ? rpu_type(*w) : RPU_F32;
  void *dxp = out.out(), *dwp = w ? dw.data_ptr() : nullptr, *dbp = w ? db.data_ptr() : nullptr, *sp = w ? scratch.data_ptr() : nullptr;
  const void *dp = d.in(), *xp = x.in(), *bp = base.in(), *wp = w ? w->const_data_ptr() : nullptr;
  const float *mp = data(*mean), *rp = data(*rstd);
  const bool ok = call(
      [&] {
        return rpu_layer_norm_backward(dp, d.ld, xp, x.ld, mp, rp, wp, w_type, bp, base.ld, dxp, out.ld, dwp, dbp, x.type, (int)x.rows, (int)x.cols, sp,
                                       bytes, device, s);
      },
      s, truth(a[7]));
  return ok ? tuple_of(std::move(dx), std::move(dw), std::move(db), 3) : nullptr;
}
PyObject *layer_norm_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return layer_norm_backward_checked(a, n); });
}

const at::Tensor *index_of(PyObject *o) {
  const at::Tensor *t = stored(o);
  return t && t->is_cuda() && t->scalar_type() == at::kInt && t->is_contiguous() && t->numel() <= 0x7fffffff ? t : nullptr;
}

// The matrices of adapters and the rows that they are beside.
struct AdapterCall {
  rpu_adapters w{};
  Rows x;
  // a, b, scale, x: [n][rank][in], [n][out][rank], [n], rows of in values
  bool take(PyObject *a, PyObject *b, PyObject *scale, PyObject *rows) {
    const at::Tensor *at = stored(a), *bt = stored(b), *st = stored(scale);
    if (!at || !bt || !st || !x.take(rows)) return false;
    if (at->dim() != 3 || bt->dim() != 3 || st->dim() != 1 || !at->is_contiguous() || !bt->is_contiguous() || !st->is_contiguous()) return false;
    const auto device = x.t->device();
    if (at->device() != device || bt->device() != device || st->device() != device) return false;
    const int type = rpu_type(*at);
    if (type < 0 || rpu_type(*bt) != type || st->scalar_type() != at::kFloat) return false;
    if (bt->size(0) != at->size(0) || st->size(0) != at->size(0) || bt->size(2) != at->size(1) || at->size(2) != x.cols) return false;
    if (at->size(0) > 0x7fffffff || at->size(1) > 0x7fffffff || bt->size(1) > 0x7fffffff) return false;
    w.a_dev = at->const_data_ptr();
    w.b_dev = bt->const_data_ptr();
    w.scale_dev = data(*st);
    w.n = (int)at->size(0);
    w.rank = (int)at->size(1);
    w.in_size = (int)at->size(2);
    w.out_size = (int)bt->size(1);
    w.w_dtype = type;
    return true;
  }
};

// the plan of an index; undefined: not the plain case
at::Tensor plan_for(const at::Tensor &index, int64_t n) {
  const size_t bytes = n >= 1 && n <= RPU_ADAPTER_MAX ? rpu_adapter_plan_bytes((int)index.numel(), (int)n) : 0;
  return bytes ? at::empty({(int64_t)bytes}, index.options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
}

// (index, n adapters) -> the plan (bytes on the GPU), or None
PyObject *adapter_plan_checked(PyObject *const *a, Py_ssize_t n) {
  if (n != 2) return PyErr_Format(PyExc_TypeError, "2 arguments expected"), nullptr;
  const at::Tensor *index = index_of(a[0]);
  if (!index) Py_RETURN_NONE;
  const long adapters = integer(a[1]);
  if (adapters < 0) PyErr_Clear(); // beyond a long: the caller words it
  at::Tensor plan = plan_for(*index, adapters);
  if (!plan.defined()) Py_RETURN_NONE;
  const hipStream_t s = stream_of(*index);
  const int32_t *ip = static_cast<const int32_t *>(index->const_data_ptr());
  void *pp = plan.data_ptr();
  const int rows = (int)index->numel(), device = index->device().index();
  const size_t bytes = (size_t)plan.numel();
  const bool ok = call([&] { return rpu_adapter_plan(ip, rows, (int)adapters, pp, bytes, device, s); }, s, true);
  return ok ? THPVariable_Wrap(std::move(plan)) : nullptr;
}
PyObject *adapter_plan(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return adapter_plan_checked(a, n); });
}

// The rows of a call: a plan of as many rows and adapters (checked by the caller), or an index, which is grouped first unless its rows are
// few.
struct GroupedRows {
  const at::Tensor *index = nullptr;
  at::Tensor plan;
  bool make = false;
  bool take(PyObject *index_or_none, PyObject *plan_or_none, const AdapterCall &c, int64_t few) {
    if (plan_or_none != Py_None) {
      const at::Tensor *p = stored(plan_or_none);
      if (!p || !p->is_cuda() || p->device() != c.x.t->device() || !p->is_contiguous()) return false;
      plan = *p;
      return true;
    }
    index = index_of(index_or_none);
    if (!index || index->device() != c.x.t->device() || index->numel() != c.x.rows) return false;
    if (index->numel() <= few) return true;
    plan = plan_for(*index, c.w.n);
    make = true;
    return plan.defined();
  }
};

// (a, b, scale, x, index, plan, base, out, return_hidden, p, seed, call, non_blocking) -> (y, hidden or None), or None
PyObject *adapter_forward_checked(PyObject *const *a, Py_ssize_t n) {
  if (n != 13) return PyErr_Format(PyExc_TypeError, "13 arguments expected"), nullptr;
  AdapterCall c;
  Rows base, out;
  rpu_dropout_params d;
  GroupedRows g;
  at::Tensor y, hidden;
  if (!c.take(a[0], a[1], a[2], a[3]) || !take_drop(a[9], a[10], a[11], d) || !g.take(a[4], a[5], c, RPU_ADAPTER_FEW_ROWS)) Py_RETURN_NONE;
  c10::SmallVector<int64_t, 6> dims(c.x.t->sizes().begin(), c.x.t->sizes().end());
  dims.back() = c.w.out_size;
  if (!take_beside(a[6], c.x, dims, base) || !take_out(a[7], c.x, dims, y, out)) Py_RETURN_NONE;
  const bool wanted = truth(a[8]);
  if (wanted || g.plan.defined()) hidden = per_row(c.x, c.w.rank);
  const hipStream_t s = stream_of(*c.x.t);
  const int rows = (int)c.x.rows, device = c.x.t->device().index();
  const int32_t *ip = g.index ? static_cast<const int32_t *>(g.index->const_data_ptr()) : nullptr;
  void *pp = g.plan.defined() ? g.plan.data_ptr() : nullptr, *yp = out.out();
  const size_t bytes = g.plan.defined() ? (size_t)g.plan.nbytes() : 0;
  const void *xp = c.x.in(), *bp = base.in();
  float *hp = hidden.defined() ? out_data(hidden) : nullptr;
  const bool ok = call(
      [&] {
        if (g.make)
          if (const int rc = rpu_adapter_plan(ip, rows, c.w.n, pp, bytes, device, s)) return rc;
        return rpu_adapter_forward(&c.w, xp, c.x.ld, ip, pp, bytes, &d, bp, base.ld, yp, out.ld, hp, c.x.type, rows, device, s);
      },
      s, truth(a[12]));
  return ok ? tuple_of(std::move(y), wanted ? std::move(hidden) : at::Tensor(), {}, 2) : nullptr;
}
PyObject *adapter_forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return adapter_forward_checked(a, n); });
}

// (a, b, scale, d, x, index, plan, hidden, base, out, p, seed, call, non_blocking) -> (dx, da, db), or None
PyObject *adapter_backward_checked(PyObject *const *a, Py_ssize_t n) {
  if (n != 14) return PyErr_Format(PyExc_TypeError, "14 arguments expected"), nullptr;
  AdapterCall c;
  Rows dy, base, out;
  rpu_dropout_params d;
  GroupedRows g;
  at::Tensor dx;
  if (!c.take(a[0], a[1], a[2], a[4]) || !take_drop(a[10], a[11], a[12], d) || !g.take(a[5], a[6], c, -1)) Py_RETURN_NONE;
  c10::SmallVector<int64_t, 6> dims(c.x.t->sizes().begin(), c.x.t->sizes().end());
  dims.back() = c.w.out_size;
  const at::Tensor *hidden;
  if (!dy.take(a[3]) || !dy.like(c.x) || dy.t->sizes() != at::IntArrayRef(dims) || !take_vector(a[7], c.x, c.x.rows * c.w.rank, 1 << RPU_F32, hidden) || !hidden ||
      !take_beside(a[8], c.x, c.x.t->sizes(), base) || !take_out(a[9], c.x, c.x.t->sizes(), dx, out))
    Py_RETURN_NONE;
  const at::Tensor &wa = *stored(a[0]), &wb = *stored(a[1]);
  at::Tensor da = at::empty(wa.sizes(), wa.options().requires_grad(false)), db = at::empty(wb.sizes(), wb.options().requires_grad(false));
  const size_t scratch_bytes = rpu_adapter_backward_scratch(&c.w, (int)c.x.rows);
  at::Tensor scratch = scratch_of(c.x, scratch_bytes);
  const hipStream_t s = stream_of(*c.x.t);
  const int rows = (int)c.x.rows, device = c.x.t->device().index();
  const int32_t *ip = g.index ? static_cast<const int32_t *>(g.index->const_data_ptr()) : nullptr;
  void *pp = g.plan.data_ptr(), *dxp = out.out(), *dap = da.data_ptr(), *dbp = db.data_ptr(), *sp = scratch.data_ptr();
  const size_t bytes = (size_t)g.plan.nbytes();
  const void *dp = dy.in(), *xp = c.x.in(), *bp = base.in();
  const float *hp = data(*hidden);
  const bool ok = call(
      [&] {
        if (g.make)
          if (const int rc = rpu_adapter_plan(ip, rows, c.w.n, pp, bytes, device, s)) return rc;
        return rpu_adapter_backward(&c.w, dp, dy.ld, xp, c.x.ld, hp, pp, bytes, &d, bp, base.ld, dxp, out.ld, dap, dbp, c.x.type, rows, sp, scratch_bytes,
                                    device, s);
      },
      s, truth(a[13]));
  return ok ? tuple_of(std::move(dx), std::move(da), std::move(db), 3) : nullptr;
}
PyObject *adapter_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&] { return adapter_backward_checked(a, n); });
}

PyMethodDef methods[] = {
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)), METH_FASTCALL, nullptr},
    {"backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(backward)), METH_FASTCALL, nullptr},
    {"update", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(update)), METH_FASTCALL, nullptr},
    {"group_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(group_forward)), METH_FASTCALL, nullptr},
    {"group_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(group_backward)), METH_FASTCALL, nullptr},
    {"group_update", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(group_update)), METH_FASTCALL, nullptr},
    {"dropout", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dropout)), METH_FASTCALL, nullptr},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm)), METH_FASTCALL, nullptr},
    {"layer_norm_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm_backward)), METH_FASTCALL, nullptr},
    {"adapter_plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adapter_plan)), METH_FASTCALL, nullptr},
    {"adapter_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adapter_forward)), METH_FASTCALL, nullptr},
    {"adapter_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adapter_backward)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "rpu_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit_rpu_torch() { return PyModule_Create(&module); }
