// Calls of the block-scaled fp8 operators (fp8_blocks.cu, gemm_fp8_blocks_tcgen05.cu) from Python: the checks of their arguments, the
// output's memory and the launch in one native call.  In Python the checks of a product took 11 us and its ctypes call 5, more than most
// products of few tokens take on the GPU: 19 us with the output's memory, and 6 so; a norm 21 and 9, a cast 15 and 7.  What is not plainly
// covered (another device than the current one, pitches that need a copy, sizes of zero, arguments that are wrong) is answered with None and
// left to the Python path (ops/fp8_blocks.py), which holds the rules; nothing is remembered between calls.  A layer's forward pass and its
// gradients are one call each: 999 tokens of 768 columns to 2304 with all gradients took 240 us call by call, and 205 so (84 of them are those of
// a node that does nothing, between autograd's threads).
//
// Included by steps.cpp, whose `tensor` tells plain tensors from wrappers.
#pragma once

namespace {

struct Fp8Blocks {
  int (*gemm)(const void*, const void*, const void*, const void*, void*, int, int, int, long long, long long, long long, long long, long long, int,
              int, int, int, int, void*) = nullptr;
  int (*norm)(const void*, const void*, const void*, void*, void*, void*, long long, void*, long long, int, int, double, void*) = nullptr;
  int (*cast)(const void*, int, int, long long, const void*, const void*, int, int, void*, long long, void*, long long, void*, long long, void*,
              long long, void*) = nullptr;
  int (*values)(const void*, long long, const void*, long long, int, int, int, void*, void*) = nullptr;
  int (*norm_grads)(const void*, const void*, const void*, const void*, const void*, void*, void*, void*, int, int, int, void*) = nullptr;
  int (*norm_grads_blocks)(int, int, int) = nullptr;
} f8;

constexpr long long kLargest = 0x7fff0000;  // kernels add a few blocks to an index in 32 bits

// A plain dense CUDA tensor of this type and rank on the given device.
const at::Tensor* dense(PyObject* o, at::ScalarType type, long rank, long device) {
  const at::Tensor* t = tensor(o);
  return t && t->is_cuda() && t->get_device() == device && t->scalar_type() == type && t->dim() == rank && !t->is_conj() && !t->is_neg() ? t : nullptr;
}

// Values and scale bytes as the kernels' bulk copies take them, with at least one value.
bool operand(PyObject* values, PyObject* scales, long device, const at::Tensor*& q, const at::Tensor*& s) {
  q = dense(values, at::kByte, 2, device);
  s = dense(scales, at::kByte, 2, device);
  if (!q || !s) return false;
  const int64_t rows = q->size(0), k = q->size(1);
  return rows > 0 && k > 0 && rows <= kLargest && k <= kLargest && s->size(0) == (k + 127) / 128 && s->size(1) == rows && q->stride(1) == 1 &&
         s->stride(1) == 1 && q->stride(0) >= k && s->stride(0) >= rows && q->stride(0) % 16 == 0 && s->stride(0) % 16 == 0 && address(*q) && address(*s);
}

bool flag(PyObject* o, int* value) {
  if (o != Py_True && o != Py_False) return false;
  *value = o == Py_True;
  return true;
}

// What the last arguments of a call say: the current device, its stream.
bool where(PyObject* const* args, long* device, void** stream) {
  *device = PyLong_AsLong(args[0]);
  *stream = reinterpret_cast<void*>(PyLong_AsLongLong(args[1]));
  return !PyErr_Occurred();
}

template <class Call>
int issued(Call&& call) {
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = call();
  Py_END_ALLOW_THREADS
  return rc;
}

void* at_(const at::Tensor& t) { return t.mutable_data_ptr(); }

// Values with rows on 128 bytes, scale bytes with rows on 16.
struct Buffers {
  at::Tensor values, scales;
  Buffers(int64_t rows, int64_t cols, const at::TensorOptions& o)
      : values(at::empty_strided({rows, cols}, {(cols + 127) / 128 * 128, 1}, o)),
        scales(at::empty_strided({(cols + 127) / 128, rows}, {(rows + 15) / 16 * 16, 1}, o)) {}
};

// ------------------------------------------------------------------ the launches, of arguments that have been checked; 0 or an error code
int product(const at::Tensor& qa, const at::Tensor& sa, int ea, const at::Tensor& qb, const at::Tensor& sb, int eb, const at::Tensor& out, int accumulate,
            long sms, void* stream) {
  return issued([&] {
    return f8.gemm(qa.const_data_ptr(), sa.const_data_ptr(), qb.const_data_ptr(), sb.const_data_ptr(), at_(out), int(qa.size(0)), int(qb.size(0)),
                   int(qa.size(1)), qa.stride(0), sa.stride(0), qb.stride(0), sb.stride(0), out.stride(0), out.scalar_type() == at::kFloat, ea, eb,
                   accumulate, int(sms), stream);
  });
}

// x, or x * gain * rstd[:, None] with both, to the row-major and the transposed copy (either null)
int cast(const at::Tensor& x, const at::Tensor* rstd, const at::Tensor* gain, int e5m2, int square, Buffers* a, Buffers* b, void* stream) {
  return issued([&] {
    return f8.cast(x.const_data_ptr(), int(x.size(0)), int(x.size(1)), x.stride(0), rstd ? rstd->const_data_ptr() : nullptr,
                   gain ? gain->const_data_ptr() : nullptr, e5m2, square, a ? at_(a->values) : nullptr, a ? a->values.stride(0) : 0,
                   a ? at_(a->scales) : nullptr, a ? a->scales.stride(0) : 0, b ? at_(b->values) : nullptr, b ? b->values.stride(0) : 0,
                   b ? at_(b->scales) : nullptr, b ? b->scales.stride(0) : 0, stream);
  });
}

int norm(const at::Tensor& x, const at::Tensor* residual, const at::Tensor& gain, double eps, const at::Tensor* t, const at::Tensor& rstd, Buffers& h,
         void* stream) {
  return issued([&] {
    return f8.norm(x.const_data_ptr(), residual ? residual->const_data_ptr() : nullptr, gain.const_data_ptr(), t ? at_(*t) : nullptr, at_(rstd),
                   at_(h.values), h.values.stride(0), at_(h.scales), h.scales.stride(0), int(x.size(0)), int(x.size(1)), eps, stream);
  });
}

// (partial sums) -> dx, dgain
int gradients(const at::Tensor& dh, const at::Tensor& t, const at::Tensor& gain, const at::Tensor& rstd, const at::Tensor* dt, const at::Tensor& dx,
              const at::Tensor& dgain, long sms, void* stream) {
  const int rows = int(t.size(0)), d = int(t.size(1));
  const at::Tensor partial = at::empty({f8.norm_grads_blocks(rows, d, int(sms)), d}, rstd.options());
  return issued([&] {
    return f8.norm_grads(dh.const_data_ptr(), t.const_data_ptr(), gain.const_data_ptr(), rstd.const_data_ptr(), dt ? dt->const_data_ptr() : nullptr,
                         at_(dx), at_(partial), at_(dgain), rows, d, int(sms), stream);
  });
}

// ------------------------------------------------------------------ checks
// A matrix that the cast takes as it is.
bool castable(const at::Tensor* x) {
  return x && x->size(0) > 0 && x->size(1) > 0 && x->size(0) <= kLargest && x->size(1) <= kLargest && x->stride(1) == 1 && x->stride(0) >= x->size(1);
}
// Rows that the norm's kernels take as they are, and a gain for them.
bool rows_of(const at::Tensor* x, const at::Tensor* gain) {
  if (!x || !gain) return false;
  const int64_t rows = x->size(0), d = x->size(1);
  return rows > 0 && rows <= kLargest && d > 0 && d % 8 == 0 && d <= 32768 && gain->size(0) == d && x->is_contiguous() && gain->is_contiguous() &&
         address(*x) && address(*gain);
}
bool like(const at::Tensor* a, const at::Tensor& x) { return a && a->sizes() == x.sizes() && a->is_contiguous() && address(*a); }
// None, or a matrix (m, n) to be written.
bool output(PyObject* o, at::ScalarType type, int64_t m, int64_t n, long device, const at::Tensor*& to) {
  to = o == Py_None ? nullptr : dense(o, type, 2, device);
  return o == Py_None || (to && to->size(0) == m && to->size(1) == n && to->stride(1) == 1 && to->stride(0) >= n);
}

PyObject* none() {
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}
PyObject* wrap(at::Tensor&& t) { return t.defined() ? THPVariable_Wrap(std::move(t)) : Py_NewRef(Py_None); }

// ------------------------------------------------------------------ calls
// fp8_mm(a values, a scales, a e5m2, b values, b scales, b e5m2, out or None, accumulate, f32, sms, device, stream) -> out (M, N), bf16 or fp32
PyObject* fp8_mm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 12 || !f8.gemm || !where(args + 10, &device, &stream)) return none();
  const long sms = PyLong_AsLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *qa, *sa, *qb, *sb, *to;
  int ea = 0, eb = 0, accumulate = 0, f32 = 0;
  if (!operand(args[0], args[1], device, qa, sa) || !operand(args[3], args[4], device, qb, sb) || qa->size(1) != qb->size(1) ||
      !flag(args[2], &ea) || !flag(args[5], &eb) || !flag(args[7], &accumulate) || !flag(args[8], &f32))
    return none();
  const at::ScalarType type = f32 ? at::kFloat : at::kBFloat16;
  if (!output(args[6], type, qa->size(0), qb->size(0), device, to) || (!to && accumulate)) return none();
  HANDLE_TH_ERRORS
  at::Tensor out = to ? *to : at::empty({qa->size(0), qb->size(0)}, qa->options().dtype(type));
  const int rc = product(*qa, *sa, ea, *qb, *sb, eb, out, accumulate, sms, stream);
  if (rc) return PyLong_FromLong(rc);
  if (!to) return THPVariable_Wrap(std::move(out));
  // what is kept by a tensor's version (saved for a gradient, 8-bit copies of a weight) learns of the write
  if (!to->is_inference()) to->unsafeGetTensorImpl()->bump_version();
  return Py_NewRef(args[6]);
  END_HANDLE_TH_ERRORS
}

// fp8_add_rmsnorm(x, residual or None, gain, eps, device, stream) -> (x + residual or None, rstd, values, scales)
PyObject* fp8_add_rmsnorm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 6 || !f8.norm || !where(args + 4, &device, &stream)) return none();
  const double eps = PyFloat_AsDouble(args[3]);
  if (PyErr_Occurred()) return nullptr;
  const bool add = args[1] != Py_None;
  const at::Tensor *x = dense(args[0], at::kBFloat16, 2, device), *r = add ? dense(args[1], at::kBFloat16, 2, device) : nullptr;
  const at::Tensor* gain = dense(args[2], at::kBFloat16, 1, device);
  if (!rows_of(x, gain) || (add && !like(r, *x))) return none();
  HANDLE_TH_ERRORS
  at::Tensor t, rstd = at::empty({x->size(0)}, x->options().dtype(at::kFloat));
  if (add) t = at::empty(x->sizes(), x->options());
  Buffers h(x->size(0), x->size(1), x->options().dtype(at::kByte));
  const int rc = norm(*x, r, *gain, eps, add ? &t : nullptr, rstd, h, stream);
  if (rc) return PyLong_FromLong(rc);
  return Py_BuildValue("(NNNN)", wrap(std::move(t)), wrap(std::move(rstd)), wrap(std::move(h.values)), wrap(std::move(h.scales)));
  END_HANDLE_TH_ERRORS
}

// fp8_cast(x, e5m2, square, want_row, want_t, rstd or None, gain or None, device, stream) -> (values, scales, transposed values, transposed
// scales), None where not wanted; with rstd and gain of x * gain * rstd[:, None]
PyObject* fp8_cast(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 9 || !f8.cast || !where(args + 7, &device, &stream)) return none();
  int e5m2, square, row, tr;
  const at::Tensor *x = dense(args[0], at::kBFloat16, 2, device), *rstd = nullptr, *gain = nullptr;
  if (!castable(x) || !flag(args[1], &e5m2) || !flag(args[2], &square) || !flag(args[3], &row) || !flag(args[4], &tr) || (!row && !tr)) return none();
  if (args[5] != Py_None) {
    rstd = dense(args[5], at::kFloat, 1, device);
    gain = dense(args[6], at::kBFloat16, 1, device);
    if (!rstd || !gain || square || e5m2 || row || rstd->size(0) != x->size(0) || gain->size(0) != x->size(1) || !rstd->is_contiguous() ||
        !gain->is_contiguous())
      return none();
  }
  HANDLE_TH_ERRORS
  const at::TensorOptions o = x->options().dtype(at::kByte);
  std::optional<Buffers> a, b;
  if (row) a.emplace(x->size(0), x->size(1), o);
  if (tr) b.emplace(x->size(1), x->size(0), o);
  const int rc = cast(*x, rstd, gain, e5m2, square, a ? &*a : nullptr, b ? &*b : nullptr, stream);
  if (rc) return PyLong_FromLong(rc);
  auto give = [](std::optional<Buffers>& v, bool scales) { return v ? wrap(std::move(scales ? v->scales : v->values)) : Py_NewRef(Py_None); };
  return Py_BuildValue("(NNNN)", give(a, false), give(a, true), give(b, false), give(b, true));
  END_HANDLE_TH_ERRORS
}

// fp8_values(values, scales, e5m2, device, stream) -> bf16
PyObject* fp8_values(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 5 || !f8.values || !where(args + 3, &device, &stream)) return none();
  const at::Tensor *q, *s;
  int e5m2 = 0;
  if (!operand(args[0], args[1], device, q, s) || !flag(args[2], &e5m2)) return none();
  HANDLE_TH_ERRORS
  at::Tensor out = at::empty(q->sizes(), q->options().dtype(at::kBFloat16));
  const int rc = issued([&] {
    return f8.values(q->const_data_ptr(), q->stride(0), s->const_data_ptr(), s->stride(0), int(q->size(0)), int(q->size(1)), e5m2, at_(out), stream);
  });
  return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// norm_grads(dh (fp32), t, gain, rstd, dt or None, sms, device, stream) -> (dt + RMSNorm'(dh), gradient of the gain), both bf16
PyObject* norm_grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 8 || !f8.norm_grads || !where(args + 6, &device, &stream)) return none();
  const long sms = PyLong_AsLong(args[5]);
  if (PyErr_Occurred()) return nullptr;
  const bool add = args[4] != Py_None;
  const at::Tensor *dh = dense(args[0], at::kFloat, 2, device), *t = dense(args[1], at::kBFloat16, 2, device);
  const at::Tensor *gain = dense(args[2], at::kBFloat16, 1, device), *rstd = dense(args[3], at::kFloat, 1, device);
  const at::Tensor* dt = add ? dense(args[4], at::kBFloat16, 2, device) : nullptr;
  if (!rows_of(t, gain) || !like(dh, *t) || !rstd || rstd->size(0) != t->size(0) || !rstd->is_contiguous() || (add && !like(dt, *t))) return none();
  HANDLE_TH_ERRORS
  at::Tensor dx = at::empty(t->sizes(), t->options()), dgain = at::empty({t->size(1)}, t->options());
  const int rc = gradients(*dh, *t, *gain, *rstd, dt, dx, dgain, sms, stream);
  return rc ? PyLong_FromLong(rc) : Py_BuildValue("(NN)", wrap(std::move(dx)), wrap(std::move(dgain)));
  END_HANDLE_TH_ERRORS
}

// fp8_norm_linear(x, residual or None, gain, eps, weight values, weight scales, sms, device, stream) -> (x + residual or None, rstd, y): the norm and
// the product of a layer
PyObject* fp8_norm_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 9 || !f8.norm || !where(args + 7, &device, &stream)) return none();
  const double eps = PyFloat_AsDouble(args[3]);
  const long sms = PyErr_Occurred() ? 0 : PyLong_AsLong(args[6]);
  if (PyErr_Occurred()) return nullptr;
  const bool add = args[1] != Py_None;
  const at::Tensor *x = dense(args[0], at::kBFloat16, 2, device), *r = add ? dense(args[1], at::kBFloat16, 2, device) : nullptr;
  const at::Tensor *gain = dense(args[2], at::kBFloat16, 1, device), *qw, *sw;
  if (!rows_of(x, gain) || (add && !like(r, *x)) || !operand(args[4], args[5], device, qw, sw) || qw->size(1) != x->size(1)) return none();
  HANDLE_TH_ERRORS
  at::Tensor t, rstd = at::empty({x->size(0)}, x->options().dtype(at::kFloat)), y = at::empty({x->size(0), qw->size(0)}, x->options());
  if (add) t = at::empty(x->sizes(), x->options());
  Buffers h(x->size(0), x->size(1), x->options().dtype(at::kByte));
  int rc = norm(*x, r, *gain, eps, add ? &t : nullptr, rstd, h, stream);
  if (!rc) rc = product(h.values, h.scales, 0, *qw, *sw, 0, y, 0, sms, stream);
  return rc ? PyLong_FromLong(rc) : Py_BuildValue("(NNN)", wrap(std::move(t)), wrap(std::move(rstd)), wrap(std::move(y)));
  END_HANDLE_TH_ERRORS
}

// fp8_norm_linear_grads(dy, dt or None, t, gain, rstd, transposed weight values or None, its scales, dw or None, accumulate, sms, device, stream) ->
// (gradient of t, of the gain), None without a weight; dw (+)= the gradient of the weight.  The gradients of a layer.
PyObject* fp8_norm_linear_grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 12 || !f8.norm_grads || !where(args + 10, &device, &stream)) return none();
  const long sms = PyLong_AsLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  const bool add = args[1] != Py_None, need_h = args[5] != Py_None, need_w = args[7] != Py_None;
  const at::Tensor *dy = dense(args[0], at::kBFloat16, 2, device), *dt = add ? dense(args[1], at::kBFloat16, 2, device) : nullptr;
  const at::Tensor *t = dense(args[2], at::kBFloat16, 2, device), *gain = dense(args[3], at::kBFloat16, 1, device);
  const at::Tensor *rstd = dense(args[4], at::kFloat, 1, device), *qw = nullptr, *sw = nullptr, *dw = nullptr;
  int accumulate = 0;
  if (!castable(dy) || !rows_of(t, gain) || !castable(t) || t->size(0) != dy->size(0) || !rstd || rstd->size(0) != t->size(0) ||
      !rstd->is_contiguous() || (add && !like(dt, *t)) || !(need_h || need_w) || !flag(args[8], &accumulate) ||
      (need_h && (!operand(args[5], args[6], device, qw, sw) || qw->size(0) != t->size(1) || qw->size(1) != dy->size(1))) ||
      !output(args[7], at::kBFloat16, dy->size(1), t->size(1), device, dw))
    return none();
  HANDLE_TH_ERRORS
  const at::TensorOptions bytes = t->options().dtype(at::kByte);
  const int64_t rows = t->size(0), d = t->size(1), n = dy->size(1);
  std::optional<Buffers> g, gt;
  if (need_h) g.emplace(rows, n, bytes);
  if (need_w) gt.emplace(n, rows, bytes);
  int rc = cast(*dy, nullptr, nullptr, 0, 0, g ? &*g : nullptr, gt ? &*gt : nullptr, stream);
  at::Tensor dx, dgain;
  if (need_h && !rc) {
    const at::Tensor dh = at::empty({rows, d}, rstd->options());
    dx = at::empty({rows, d}, t->options());
    dgain = at::empty({d}, t->options());
    rc = product(g->values, g->scales, 0, *qw, *sw, 0, dh, 0, sms, stream);
    if (!rc) rc = gradients(dh, *t, *gain, *rstd, dt, dx, dgain, sms, stream);
  }
  if (need_w && !rc) {
    Buffers h(d, rows, bytes);
    rc = cast(*t, rstd, gain, 0, 0, nullptr, &h, stream);
    if (!rc) rc = product(gt->values, gt->scales, 0, h.values, h.scales, 0, *dw, accumulate, sms, stream);
  }
  return rc ? PyLong_FromLong(rc) : Py_BuildValue("(NN)", wrap(std::move(dx)), wrap(std::move(dgain)));
  END_HANDLE_TH_ERRORS
}

// fp8_linear_grads(dy, transposed weight values or None, its scales, transposed x values or None, its scales, dw or None, accumulate, sms, device,
// stream) -> gradient of x, None without a weight (True then); dw (+)= the gradient of the weight
PyObject* fp8_linear_grads(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 10 || !f8.cast || !where(args + 8, &device, &stream)) return none();
  const long sms = PyLong_AsLong(args[7]);
  if (PyErr_Occurred()) return nullptr;
  const bool need_x = args[1] != Py_None, need_w = args[5] != Py_None;
  const at::Tensor *dy = dense(args[0], at::kBFloat16, 2, device), *qw = nullptr, *sw = nullptr, *qx = nullptr, *sx = nullptr, *dw = nullptr;
  int accumulate = 0;
  if (!castable(dy) || !(need_x || need_w) || !flag(args[6], &accumulate) ||
      (need_x && (!operand(args[1], args[2], device, qw, sw) || qw->size(1) != dy->size(1))) ||
      (need_w && (!operand(args[3], args[4], device, qx, sx) || qx->size(1) != dy->size(0) ||
                  !output(args[5], at::kBFloat16, dy->size(1), qx->size(0), device, dw))))
    return none();
  HANDLE_TH_ERRORS
  const at::TensorOptions bytes = dy->options().dtype(at::kByte);
  const int64_t rows = dy->size(0), n = dy->size(1);
  std::optional<Buffers> g, gt;
  if (need_x) g.emplace(rows, n, bytes);
  if (need_w) gt.emplace(n, rows, bytes);
  int rc = cast(*dy, nullptr, nullptr, 0, 0, g ? &*g : nullptr, gt ? &*gt : nullptr, stream);
  at::Tensor dx;
  if (need_x && !rc) {
    dx = at::empty({rows, qw->size(0)}, dy->options());
    rc = product(g->values, g->scales, 0, *qw, *sw, 0, dx, 0, sms, stream);
  }
  if (need_w && !rc) rc = product(gt->values, gt->scales, 0, *qx, *sx, 0, *dw, accumulate, sms, stream);
  if (rc) return PyLong_FromLong(rc);
  return need_x ? THPVariable_Wrap(std::move(dx)) : Py_NewRef(Py_True);
  END_HANDLE_TH_ERRORS
}

// fp8_configure(addresses of kf_gemm_fp8_blocks, kf_add_rmsnorm_fp8_blocks, kf_fp8_blocks_cast_bf16, kf_fp8_blocks_values_bf16,
// kf_norm_grads_f32, kf_norm_grads_blocks)
PyObject* fp8_configure(PyObject*, PyObject* args) {
  unsigned long long gemm = 0, norm = 0, cast = 0, values = 0, grads = 0, grads_blocks = 0;
  if (!PyArg_ParseTuple(args, "KKKKKK", &gemm, &norm, &cast, &values, &grads, &grads_blocks)) return nullptr;
  f8.gemm = reinterpret_cast<decltype(f8.gemm)>(gemm);
  f8.norm = reinterpret_cast<decltype(f8.norm)>(norm);
  f8.cast = reinterpret_cast<decltype(f8.cast)>(cast);
  f8.values = reinterpret_cast<decltype(f8.values)>(values);
  f8.norm_grads = reinterpret_cast<decltype(f8.norm_grads)>(grads);
  f8.norm_grads_blocks = reinterpret_cast<decltype(f8.norm_grads_blocks)>(grads_blocks);
  Py_RETURN_NONE;
}

}  // namespace
