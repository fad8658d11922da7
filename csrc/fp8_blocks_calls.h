// Calls of the block-scaled fp8 operators (fp8_blocks.cu, gemm_fp8_blocks_tcgen05.cu) from Python: the checks of their arguments, the
// output's memory and the launch in one native call.  In Python the checks of a product took 11 us and its ctypes call 5, more than most
// products of few tokens take on the GPU: 19 us with the output's memory, and 6 so; a norm 21 and 9, a cast 15 and 7.  What is not plainly
// covered (another device than the current one, pitches that need a copy, sizes of zero, arguments that are wrong) is answered with None and
// left to the Python path (ops/fp8_blocks.py), which holds the rules; nothing is remembered between calls.
//
// Included by steps.cpp, whose `tensor` tells plain tensors from wrappers.
#pragma once

namespace {

struct Fp8Blocks {
  int (*gemm)(const void*, const void*, const void*, const void*, void*, int, int, int, long long, long long, long long, long long, long long, int,
              int, int, int, int, void*) = nullptr;
  int (*norm)(const void*, const void*, const void*, void*, void*, void*, long long, void*, long long, int, int, float, void*) = nullptr;
  int (*cast)(const void*, int, int, long long, const void*, const void*, int, int, void*, long long, void*, long long, void*, long long, void*,
              long long, void*) = nullptr;
  int (*values)(const void*, long long, const void*, long long, int, int, int, void*, void*) = nullptr;
  int (*norm_grads)(const void*, const void*, const void*, const void*, const void*, void*, void*, void*, int, int, int, void*) = nullptr;
  int (*norm_grads_blocks)(int, int, int) = nullptr;
} f8;

constexpr long long kLargest = 0x7fffffff;

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

// fp8_mm(a values, a scales, a e5m2, b values, b scales, b e5m2, out or None, accumulate, f32, sms, device, stream) -> out (M, N), bf16 or fp32
PyObject* fp8_mm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 12 || !f8.gemm || !where(args + 10, &device, &stream)) return PyErr_Occurred() ? nullptr : Py_NewRef(Py_None);
  const long sms = PyLong_AsLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *qa, *sa, *qb, *sb;
  int ea = 0, eb = 0, accumulate = 0, f32 = 0;
  if (!operand(args[0], args[1], device, qa, sa) || !operand(args[3], args[4], device, qb, sb) || qa->size(1) != qb->size(1) ||
      !flag(args[2], &ea) || !flag(args[5], &eb) || !flag(args[7], &accumulate) || !flag(args[8], &f32))
    Py_RETURN_NONE;
  const at::ScalarType type = f32 ? at::kFloat : at::kBFloat16;
  const at::Tensor* to = args[6] == Py_None ? nullptr : dense(args[6], type, 2, device);
  if (args[6] == Py_None ? accumulate != 0
                         : !to || to->size(0) != qa->size(0) || to->size(1) != qb->size(0) || to->stride(1) != 1 || to->stride(0) < to->size(1))
    Py_RETURN_NONE;
  HANDLE_TH_ERRORS
  at::Tensor out = to ? *to : at::empty({qa->size(0), qb->size(0)}, qa->options().dtype(type));
  const int rc = issued([&] {
    return f8.gemm(qa->const_data_ptr(), sa->const_data_ptr(), qb->const_data_ptr(), sb->const_data_ptr(), at_(out), int(qa->size(0)), int(qb->size(0)),
                   int(qa->size(1)), qa->stride(0), sa->stride(0), qb->stride(0), sb->stride(0), out.stride(0), f32, ea, eb, accumulate, int(sms), stream);
  });
  return rc ? PyLong_FromLong(rc) : to ? Py_NewRef(args[6]) : THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// fp8_add_rmsnorm(x, residual or None, gain, eps, device, stream) -> (x + residual or None, rstd, values, scales)
PyObject* fp8_add_rmsnorm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 6 || !f8.norm || !where(args + 4, &device, &stream)) return PyErr_Occurred() ? nullptr : Py_NewRef(Py_None);
  const double eps = PyFloat_AsDouble(args[3]);
  if (PyErr_Occurred()) return nullptr;
  const bool add = args[1] != Py_None;
  const at::Tensor *x = dense(args[0], at::kBFloat16, 2, device), *r = add ? dense(args[1], at::kBFloat16, 2, device) : nullptr;
  const at::Tensor* gain = dense(args[2], at::kBFloat16, 1, device);
  if (!x || !gain || (add && !r)) Py_RETURN_NONE;
  const int64_t rows = x->size(0), d = x->size(1);
  if (rows < 1 || rows > kLargest || d < 8 || d % 8 || d > 32768 || gain->size(0) != d || !x->is_contiguous() || !gain->is_contiguous() || !address(*x) ||
      !address(*gain) || (add && (r->sizes() != x->sizes() || !r->is_contiguous() || !address(*r))))
    Py_RETURN_NONE;
  HANDLE_TH_ERRORS
  at::Tensor t, rstd = at::empty({rows}, x->options().dtype(at::kFloat));
  if (add) t = at::empty({rows, d}, x->options());
  Buffers h(rows, d, x->options().dtype(at::kByte));
  const int rc = issued([&] {
    return f8.norm(x->const_data_ptr(), add ? r->const_data_ptr() : nullptr, gain->const_data_ptr(), add ? at_(t) : nullptr, at_(rstd), at_(h.values),
                   h.values.stride(0), at_(h.scales), h.scales.stride(0), int(rows), int(d), float(eps), stream);
  });
  if (rc) return PyLong_FromLong(rc);
  PyObject* first = add ? THPVariable_Wrap(std::move(t)) : Py_NewRef(Py_None);
  return Py_BuildValue("(NNNN)", first, THPVariable_Wrap(std::move(rstd)), THPVariable_Wrap(std::move(h.values)), THPVariable_Wrap(std::move(h.scales)));
  END_HANDLE_TH_ERRORS
}

// fp8_cast(x, e5m2, square, want_row, want_t, rstd or None, gain or None, device, stream) -> (values, scales, transposed values, transposed
// scales), None where not wanted; with rstd and gain of x * rstd[:, None] * gain
PyObject* fp8_cast(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 9 || !f8.cast || !where(args + 7, &device, &stream)) return PyErr_Occurred() ? nullptr : Py_NewRef(Py_None);
  int e5m2, square, row, tr;
  const at::Tensor* x = dense(args[0], at::kBFloat16, 2, device);
  if (!x || !flag(args[1], &e5m2) || !flag(args[2], &square) || !flag(args[3], &row) || !flag(args[4], &tr)) Py_RETURN_NONE;
  const int64_t rows = x->size(0), cols = x->size(1);
  if ((!row && !tr) || rows < 1 || cols < 1 || rows > 128 * 65535 || cols > kLargest || x->stride(1) != 1 || x->stride(0) < cols) Py_RETURN_NONE;
  const at::Tensor *rstd = nullptr, *gain = nullptr;
  if (args[5] != Py_None) {
    rstd = dense(args[5], at::kFloat, 1, device);
    gain = dense(args[6], at::kBFloat16, 1, device);
    if (!rstd || !gain || square || e5m2 || rstd->size(0) != rows || gain->size(0) != cols || !rstd->is_contiguous() || !gain->is_contiguous()) Py_RETURN_NONE;
  }
  HANDLE_TH_ERRORS
  const at::TensorOptions o = x->options().dtype(at::kByte);
  std::optional<Buffers> a, b;
  if (row) a.emplace(rows, cols, o);
  if (tr) b.emplace(cols, rows, o);
  const int rc = issued([&] {
    return f8.cast(x->const_data_ptr(), int(rows), int(cols), x->stride(0), rstd ? rstd->const_data_ptr() : nullptr,
                   gain ? gain->const_data_ptr() : nullptr, e5m2, square, a ? at_(a->values) : nullptr,
                   a ? a->values.stride(0) : 0, a ? at_(a->scales) : nullptr, a ? a->scales.stride(0) : 0, b ? at_(b->values) : nullptr,
                   b ? b->values.stride(0) : 0, b ? at_(b->scales) : nullptr, b ? b->scales.stride(0) : 0, stream);
  });
  if (rc) return PyLong_FromLong(rc);
  auto give = [](std::optional<Buffers>& v, bool scales) {
    return v ? THPVariable_Wrap(std::move(scales ? v->scales : v->values)) : Py_NewRef(Py_None);
  };
  return Py_BuildValue("(NNNN)", give(a, false), give(a, true), give(b, false), give(b, true));
  END_HANDLE_TH_ERRORS
}

// fp8_values(values, scales, e5m2, device, stream) -> bf16
PyObject* fp8_values(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 5 || !f8.values || !where(args + 3, &device, &stream)) return PyErr_Occurred() ? nullptr : Py_NewRef(Py_None);
  const at::Tensor *q, *s;
  int e5m2 = 0;
  if (!operand(args[0], args[1], device, q, s) || !flag(args[2], &e5m2)) Py_RETURN_NONE;
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
  if (nargs != 8 || !f8.norm_grads || !where(args + 6, &device, &stream)) return PyErr_Occurred() ? nullptr : Py_NewRef(Py_None);
  const long sms = PyLong_AsLong(args[5]);
  if (PyErr_Occurred()) return nullptr;
  const bool add = args[4] != Py_None;
  const at::Tensor *dh = dense(args[0], at::kFloat, 2, device), *t = dense(args[1], at::kBFloat16, 2, device);
  const at::Tensor *gain = dense(args[2], at::kBFloat16, 1, device), *rstd = dense(args[3], at::kFloat, 1, device);
  const at::Tensor* dt = add ? dense(args[4], at::kBFloat16, 2, device) : nullptr;
  if (!dh || !t || !gain || !rstd || (add && !dt)) Py_RETURN_NONE;
  const int64_t rows = t->size(0), d = t->size(1);
  if (rows < 1 || rows > kLargest || d < 8 || d % 8 || d > 8192 || dh->sizes() != t->sizes() || gain->size(0) != d || rstd->size(0) != rows ||
      !dh->is_contiguous() || !t->is_contiguous() || !gain->is_contiguous() || !rstd->is_contiguous() || !address(*dh) || !address(*t) ||
      !address(*gain) || (add && (dt->sizes() != t->sizes() || !dt->is_contiguous() || !address(*dt))))
    Py_RETURN_NONE;
  HANDLE_TH_ERRORS
  at::Tensor partial = at::empty({f8.norm_grads_blocks(int(rows), int(d), int(sms)), d}, rstd->options()), dx = at::empty({rows, d}, t->options());
  at::Tensor dgain = at::empty({d}, t->options());
  const int rc = issued([&] {
    return f8.norm_grads(dh->const_data_ptr(), t->const_data_ptr(), gain->const_data_ptr(), rstd->const_data_ptr(), add ? dt->const_data_ptr() : nullptr,
                         at_(dx), at_(partial), at_(dgain), int(rows), int(d), int(sms), stream);
  });
  return rc ? PyLong_FromLong(rc) : Py_BuildValue("(NN)", THPVariable_Wrap(std::move(dx)), THPVariable_Wrap(std::move(dgain)));
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
