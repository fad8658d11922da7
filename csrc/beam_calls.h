// Calls of beam search's operators (beam.cu) and of the attention over a shared prefix (shared_prefix_own.cu) from Python: the checks of
// their arguments, the memory of results and the launches in one native call.  In Python the checks, the ctypes call and five allocations of a
// selection took 29 us and those of an attention 37, several times what small ones take on the GPU, and a reordering 20 us a state.  What is
// not plainly covered (another device than the current one, steps that need a copy, gradients, states that lie between each other, arguments
// that are wrong) is answered with None and left to the Python path (ops/beam.py, ops/functional.py), which holds the rules; nothing is
// remembered between calls.
//
// Included by steps.cpp behind fp8_blocks_calls.h, whose `where`, `none` and `issued` serve here too.
#pragma once

#include <ATen/core/grad_mode.h>

namespace {

struct Beam {
  int (*select)(const void*, int, long long, long long, const void*, const void*, int, int, int, long long, long long, void*, void*, void*,
                void*, int, void*) = nullptr;
  int (*reorder)(const long long*, int, int, int, const void*, int, void*) = nullptr;
  long long (*scratch)(int, int, int, int, int, int, int, int) = nullptr;
  int (*attention)(const void*, const void*, const void*, const void*, const void*, const void*, const void*, void*, void*, int, int, int,
                   int, int, int, int, const long long*, float, int, int, void*) = nullptr;
  int max_beams = 0, max_states = 0;
} bm;

// A plain CUDA tensor of this rank on the given device.
const at::Tensor* on_device(PyObject* o, long rank, long device) {
  const at::Tensor* t = tensor(o);
  return t && t->is_cuda() && t->get_device() == device && t->dim() == rank && !t->is_conj() && !t->is_neg() ? t : nullptr;
}

constexpr double kScales[2] = {0x1p-100, 0x1p100};   // of an attention: beyond, products with scores leave 32 bits

bool wants_gradient(const at::Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

// A dense tensor in `base`'s memory from byte `at` on; an allocation of its own takes 1 us.
at::Tensor within(const at::Tensor& base, at::ScalarType type, int64_t at, at::IntArrayRef sizes) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), c10::scalarTypeToTypeMeta(type));
  impl->set_sizes_contiguous(sizes);
  impl->set_storage_offset(at / static_cast<int64_t>(c10::elementSize(type)));
  return at::Tensor(std::move(impl));
}

// beam_select(logits, scores, finished or None, eos, pad, sms, device, stream) -> (scores, parents, tokens, finished)
PyObject* beam_select(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 8 || !bm.select || !where(args + 6, &device, &stream)) return none();
  const long long eos = PyLong_AsLongLong(args[3]), pad = PyErr_Occurred() ? 0 : PyLong_AsLongLong(args[4]);
  const long sms = PyErr_Occurred() ? 0 : PyLong_AsLong(args[5]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *x = on_device(args[0], 3, device), *s = on_device(args[1], 2, device);
  const at::Tensor* f = args[2] == Py_None ? nullptr : on_device(args[2], 2, device);
  if (!x || !s || (args[2] != Py_None && !f)) Py_RETURN_NONE;
  const int64_t b = x->size(0), w = x->size(1), v = x->size(2);
  const at::ScalarType t = x->scalar_type();
  const int type = t == at::kBFloat16 ? 0 : t == at::kFloat ? 1 : t == at::kHalf ? 2 : -1;
  if (type < 0 || b < 1 || w < 1 || v < 1 || w > bm.max_beams || v > 1 << 28 || b * w >= 1 << 27 || (x->stride(2) != 1 && v > 1) ||
      s->scalar_type() != at::kFloat || s->size(0) != b || s->size(1) != w || !s->is_contiguous() ||
      (f && (f->scalar_type() != at::kBool || f->sizes() != s->sizes() || !f->is_contiguous())))
    Py_RETURN_NONE;
  HANDLE_TH_ERRORS
  const int64_t n = b * w;
  const at::Tensor all = at::empty({n * 21}, s->options().dtype(at::kByte));
  at::Tensor parents = within(all, at::kLong, 0, {b, w}), tokens = within(all, at::kLong, 8 * n, {b, w});
  at::Tensor scores = within(all, at::kFloat, 16 * n, {b, w}), finished = within(all, at::kBool, 20 * n, {b, w});
  const int rc = issued([&] {
    return bm.select(x->const_data_ptr(), type, x->stride(0), x->stride(1), s->const_data_ptr(), f ? f->const_data_ptr() : nullptr, int(b), int(w),
                     int(v), eos, pad, at_(scores), at_(parents), at_(tokens), at_(finished), int(sms), stream);
  });
  if (rc) return PyLong_FromLong(rc);
  return Py_BuildValue("(NNNN)", wrap(std::move(scores)), wrap(std::move(parents)), wrap(std::move(tokens)), wrap(std::move(finished)));
  END_HANDLE_TH_ERRORS
}

// beam_reorder(states, parents, length or None, out or None, device, stream) -> launches; states and out are lists
PyObject* beam_reorder(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 6 || !bm.reorder || !where(args + 4, &device, &stream)) return none();
  const bool whole = args[2] == Py_None, in_place = args[3] == Py_None;
  if (!PyList_Check(args[0]) || (!in_place && (!PyList_Check(args[3]) || PyList_GET_SIZE(args[3]) != PyList_GET_SIZE(args[0])))) Py_RETURN_NONE;
  const long long length = whole ? 0 : PyLong_AsLongLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* p = on_device(args[1], 2, device);
  if (!p || !p->is_contiguous() || (p->scalar_type() != at::kLong && p->scalar_type() != at::kInt) || (!whole && length < 1)) Py_RETURN_NONE;
  const int64_t b = p->size(0), w = p->size(1);
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  if (b < 1 || w < 1 || w > bm.max_beams || b > 65535 || n < 1) Py_RETURN_NONE;
  HANDLE_TH_ERRORS
  struct Span {
    long long begin, end;
    bool written;
  };
  std::vector<long long> table;
  std::vector<Span> spans;   // of what is read and written: parents too
  std::vector<const at::Tensor*> to;
  table.reserve(size_t(n) * 7);
  const auto first = reinterpret_cast<long long>(p->const_data_ptr());
  spans.push_back({first, first + b * w * static_cast<long long>(p->element_size()), false});
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor *x = tensor(PyList_GET_ITEM(args[0], i)), *y = in_place ? x : tensor(PyList_GET_ITEM(args[3], i));
    if (!x || !y || x->dim() < 2 || wants_gradient(*x) || wants_gradient(*y)) Py_RETURN_NONE;
    if (!whole && (x->dim() < 3 || x->size(2) < length)) Py_RETURN_NONE;
    if (y->sizes() != x->sizes() || y->scalar_type() != x->scalar_type()) Py_RETURN_NONE;
    const long long size = x->element_size();
    for (int j = in_place ? 1 : 0; j < 2; ++j) {   // in place the two are one, and one span
      const at::Tensor* t = j ? y : x;
      if (!t->is_cuda() || t->get_device() != device || t->size(0) != b || t->size(1) != w || t->is_conj() || t->is_neg()) Py_RETURN_NONE;
      long long step = 1;   // what a beam holds is dense, beams do not overlap
      for (int64_t d = t->dim() - 1; d >= 2; --d) {
        if (t->size(d) != 1 && t->stride(d) != step) Py_RETURN_NONE;
        step *= t->size(d);
      }
      if (step < 1 || (w > 1 && t->stride(1) < step) || (b > 1 && t->stride(0) < step) ||
          (b > 1 && w > 1 && t->stride(0) < w * t->stride(1) && t->stride(1) < b * t->stride(0)))
        Py_RETURN_NONE;
      const auto base = reinterpret_cast<long long>(t->const_data_ptr());
      spans.push_back({base, base + ((b - 1) * t->stride(0) + (w - 1) * t->stride(1) + step) * size, j == 1});
    }
    const long long inner = x->dim() > 2 ? x->size(2) : 1;
    const long long beam = x->numel() / (b * w) / inner * (whole ? inner : length) * size;
    if (beam > 1LL << 37) Py_RETURN_NONE;
    const auto dst = reinterpret_cast<long long>(at_(*y));   // first: memory that a lazy clone shares is y's own after this
    const long long row[7] = {in_place ? dst : reinterpret_cast<long long>(x->const_data_ptr()), dst, x->stride(0) * size, x->stride(1) * size,
                              y->stride(0) * size, y->stride(1) * size, beam};
    table.insert(table.end(), row, row + 7);
    to.push_back(y);
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& c) { return a.begin < c.begin; });
  long long end_any = 0, end_written = 0;   // where what began before ends
  for (const Span& s : spans) {
    if (s.begin < (s.written ? end_any : end_written)) Py_RETURN_NONE;
    end_any = std::max(end_any, s.end);
    if (s.written) end_written = std::max(end_written, s.end);
  }
  long launches = 0;
  for (Py_ssize_t i = 0; i < n; i += bm.max_states, ++launches) {
    const int rc = issued([&] {
      return bm.reorder(table.data() + 7 * i, int(std::min<Py_ssize_t>(bm.max_states, n - i)), int(b), int(w), p->const_data_ptr(),
                        p->scalar_type() == at::kLong, stream);
    });
    if (rc) return PyLong_FromLong(-rc);
  }
  for (const at::Tensor* y : to)
    if (!y->is_inference()) y->unsafeGetTensorImpl()->bump_version();
  return PyLong_FromLong(launches);
  END_HANDLE_TH_ERRORS
}

// A cache or a query as 16-byte copies take it; its steps are appended.  `one`: the first may be 0.
bool steps_of(const at::Tensor& t, bool one, long long*& steps) {
  const int64_t last = t.dim() - 1;
  if (t.numel() > 0 && ((t.stride(last) != 1) || !address(t))) return false;
  for (int64_t d = 0; d < last; ++d) {
    if (t.size(d) > 1 && t.numel() > 0 && (t.stride(d) < (one && d == 0 ? 0 : 1) || t.stride(d) % 8)) return false;
    *steps++ = t.size(d) > 1 && t.numel() > 0 ? t.stride(d) : 0;
  }
  return true;
}

// shared_prefix_attn(q, k, v, own_k, own_v, prefix_lens or None, own_rows or None, scale or None, sms, device, stream) -> ((B, W, H, hd), launches)
PyObject* shared_prefix_attn(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  long device = 0;
  void* stream = nullptr;
  if (nargs != 11 || !bm.attention || !where(args + 9, &device, &stream)) return none();
  const long sms = PyLong_AsLong(args[8]);
  double scale = PyErr_Occurred() || args[7] == Py_None ? 0.0 : PyFloat_AsDouble(args[7]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i) {
    t[i] = on_device(args[i], i < 3 ? 4 : 5, device);
    if (!t[i] || t[i]->scalar_type() != at::kBFloat16 || wants_gradient(*t[i])) Py_RETURN_NONE;
  }
  const at::Tensor &q = *t[0], &k = *t[1], &ok = *t[3];
  const at::Tensor* lens = args[5] == Py_None ? nullptr : on_device(args[5], 1, device);
  const at::Tensor* rows = args[6] == Py_None ? nullptr : on_device(args[6], 3, device);
  const int64_t b = q.size(0), w = q.size(1), h = q.size(2), hd = q.size(3), p = k.size(1), hkv = k.size(2), s = ok.size(2);
  if ((args[5] != Py_None && !lens) || (args[6] != Py_None && !rows) || b < 1 || w < 1 || h < 1 || hkv < 1 || b * w * h >= 1 << 27 || h % hkv ||
      (hd != 64 && hd != 128) || h / hkv > 128 || p > kLargest || s > kLargest || k.size(0) != b || k.size(3) != hd || k.sizes() != t[2]->sizes() ||
      ok.size(0) != b || ok.size(1) != w || ok.size(3) != hkv || ok.size(4) != hd || ok.sizes() != t[4]->sizes() ||
      (lens && (lens->scalar_type() != at::kInt || lens->size(0) != b || !lens->is_contiguous())) ||
      (rows && (rows->scalar_type() != at::kByte || rows->size(0) != b || rows->size(1) != w || rows->size(2) != s ||
                (s > 1 && rows->stride(2) != 1))))
    Py_RETURN_NONE;
  if (args[7] == Py_None) scale = 1.0 / std::sqrt(static_cast<double>(hd));
  if (!(scale >= kScales[0] && scale <= kScales[1])) Py_RETURN_NONE;
  long long steps[19], *next = steps;
  for (int i = 0; i < 5; ++i)
    if (!steps_of(*t[i], i == 1 || i == 2, next)) Py_RETURN_NONE;
  steps[17] = rows ? rows->stride(0) : 0;
  steps[18] = rows ? rows->stride(1) : 0;
  HANDLE_TH_ERRORS
  const long long bytes = bm.scratch(int(b), int(w), int(p), int(h), int(hkv), int(hd), -1, int(sms));
  if (bytes < 0) Py_RETURN_NONE;
  at::Tensor scratch, out = at::empty({b, w, h, hd}, q.options());
  if (bytes) scratch = at::empty({bytes}, q.options().dtype(at::kByte));
  const int rc = issued([&] {
    return bm.attention(q.const_data_ptr(), k.const_data_ptr(), t[2]->const_data_ptr(), ok.const_data_ptr(), t[4]->const_data_ptr(),
                        lens ? lens->const_data_ptr() : nullptr, rows ? rows->const_data_ptr() : nullptr, at_(out), bytes ? at_(scratch) : nullptr,
                        int(b), int(w), int(p), int(s), int(h), int(hkv), int(hd), steps, float(scale), -1, int(sms), stream);
  });
  return rc ? PyLong_FromLong(rc) : Py_BuildValue("(Ni)", wrap(std::move(out)), bytes ? 2 : 1);
  END_HANDLE_TH_ERRORS
}

// beam_configure(addresses of kf_beam_select, kf_beam_reorder, kf_shared_prefix_scratch, kf_shared_prefix_attn_bf16, beams and
// states that the kernels take at most)
PyObject* beam_configure(PyObject*, PyObject* args) {
  unsigned long long select = 0, reorder = 0, scratch = 0, attention = 0;
  Beam c;
  if (!PyArg_ParseTuple(args, "KKKKii", &select, &reorder, &scratch, &attention, &c.max_beams, &c.max_states)) return nullptr;
  c.select = reinterpret_cast<decltype(c.select)>(select);
  c.reorder = reinterpret_cast<decltype(c.reorder)>(reorder);
  c.scratch = reinterpret_cast<decltype(c.scratch)>(scratch);
  c.attention = reinterpret_cast<decltype(c.attention)>(attention);
  bm = c;
  Py_RETURN_NONE;
}

}  // namespace
