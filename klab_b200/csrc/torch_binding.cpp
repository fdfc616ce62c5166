// Host path of the batched operators for torch callers: a CPython module that checks tensors, allocates results, takes
// torch's current stream and calls the C entry points, in a few microseconds. A decode step makes several of these calls per
// layer, and through ctypes each takes 17 to 23 us of host time, more than its kernels at ordinary batch sizes.
//
// Every function answers None for a call that is not one of its plain cases (an argument out of order, a module that is
// not loaded yet); the Python wrapper then does its own checks, which raise or take the ctypes path. Nothing is decided
// here that the wrappers do not decide alike. The entry points come as addresses from _native's library, so that the two
// paths use one library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>

#include "klab_b200.h"

namespace {

using at::Tensor;

struct Entries {
  decltype(&klab_kv_build_step) build_step = nullptr;
  decltype(&klab_kv_store) store = nullptr;
  decltype(&klab_kv_read) read = nullptr;
  decltype(&klab_kv_attention) attention = nullptr, attention_new = nullptr;
  decltype(&klab_kv_attention_scratch) attention_scratch = nullptr;
  decltype(&klab_adapter_linear) adapter = nullptr;
  decltype(&klab_adapter_scratch) adapter_scratch = nullptr;
} g_entry;

bool g_ready[64];

struct Failed {
  int code;
};

constexpr int kMaxRequests = KLAB_KV_MAX_REQUESTS, kMaxNew = KLAB_KV_MAX_NEW, kMaxGroup = KLAB_KV_MAX_GROUP;
constexpr int kMaxRank = KLAB_ADAPTER_MAX_RANK;

// ---------------------------------------------------------------- arguments

bool tensor_of(PyObject* o, const Tensor*& t) {
  if (!THPVariable_Check(o)) return false;
  t = &THPVariable_Unpack(o);
  return t->defined() && t->layout() == at::kStrided && !t->requires_grad();
}

bool int_of(PyObject* o, long long low, long long high, long long& v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  v = PyLong_AsLongLongAndOverflow(o, &over);
  return !over && v >= low && v <= high;
}

bool on(const Tensor& t, int index) { return t.is_cuda() && t.device().index() == index; }

bool ints(const Tensor& t, int index) { return t.scalar_type() == at::kInt && on(t, index) && t.is_contiguous(); }

bool aligned(const Tensor& t, uintptr_t to) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (to - 1)) == 0; }

int dtype_code(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? KLAB_DT_BF16 : t.scalar_type() == at::kHalf ? KLAB_DT_F16 : -1;
}

struct Span {
  uintptr_t begin, end;
};

Span span(const Tensor& t) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
  long long last = 1;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {p, p + static_cast<uintptr_t>(last) * t.element_size()};
}

bool apart(const Tensor& a, const Tensor& b) {
  const Span x = span(a), y = span(b);
  return x.end <= y.begin || y.end <= x.begin;
}

bool page_size_ok(long long n) { return n >= 16 && n <= 1024 && (n & (n - 1)) == 0; }

// pages [num_pages, kv_heads, page bytes] for heads of `dim`.
bool pages_of(const Tensor& t, long long dim, int index, long long& num, long long& kv_heads, long long& page_size) {
  if ((dim != 64 && dim != 128 && dim != 256) || t.scalar_type() != at::kByte || t.dim() != 3 || !on(t, index) ||
      !t.is_contiguous() || !aligned(t, 16))
    return false;
  num = t.size(0), kv_heads = t.size(1), page_size = t.size(2) * 8 / (9 * dim);
  return num > 0 && kv_heads > 0 && page_size * dim * 9 == t.size(2) * 8 && page_size_ok(page_size) &&
         num * page_size < (1ll << 31);
}

// ---------------------------------------------------------------- launch

// The device, its current stream, and what was used there.
class Launch {
 public:
  explicit Launch(int index) : guard_(static_cast<c10::DeviceIndex>(index)), stream_(c10::cuda::getCurrentCUDAStream(index)) {}
  void* stream() const { return stream_.stream(); }
  void done(int rc) const {
    if (rc) throw Failed{rc};
  }
  // The caching allocator learns which stream used a tensor (not while a graph is captured).
  template <typename... T>
  void used(const T&... t) const {
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream_.stream(), &capturing) != cudaSuccess || capturing != cudaStreamCaptureStatusNone) return;
    (c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), stream_), ...);
  }

 private:
  c10::cuda::CUDAGuard guard_;
  c10::cuda::CUDAStream stream_;
};

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int index) {
  return at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(index)), std::nullopt);
}

// Elements [at, at + n) of a flat tensor as a tensor of their own on the same storage.
Tensor part(const Tensor& t, int64_t at, int64_t n) {
  Tensor p = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
  p.unsafeGetTensorImpl()->set_storage_offset(at);
  p.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return p;
}

PyObject* none() { Py_RETURN_NONE; }

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Failed& e) {
    return PyLong_FromLong(e.code);  // the wrapper raises it
  } catch (const c10::OutOfMemoryError&) {
    return none();  // nothing was launched: the wrapper allocates, and raises torch's own error where it cannot
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

int ready_index(const Tensor& t) {
  if (!t.is_cuda()) return -1;
  const int index = t.device().index();
  return index >= 0 && index < 64 && g_ready[index] ? index : -1;
}

// ---------------------------------------------------------------- functions

// (new_tokens, lengths, table, free_pages, free_count, page_size, max_tokens, inplace) -> 7 tensors
PyObject* build_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *fresh, *lengths, *table, *pages, *count;
    long long page_size, most;
    if (n != 8 || !tensor_of(a[0], fresh) || !tensor_of(a[1], lengths) || !tensor_of(a[2], table) || !tensor_of(a[3], pages) ||
        !tensor_of(a[4], count) || !int_of(a[5], 16, 1024, page_size) || !int_of(a[6], 1, INT_MAX, most))
      return none();
    const bool inplace = a[7] == Py_True;
    const int index = ready_index(*lengths);
    if (index < 0 || (!inplace && a[7] != Py_False) || !page_size_ok(page_size) || !ints(*fresh, index) ||
        !ints(*lengths, index) || !ints(*table, index) || !ints(*pages, index) || !ints(*count, index) || table->dim() != 2 ||
        lengths->dim() != 1 || fresh->dim() != 1 || pages->dim() != 1 || count->numel() != 1)
      return none();
    const int64_t requests = table->size(0), width = table->size(1), num = pages->size(0);
    if (requests < 1 || requests > kMaxRequests || width < 1 || num < 1 || lengths->size(0) != requests ||
        fresh->size(0) != requests || num * page_size >= (1ll << 31) || width * page_size >= (1ll << 31))
      return none();
    if (!apart(*table, *fresh) || !apart(*table, *lengths) || !apart(*table, *pages) || !apart(*table, *count)) return none();
    if (inplace && (!apart(*lengths, *fresh) || !apart(*lengths, *pages) || !apart(*lengths, *count) ||
                    !apart(*count, *fresh) || !apart(*count, *pages)))
      return none();
    const Launch launch(index);
    const int64_t state = inplace ? 0 : requests + 1;
    const Tensor all = empty({3 * most + requests + 2 + state}, at::kInt, index);
    const Tensor slots = part(all, 0, most), positions = part(all, most, most), rows = part(all, 2 * most, most),
                 starts = part(all, 3 * most, requests + 1), result = part(all, 3 * most + requests + 1, 1);
    const int64_t at_state = 3 * most + requests + 2;
    const Tensor lengths_out = inplace ? *lengths : part(all, at_state, requests);
    const Tensor count_out = inplace ? *count : part(all, at_state + requests, 1);
    auto p = [](const Tensor& t) { return static_cast<int*>(t.data_ptr()); };
    launch.done(g_entry.build_step(p(*fresh), p(*lengths), p(*table), p(*pages), p(*count), static_cast<int>(requests),
                                   static_cast<int>(width), static_cast<int>(num), static_cast<int>(page_size),
                                   static_cast<int>(most), p(slots), p(positions), p(rows), p(starts), p(lengths_out),
                                   p(count_out), p(result), launch.stream()));
    launch.used(*fresh, *lengths, *table, *pages, *count);
    PyObject* out = PyTuple_New(7);
    if (!out) return nullptr;
    const Tensor* order[7] = {&slots, &positions, &rows, &starts, &lengths_out, &count_out, &result};
    for (int i = 0; i < 7; ++i) {
      PyObject* o;
      if (inplace && (i == 4 || i == 5)) {
        o = a[i == 4 ? 1 : 4];
        Py_INCREF(o);
      } else {
        o = THPVariable_Wrap(*order[i]);
      }
      if (!o) {
        Py_DECREF(out);
        return nullptr;
      }
      PyTuple_SET_ITEM(out, i, o);
    }
    return out;
  });
}

// (k, v, pages, slots) -> True
PyObject* store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *k, *v, *pages, *slots;
    if (n != 4 || !tensor_of(a[0], k) || !tensor_of(a[1], v) || !tensor_of(a[2], pages) || !tensor_of(a[3], slots))
      return none();
    const int index = ready_index(*pages), type = dtype_code(*k);
    long long num, kv_heads, page_size;
    if (index < 0 || type < 0 || k->dim() != 3 || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() ||
        !on(*k, index) || !on(*v, index) || !pages_of(*pages, k->size(2), index, num, kv_heads, page_size) ||
        k->size(1) != kv_heads || !ints(*slots, index) || slots->dim() != 1 || slots->size(0) != k->size(0))
      return none();
    const int64_t tokens = k->size(0), dim = k->size(2);
    const int64_t ks = tokens > 1 ? k->stride(0) : 0, vs = tokens > 1 ? v->stride(0) : 0;
    const int64_t kh = kv_heads > 1 ? k->stride(1) : 0, vh = kv_heads > 1 ? v->stride(1) : 0;
    if (tokens < 1 || tokens * kv_heads * dim >= (1ll << 31) || k->stride(2) != 1 || v->stride(2) != 1 ||
        (ks | vs | kh | vh) & 3 || !aligned(*k, 8) || !aligned(*v, 8) || !apart(*pages, *k) || !apart(*pages, *v) ||
        !apart(*pages, *slots))
      return none();
    const Launch launch(index);
    launch.done(g_entry.store(k->data_ptr(), v->data_ptr(), type, ks, vs, kh, vh, pages->data_ptr(),
                              static_cast<const int*>(slots->data_ptr()), static_cast<int>(tokens), static_cast<int>(num),
                              static_cast<int>(page_size), static_cast<int>(kv_heads), static_cast<int>(dim),
                              launch.stream()));
    launch.used(*k, *v, *pages, *slots);
    Py_RETURN_TRUE;
  });
}

// (pages, slots, head_dim, dtype code) -> (k, v)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *pages, *slots;
    long long dim, type, num, kv_heads, page_size;
    if (n != 4 || !tensor_of(a[0], pages) || !tensor_of(a[1], slots) || !int_of(a[2], 64, 256, dim) ||
        !int_of(a[3], KLAB_DT_BF16, KLAB_DT_F32, type))
      return none();
    const int index = ready_index(*pages);
    if (index < 0 || !pages_of(*pages, dim, index, num, kv_heads, page_size) || !ints(*slots, index) || slots->dim() != 1)
      return none();
    const int64_t tokens = slots->size(0);
    if (tokens < 1 || tokens * kv_heads * dim >= (1ll << 31)) return none();
    const Launch launch(index);
    const at::ScalarType out = type == KLAB_DT_BF16 ? at::kBFloat16 : type == KLAB_DT_F16 ? at::kHalf : at::kFloat;
    const Tensor k = empty({tokens, kv_heads, dim}, out, index), v = empty({tokens, kv_heads, dim}, out, index);
    launch.done(g_entry.read(pages->data_ptr(), static_cast<const int*>(slots->data_ptr()), k.data_ptr(), v.data_ptr(),
                             static_cast<int>(type), static_cast<int>(tokens), static_cast<int>(num),
                             static_cast<int>(page_size), static_cast<int>(kv_heads), static_cast<int>(dim),
                             launch.stream()));
    launch.used(*pages, *slots);
    PyObject *ko = THPVariable_Wrap(k), *vo = THPVariable_Wrap(v);
    PyObject* both = ko && vo ? PyTuple_Pack(2, ko, vo) : nullptr;
    Py_XDECREF(ko);
    Py_XDECREF(vo);
    return both;
  });
}

// (q, pages, table, lengths, starts, max_new, scale or None, out or None) -> out
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *q, *pages, *table, *lengths, *starts, *given = nullptr;
    long long max_new, num, kv_heads, page_size;
    if (n != 8 || !tensor_of(a[0], q) || !tensor_of(a[1], pages) || !tensor_of(a[2], table) || !tensor_of(a[3], lengths) ||
        !tensor_of(a[4], starts) || !int_of(a[5], 1, kMaxNew, max_new) || (a[7] != Py_None && !tensor_of(a[7], given)))
      return none();
    const int index = ready_index(*pages), type = dtype_code(*q);
    if (index < 0 || type < 0 || q->dim() != 3 || !on(*q, index) ||
        !pages_of(*pages, q->size(2), index, num, kv_heads, page_size) || !ints(*table, index) || !ints(*lengths, index) ||
        !ints(*starts, index) || table->dim() != 2 || lengths->dim() != 1 || starts->numel() != table->size(0) + 1 ||
        lengths->size(0) != table->size(0))
      return none();
    const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2), requests = table->size(0), width = table->size(1);
    const int64_t stride = tokens > 1 ? q->stride(0) : 0;
    double scale = 1.0 / std::sqrt(static_cast<double>(dim));
    if (a[6] != Py_None) {
      if (!PyFloat_CheckExact(a[6])) return none();
      scale = PyFloat_AS_DOUBLE(a[6]);
    }
    if (tokens < 1 || heads < 1 || heads % kv_heads || heads / kv_heads > kMaxGroup || q->stride(2) != 1 ||
        (heads > 1 && q->stride(1) != dim) || stride % 8 || !aligned(*q, 16) || requests < 1 || requests > kMaxRequests ||
        width < 1 || width * page_size >= (1ll << 31) || !(scale > 0.0) || !(scale < 3.0e38))
      return none();
    if (given && (given->scalar_type() != q->scalar_type() || !on(*given, index) || given->sizes() != q->sizes() ||
                  !given->is_contiguous() || !aligned(*given, 16) || !apart(*given, *q) || !apart(*given, *pages) ||
                  !apart(*given, *table) || !apart(*given, *lengths) || !apart(*given, *starts)))
      return none();
    const Launch launch(index);
    auto i = [](int64_t v) { return static_cast<int>(v); };
    const long long need = g_entry.attention_scratch(i(requests), i(width), i(page_size), i(heads), i(kv_heads), i(dim),
                                                     i(max_new));
    if (need < 0) return none();
    const Tensor out = given ? *given : empty({tokens, heads, dim}, q->scalar_type(), index);
    const Tensor scratch = empty({need}, at::kByte, index);  // of this call alone
    auto p = [](const Tensor& t) { return static_cast<const int*>(t.data_ptr()); };
    const auto attend = given ? g_entry.attention : g_entry.attention_new;
    launch.done(attend(q->data_ptr(), stride, type, pages->data_ptr(), p(*table), p(*lengths), p(*starts), out.data_ptr(),
                       scratch.data_ptr(), need, i(tokens), i(requests), i(width), i(num), i(page_size), i(heads),
                       i(kv_heads), i(dim), i(max_new), static_cast<float>(scale), launch.stream()));
    launch.used(*q, *pages, *table, *lengths, *starts);
    if (!given) return THPVariable_Wrap(out);
    launch.used(out);
    Py_INCREF(a[7]);
    return a[7];
  });
}

// (wfmt, x, w, side or None, a, b, scales, ids, out or None, fp32) -> out; BF16, INT8 per-row and FP4/FP16-per-32 weights
// with 16-byte rows.
PyObject* adapter_linear(PyObject*, PyObject* const* o, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    const Tensor *x, *w, *side = nullptr, *a, *b, *c, *ids, *given = nullptr;
    long long wfmt;
    if (count != 10 || !int_of(o[0], KLAB_W_BF16, KLAB_W_FP4_G32H, wfmt) || !tensor_of(o[1], x) || !tensor_of(o[2], w) ||
        (o[3] != Py_None && !tensor_of(o[3], side)) || !tensor_of(o[4], a) || !tensor_of(o[5], b) || !tensor_of(o[6], c) ||
        !tensor_of(o[7], ids) || (o[8] != Py_None && !tensor_of(o[8], given)))
      return none();
    const bool f32 = o[9] == Py_True;
    const int index = ready_index(*x);
    if (index < 0 || (!f32 && o[9] != Py_False) || x->scalar_type() != at::kBFloat16 || x->dim() != 2 || w->dim() != 2)
      return none();
    const int64_t m = x->size(0), k = x->size(1), n = w->size(0);
    int64_t row = 0;
    if (wfmt == KLAB_W_BF16) {
      if (side || w->scalar_type() != at::kBFloat16 || w->size(1) != k) return none();
      row = 2 * k;
    } else if (wfmt == KLAB_W_I8_ROW) {
      if (!side || w->scalar_type() != at::kChar || w->size(1) != k || side->scalar_type() != at::kFloat || side->dim() != 1 ||
          side->size(0) != n)
        return none();
      row = k;
    } else if (wfmt == KLAB_W_FP4_G32H) {
      if (!side || k % 32 || w->scalar_type() != at::kByte || w->size(1) * 2 != k || side->scalar_type() != at::kHalf ||
          side->dim() != 2 || side->size(0) != n || side->size(1) * 32 != k)
        return none();
      row = k / 2;
    } else {
      return none();
    }
    if (a->dim() != 3 || b->dim() != 3 || a->scalar_type() != at::kBFloat16 || b->scalar_type() != at::kBFloat16) return none();
    const int64_t adapters = a->size(0), rank = a->size(1);
    if (m < 1 || n < 1 || k < 1 || adapters < 1 || rank < 1 || rank % 8 || rank > kMaxRank || k % 8 || m > 65535 || row % 16 ||
        a->size(2) != k || b->size(0) != adapters || b->size(1) != n || b->size(2) != rank || c->dim() != 1 ||
        c->size(0) != adapters || c->scalar_type() != at::kFloat || ids->dim() != 1 || ids->size(0) != m ||
        ids->scalar_type() != at::kInt || m * k >= (1ll << 31) || n * k >= (1ll << 31) || m * n >= (1ll << 31))
      return none();
    const Tensor* read[] = {x, w, a, b, c, ids, side};
    for (const Tensor* t : read)
      if (t && (!on(*t, index) || !t->is_contiguous() || (given && !apart(*given, *t)))) return none();
    if (!aligned(*x, 16) || !aligned(*w, 16) || !aligned(*a, 16) || !aligned(*b, 16)) return none();
    const at::ScalarType type = f32 ? at::kFloat : at::kBFloat16;
    if (given && (given->scalar_type() != type || !on(*given, index) || given->dim() != 2 || given->size(0) != m ||
                  given->size(1) != n || !given->is_contiguous()))
      return none();
    const Launch launch(index);
    auto i = [](int64_t v) { return static_cast<int>(v); };
    const long long need = g_entry.adapter_scratch(i(wfmt), i(m), i(n), i(k), i(rank));
    if (need < 0) return none();
    const Tensor out = given ? *given : empty({m, n}, type, index);
    const Tensor scratch = empty({need}, at::kByte, index);
    launch.done(g_entry.adapter(i(wfmt), x->data_ptr(), w->data_ptr(), side ? side->data_ptr() : nullptr, a->data_ptr(),
                                b->data_ptr(), static_cast<const float*>(c->data_ptr()),
                                static_cast<const int*>(ids->data_ptr()), out.data_ptr(), f32 ? KLAB_DT_F32 : KLAB_DT_BF16,
                                i(m), i(n), i(k), i(rank), i(adapters), scratch.data_ptr(), need, nullptr, 0,
                                launch.stream()));
    launch.used(*x, *w, *a, *b, *c, *ids);
    if (side) launch.used(*side);
    if (!given) return THPVariable_Wrap(out);
    launch.used(out);
    Py_INCREF(o[8]);
    return o[8];
  });
}

// bind(addresses of the entry points, in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[8];
  if (n != 8) {
    PyErr_SetString(PyExc_ValueError, "bind takes the addresses of 8 entry points");
    return nullptr;
  }
  for (int i = 0; i < 8; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an entry point is null");
      return nullptr;
    }
  }
  g_entry.build_step = reinterpret_cast<decltype(g_entry.build_step)>(p[0]);
  g_entry.store = reinterpret_cast<decltype(g_entry.store)>(p[1]);
  g_entry.read = reinterpret_cast<decltype(g_entry.read)>(p[2]);
  g_entry.attention = reinterpret_cast<decltype(g_entry.attention)>(p[3]);
  g_entry.attention_new = reinterpret_cast<decltype(g_entry.attention_new)>(p[4]);
  g_entry.attention_scratch = reinterpret_cast<decltype(g_entry.attention_scratch)>(p[5]);
  g_entry.adapter = reinterpret_cast<decltype(g_entry.adapter)>(p[6]);
  g_entry.adapter_scratch = reinterpret_cast<decltype(g_entry.adapter_scratch)>(p[7]);
  Py_RETURN_NONE;
}

// mark_ready(device index): the device's module is loaded and the entry points are bound.
PyObject* mark_ready(PyObject*, PyObject* const* a, Py_ssize_t n) {
  long long index;
  if (n != 1 || !int_of(a[0], 0, 63, index) || !g_entry.build_step) {
    PyErr_SetString(PyExc_ValueError, "mark_ready takes a device index, after bind");
    return nullptr;
  }
  g_ready[index] = true;
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FAST(build_step), FAST(store),      FAST(read), FAST(attention), FAST(adapter_linear),
                           FAST(bind),       FAST(mark_ready), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "klab_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_klab_torch() { return PyModule_Create(&g_module); }
