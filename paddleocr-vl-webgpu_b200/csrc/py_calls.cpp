// py_calls.cpp -- the argument checks of pvlc_b200.kv8 and ops.beam_topk as a CPython module
// (pvlc_b200/_calls): a call whose arguments are all as they should be goes from here to the
// C ABI; any other returns None, and the Python function checks again, names what is wrong
// and raises.  A decode step that is not captured makes such a call per layer, and a call's
// checks in Python took longer (about 11 us) than most of the kernels that they lead to.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/pvlc_cuda_attn.h"

namespace {

// The C ABI's functions, from the library that pvlc_b200.abi loaded.
decltype(&pvlc_attn_kv8_store) store_fn;
decltype(&pvlc_attn_kv8_decode) decode_fn;
decltype(&pvlc_attn_kv8_grow) grow_fn;
decltype(&pvlc_attn_kv8_fork) fork_fn;
decltype(&pvlc_attn_kv8_compact) compact_fn;
decltype(&pvlc_lm_head_beam_topk) beam_fn;

constexpr int64_t kHeadDim = 128;

// Reads arguments one after the other; `ok` turns false at the first that does not fit.
struct Args {
  PyObject* const* at;
  Py_ssize_t left;
  bool ok = true;

  PyObject* next() {
    if (left == 0) ok = false;
    return ok ? (--left, *at++) : nullptr;
  }
  bool done() const { return ok && left == 0; }
  uint64_t number(uint64_t most) {
    PyObject* o = next();
    if (!o || !PyLong_CheckExact(o)) return ok = false, 0;
    const unsigned long long x = PyLong_AsUnsignedLongLong(o);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return ok = false, 0;
    }
    if (x > most) ok = false;
    return x;
  }
  uint32_t u32() { return static_cast<uint32_t>(number(0xffffffffull)); }
  void* pointer() { return reinterpret_cast<void*>(number(~0ull)); }
  // A plain strided CUDA tensor of this type on device `index`.
  const at::Tensor* tensor_of(PyObject* o, at::ScalarType type, int64_t index) {
    if (!ok || !o || !THPVariable_CheckExact(o)) return ok = false, nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.scalar_type() != type || t.layout() != at::kStrided ||
        !t.device().is_cuda() || t.device().index() != index)
      return ok = false, nullptr;
    return &t;
  }
  // .. contiguous and of this shape
  const at::Tensor* exact_of(PyObject* o, at::ScalarType type, int64_t index,
                             at::IntArrayRef shape) {
    const at::Tensor* t = tensor_of(o, type, index);
    if (t && !(t->sizes() == shape && t->is_contiguous())) ok = false;
    return ok ? t : nullptr;
  }
  const at::Tensor* exact(at::ScalarType type, int64_t index, at::IntArrayRef shape) {
    return exact_of(next(), type, index, shape);
  }
  int32_t* ints(int64_t index, int64_t n) {
    const at::Tensor* t = exact(at::kInt, index, {n});
    return t ? static_cast<int32_t*>(t->data_ptr()) : nullptr;
  }
  // [rows, heads, 128] fp16 with rows `stride` apart
  const pvlc_half* rows(int64_t index, int64_t heads, int64_t* n, uint32_t* stride) {
    const at::Tensor* t = tensor_of(next(), at::kHalf, index);
    if (!t) return nullptr;
    if (t->dim() != 3 || (heads && t->size(1) != heads) || t->size(2) != kHeadDim ||
        t->stride(2) != 1 || (t->size(1) > 1 && t->stride(1) != kHeadDim))
      return ok = false, nullptr;
    *n = t->size(0);
    const int64_t s = *n == 1 ? t->size(1) * kHeadDim : t->stride(0);
    if (s < 0 || s > 0xffffffffll || *n > 0xffffffffll) return ok = false, nullptr;
    *stride = static_cast<uint32_t>(s);
    return static_cast<const pvlc_half*>(t->data_ptr());
  }
  // a number of rows for all sequences, or a tensor of them
  const int32_t* amount(int64_t index, int64_t n, uint32_t* all) {
    PyObject* o = next();
    *all = 0;
    if (o && THPVariable_Check(o)) {
      const at::Tensor* t = exact_of(o, at::kInt, index, {n});
      return t ? static_cast<const int32_t*>(t->data_ptr()) : nullptr;
    }
    if (o) --at, ++left;
    *all = static_cast<uint32_t>(number(0x7fffffffull));
    return nullptr;
  }
};

bool current(int64_t index) {
  c10::DeviceIndex now = -1;
  return c10::cuda::GetDevice(&now) == cudaSuccess && now == index;
}

// The cache, the workspace and the current device that every kv8 call starts with.
struct Call {
  const pvlc_kv8_cache* cache;
  void* ws;
  size_t ws_bytes;
  int64_t index;
  explicit Call(Args& a) {
    cache = static_cast<const pvlc_kv8_cache*>(a.pointer());
    index = static_cast<int64_t>(a.number(0x7f));
    ws = a.pointer();
    ws_bytes = a.number(~0ull);
    if (a.number(0x7f) != static_cast<uint64_t>(index)) a.ok = false;
    if (a.ok && !current(index)) a.ok = false;
  }
  void* stream() const {
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
  }
};

template <typename F>
int without_gil(F call) {
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = call();
  Py_END_ALLOW_THREADS
  return st;
}

// The named number of sequences of a slot tensor, which comes first of a call's tensors.
int64_t batch_of(Args& a, int64_t index, int32_t** slot) {
  const at::Tensor* t = a.tensor_of(a.next(), at::kInt, index);
  if (t && (t->dim() != 1 || !t->is_contiguous() || t->size(0) > 0xffffffffll)) a.ok = false;
  if (!a.ok) return 0;
  *slot = static_cast<int32_t*>(t->data_ptr());
  return t->size(0);
}

// store(cache, index, ws, bytes, ws index, layer, slot, k, v, begin, count, max_count) -> status
PyObject* store(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{args, n};
  const Call c(a);
  const uint32_t layer = a.u32();
  int32_t* slot = nullptr;
  int64_t kn = 0, vn = 0;
  uint32_t ks = 0, vs = 0;
  const int64_t B = batch_of(a, c.index, &slot);
  const int64_t H = a.ok ? c.cache->kv_heads : 1;
  const pvlc_half* k = a.rows(c.index, H, &kn, &ks);
  const pvlc_half* v = a.rows(c.index, H, &vn, &vs);
  const int32_t* begin = a.ints(c.index, B);
  const int32_t* count = a.ints(c.index, B);
  const uint32_t most = a.u32();
  if (!a.done() || kn != vn || ks != vs || layer >= c.cache->layers) Py_RETURN_NONE;
  void* stream = c.stream();
  return PyLong_FromLong(without_gil([&] {
    return store_fn(c.cache, layer, k, v, static_cast<uint32_t>(kn), ks, begin, count, slot,
                    static_cast<uint32_t>(B), most, c.ws, c.ws_bytes, stream);
  }));
  END_HANDLE_TH_ERRORS
}

// decode(cache, index, ws, bytes, ws index, layer, q, k, v, cos, sin, slot, rope_row, out)
// -> out or the status
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{args, n};
  const Call c(a);
  const uint32_t layer = a.u32();
  if (!a.ok || a.left != 8 || !THPVariable_CheckExact(a.at[0])) Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(a.at[0]);
  int64_t B = 0, kn = 0, vn = 0;
  uint32_t qs = 0, ks = 0, vs = 0;
  const pvlc_half* qp = a.rows(c.index, 0, &B, &qs);
  const pvlc_half* k = a.rows(c.index, c.cache->kv_heads, &kn, &ks);
  const pvlc_half* v = a.rows(c.index, c.cache->kv_heads, &vn, &vs);
  const at::Tensor* cos = a.tensor_of(a.next(), at::kFloat, c.index);
  if (!a.ok || kn != B || vn != B || vs != ks || layer >= c.cache->layers || cos->dim() != 3)
    Py_RETURN_NONE;
  const int64_t QH = q.size(1), R = cos->size(1);
  if (cos->size(0) != 3 || cos->size(2) != kHeadDim || !cos->is_contiguous() || R > 0xffffffffll ||
      QH > 0xffffffffll)
    Py_RETURN_NONE;
  const at::Tensor* sin = a.exact(at::kFloat, c.index, {3, R, kHeadDim});
  const int32_t* slot = a.ok && a.at[0] == Py_None ? (a.next(), nullptr) : a.ints(c.index, B);
  const int32_t* row = a.ok && a.at[0] == Py_None ? (a.next(), nullptr) : a.ints(c.index, B);
  PyObject* given = a.next();
  at::Tensor made;
  const at::Tensor* out = &made;
  if (given && given != Py_None) out = a.exact_of(given, at::kHalf, c.index, {B, QH, kHeadDim});
  if (!a.done()) Py_RETURN_NONE;
  if (given == Py_None) made = at::empty({B, QH, kHeadDim}, q.options());
  pvlc_half* to = static_cast<pvlc_half*>(out->data_ptr());
  const float *cp = cos->const_data_ptr<float>(), *sp = sin->const_data_ptr<float>();
  void* stream = c.stream();
  const int st = without_gil([&] {
    return decode_fn(c.cache, layer, qp, qs, k, v, ks, static_cast<uint32_t>(QH), cp, sp,
                     static_cast<uint32_t>(R), row, slot, static_cast<uint32_t>(B), c.ws,
                     c.ws_bytes, to, stream);
  });
  if (st) return PyLong_FromLong(st);
  if (given == Py_None) return THPVariable_Wrap(std::move(made));
  Py_INCREF(given);
  return given;
  END_HANDLE_TH_ERRORS
}

// grow(cache, index, ws, bytes, ws index, slot, advance, ahead) -> status
PyObject* grow(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{args, n};
  const Call c(a);
  int32_t* slot = nullptr;
  uint32_t advance_by = 0, ahead_by = 0;
  const int64_t B = batch_of(a, c.index, &slot);
  const int32_t* advance = a.amount(c.index, B, &advance_by);
  const int32_t* ahead = a.amount(c.index, B, &ahead_by);
  if (!a.done()) Py_RETURN_NONE;
  void* stream = c.stream();
  return PyLong_FromLong(without_gil([&] {
    return grow_fn(c.cache, slot, static_cast<uint32_t>(B), advance, advance_by, ahead, ahead_by,
                   c.ws, c.ws_bytes, stream);
  }));
  END_HANDLE_TH_ERRORS
}

// fork(cache, index, ws, bytes, ws index, slot, parent, advance, out) -> out or the status
PyObject* fork(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{args, n};
  const Call c(a);
  int32_t* slot = nullptr;
  PyObject* first = a.ok && a.left ? a.at[0] : nullptr;
  const int64_t B = batch_of(a, c.index, &slot);
  const int32_t* parent = a.ints(c.index, B);
  const uint32_t advance = static_cast<uint32_t>(a.number(0x7fffffffull));
  PyObject* given = a.next();
  at::Tensor made;
  const at::Tensor* out = &made;
  if (given && given != Py_None) out = a.exact_of(given, at::kInt, c.index, {B});
  if (!a.done()) Py_RETURN_NONE;
  if (given == Py_None) made = at::empty({B}, THPVariable_Unpack(first).options());
  int32_t* to = static_cast<int32_t*>(out->data_ptr());
  void* stream = c.stream();
  const int st = without_gil([&] {
    return fork_fn(c.cache, slot, parent, static_cast<uint32_t>(B), advance, to, c.ws, c.ws_bytes,
                   stream);
  });
  if (st) return PyLong_FromLong(st);
  if (given == Py_None) return THPVariable_Wrap(std::move(made));
  Py_INCREF(given);
  return given;
  END_HANDLE_TH_ERRORS
}

// compact(cache, index, ws, bytes, ws index, into, into's index, live) -> status
PyObject* compact(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{args, n};
  const Call c(a);
  const pvlc_kv8_cache* into = static_cast<const pvlc_kv8_cache*>(a.pointer());
  if (a.number(0x7f) != static_cast<uint64_t>(c.index)) a.ok = false;
  int32_t* live = a.ok && a.left && a.at[0] == Py_None ? (a.next(), nullptr) : a.ints(c.index, 1);
  if (!a.done()) Py_RETURN_NONE;
  void* stream = c.stream();
  return PyLong_FromLong(
      without_gil([&] { return compact_fn(c.cache, into, live, c.ws, c.ws_bytes, stream); }));
  END_HANDLE_TH_ERRORS
}

// beam_topk(logits, scores, topk, ws tensor) -> (score, beam, token) or the status
PyObject* beam_topk(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{args, n};
  if (n != 4 || !THPVariable_CheckExact(args[0])) Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(args[0]);
  const bool half = x.scalar_type() == at::kHalf;
  const int64_t index = x.device().index();
  a.tensor_of(a.next(), half ? at::kHalf : at::kFloat, index);
  const at::Tensor* s = a.tensor_of(a.next(), at::kFloat, index);
  const int64_t K = static_cast<int64_t>(a.number(PVLC_BEAM_MAX_TOPK));
  const at::Tensor* ws = a.tensor_of(a.next(), at::kByte, index);
  if (!a.done() || x.dim() != 2 || s->dim() != 2 || !s->is_contiguous() || x.stride(1) != 1 ||
      !current(index))
    Py_RETURN_NONE;
  const int64_t B = s->size(0), W = s->size(1), rows = x.size(0), V = x.size(1);
  if (B > 65535 || W > 65535 || rows != B * W || V > 0xffffffffll) Py_RETURN_NONE;
  const auto like = x.options();
  at::Tensor score = at::empty({B, K}, like.dtype(at::kFloat));
  at::Tensor beam = at::empty({B, K}, like.dtype(at::kInt));
  at::Tensor token = at::empty({B, K}, like.dtype(at::kInt));
  const int64_t stride = rows > 1 ? x.stride(0) : std::max(V, x.stride(0));
  void* stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
  const void* xp = x.data_ptr();
  void* wp = ws->data_ptr();
  const size_t wn = static_cast<size_t>(ws->numel());
  const float* sp = s->const_data_ptr<float>();
  float* op = score.mutable_data_ptr<float>();
  int32_t *bp = beam.mutable_data_ptr<int32_t>(), *tp = token.mutable_data_ptr<int32_t>();
  const int st = without_gil([&] {
    return beam_fn(xp, half, static_cast<uint64_t>(stride), sp, static_cast<uint32_t>(B),
                   static_cast<uint32_t>(W), static_cast<uint32_t>(V), static_cast<uint32_t>(K), wp,
                   wn, op, bp, tp, stream);
  });
  if (st) return PyLong_FromLong(st);
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(score)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(beam)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(token)));
  return r;
  END_HANDLE_TH_ERRORS
}

// bind(store, decode, grow, fork, compact, beam_topk): the functions' addresses
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Args a{args, n};
  void* f[6];
  for (void*& x : f) x = a.pointer();
  if (!a.done()) {
    PyErr_SetString(PyExc_TypeError, "expected six addresses");
    return nullptr;
  }
  store_fn = reinterpret_cast<decltype(store_fn)>(f[0]);
  decode_fn = reinterpret_cast<decltype(decode_fn)>(f[1]);
  grow_fn = reinterpret_cast<decltype(grow_fn)>(f[2]);
  fork_fn = reinterpret_cast<decltype(fork_fn)>(f[3]);
  compact_fn = reinterpret_cast<decltype(compact_fn)>(f[4]);
  beam_fn = reinterpret_cast<decltype(beam_fn)>(f[5]);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind), FAST(store), FAST(decode), FAST(grow), FAST(fork),
                         FAST(compact), FAST(beam_topk), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: "<torch version> <Python's cache tag>" of the headers above, which say where a tensor's
// sizes, strides and address are.  Nothing here may be called under any other.
PyMODINIT_FUNC PyInit__calls() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
