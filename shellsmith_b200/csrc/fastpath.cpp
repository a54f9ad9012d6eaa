// The group-decode operators' calls without the Python wrappers' cost: the same checks, the
// outputs' allocation and the C ABI call, from the tensors themselves. At one token a step
// the wrapper is most of the call (about 15 us of Python and ctypes for rotary_append
// against 3 us on the GPU), so it counts.
//
// Every function returns None when an argument is not what the operator takes, or when
// the entry point refuses; the Python wrapper then goes through its own checks and raises
// what belongs to it. Nothing is launched in that case.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>

#include "../../include/shellcache.h"

namespace {

PyObject* none() { Py_RETURN_NONE; }

// A tensor argument, or NULL for None or for something else (then *ok is cleared).
const at::Tensor* tensor(PyObject* o, bool* ok) {
  if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
  if (o != Py_None) *ok = false;
  return nullptr;
}

bool aligned(const at::Tensor& t, size_t n) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % n == 0;
}

// A dense CUDA operand on `device`, `align` bytes aligned.
bool dense(const at::Tensor* t, int device, at::ScalarType type, int64_t ndim, size_t align) {
  return t != nullptr && t->is_cuda() && t->get_device() == device && t->scalar_type() == type &&
         t->dim() == ndim && t->is_contiguous() && aligned(*t, align);
}

// The current stream, on which a call reads a plan's tables (the tuple's items from `first` on).
// If those came from another stream, the allocator does not hand their memory out before the
// call is done.
void* stream_of(int device, PyObject* plan = nullptr, Py_ssize_t first = 0, long long home = 0) {
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
  if (plan != nullptr && reinterpret_cast<uintptr_t>(stream.stream()) != (uintptr_t)home)
    for (Py_ssize_t i = first; i < PyTuple_GET_SIZE(plan); ++i)
      if (THPVariable_Check(PyTuple_GET_ITEM(plan, i)))
        THPVariable_Unpack(PyTuple_GET_ITEM(plan, i)).record_stream(stream.unwrap());
  return stream.stream();
}

template <typename T>
T* data(const at::Tensor* t) {
  return t == nullptr ? nullptr : static_cast<T*>(t->data_ptr());
}

long long integer(PyObject* o, bool* ok) {
  if (o == Py_None) {
    *ok = false;
    return 0;
  }
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    *ok = false;
  }
  return v;
}
long long item(PyObject* tuple, int i, bool* ok) { return integer(PyTuple_GET_ITEM(tuple, i), ok); }

// rotary_append(q, k, v, positions, pool, slots, q_weight, k_weight, eps, out, plan): q
// plan: (head_dim, rotary_dim, axes, turns, axis, device, home stream, its tables)
PyObject* rotary_append(PyObject*, PyObject* const* a, Py_ssize_t n) try {
  if (n != 11 || !PyTuple_Check(a[10]) || PyTuple_GET_SIZE(a[10]) != 9) return none();
  bool ok = true;
  const at::Tensor *q = tensor(a[0], &ok), *k = tensor(a[1], &ok), *v = tensor(a[2], &ok),
                   *pos = tensor(a[3], &ok), *pool = tensor(a[4], &ok), *slots = tensor(a[5], &ok),
                   *qw = tensor(a[6], &ok), *kw = tensor(a[7], &ok), *out = tensor(a[9], &ok);
  const double eps = PyFloat_AsDouble(a[8]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  const long long dim = item(a[10], 0, &ok), rot = item(a[10], 1, &ok), axes = item(a[10], 2, &ok);
  const long long turns = item(a[10], 3, &ok), axis = item(a[10], 4, &ok);
  const int device = (int)item(a[10], 5, &ok);
  const long long home = item(a[10], 6, &ok);
  if (!ok || q == nullptr || k == nullptr || v == nullptr || pos == nullptr) return none();
  for (const at::Tensor* t : {q, k, v})
    if (!t->is_cuda() || t->get_device() != device || t->scalar_type() != at::kBFloat16 ||
        t->dim() != 3 || t->size(2) != dim || t->stride(2) != 1)
      return none();
  const int64_t ntok = q->size(0), hq = q->size(1), hkv = k->size(1);
  if (!dense(pool, device, at::kBFloat16, 5, 16) || !dense(slots, device, at::kLong, 1, 8))
    return none();
  if (k->size(0) != ntok || v->sizes() != k->sizes() || slots->size(0) != ntok ||
      pool->size(1) != hkv || pool->size(2) != 2 || pool->size(4) != dim)
    return none();
  const bool flat = pos->dim() == 1;
  if (!pos->is_cuda() || pos->get_device() != device || pos->scalar_type() != at::kInt ||
      (!flat && pos->dim() != 2) || (flat ? 1 : pos->size(0)) != axes ||
      pos->size(flat ? 0 : 1) != ntok || (ntok > 1 && pos->stride(flat ? 0 : 1) != 1))
    return none();
  for (const at::Tensor* w : {qw, kw})
    if (w != nullptr && (!dense(w, device, at::kBFloat16, 1, 16) || w->size(0) != dim)) return none();
  if (out != nullptr && (!dense(out, device, at::kBFloat16, 3, 16) || out->sizes() != q->sizes()))
    return none();
  const at::Tensor fresh = out != nullptr ? *out : at::empty(q->sizes(), q->options());
  const int64_t strides[6] = {q->stride(0), q->stride(1), k->stride(0),
                              k->stride(1), v->stride(0), v->stride(1)};
  const int rc = sc_rotary_append(
      data<sc_bf16>(q), data<sc_bf16>(k), data<sc_bf16>(v), strides, data<int32_t>(pos),
      flat ? 0 : pos->stride(0), (int)axes, reinterpret_cast<const double*>(turns),
      reinterpret_cast<const int32_t*>(axis), data<sc_bf16>(qw), data<sc_bf16>(kw), (float)eps,
      data<sc_bf16>(&fresh), nullptr, data<sc_bf16>(pool), data<int64_t>(slots), (int)ntok, (int)hq,
      (int)hkv, (int)dim, (int)rot, (int)pool->size(3), pool->size(0),
      stream_of(device, a[10], 7, home));
  return rc != 0 ? none() : THPVariable_Wrap(fresh);
} catch (const std::exception&) {
  return none();
}

// beam_select(logits, scores, n, finished, pad_token): (scores, parents, tokens)
PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t n) try {
  if (n != 5) return none();
  bool ok = true;
  const at::Tensor *x = tensor(a[0], &ok), *scores = tensor(a[1], &ok), *fin = tensor(a[3], &ok);
  const long long want = integer(a[2], &ok), pad = integer(a[4], &ok);
  if (!ok || x == nullptr || !x->is_cuda() || x->dim() != 3 || want < 1 || want > 64 ||
      pad != (int)pad)
    return none();
  const bool fp32 = x->scalar_type() == at::kFloat;
  if (!fp32 && x->scalar_type() != at::kBFloat16) return none();
  const int device = x->get_device();
  const int64_t groups = x->size(0), beams = x->size(1), vocab = x->size(2);
  if (!x->is_contiguous() || groups < 1 || beams < 1 || vocab < 1 || groups * beams > 65535 ||
      beams * vocab >= (1ll << 31))
    return none();
  if (!dense(scores, device, at::kFloat, 2, 4) || scores->size(0) != groups ||
      scores->size(1) != beams)
    return none();
  if (fin != nullptr && (!dense(fin, device, at::kBool, 2, 1) || fin->sizes() != scores->sizes()))
    return none();
  const size_t need =
      sc_beam_select_workspace((int)groups, (int)beams, (int)vocab, (int)want, fp32);
  const at::Tensor work = at::empty({(int64_t)need / 4}, scores->options());
  const at::Tensor best = at::empty({groups, want}, scores->options());
  const auto ints = scores->options().dtype(at::kInt);
  const at::Tensor parents = at::empty({groups, want}, ints), tokens = at::empty({groups, want}, ints);
  const int rc = sc_beam_select(x->data_ptr(), fp32, vocab, data<float>(scores), data<uint8_t>(fin),
                                (int)pad, data<float>(&best), data<int32_t>(&parents),
                                data<int32_t>(&tokens), work.data_ptr(), need, (int)groups,
                                (int)beams, (int)vocab, (int)want, stream_of(device));
  if (rc != 0) return none();
  PyObject* out = PyTuple_New(3);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(best));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(parents));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(tokens));
  return out;
} catch (const std::exception&) {
  return none();
}

// reorder_rows(pools, slots, parents): new slots
PyObject* reorder_rows(PyObject*, PyObject* const* a, Py_ssize_t n) try {
  if (n != 3 || !(PyList_Check(a[0]) || PyTuple_Check(a[0]))) return none();
  bool ok = true;
  const at::Tensor *slots = tensor(a[1], &ok), *parents = tensor(a[2], &ok);
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(a[0]);
  if (!ok || slots == nullptr || !slots->is_cuda() || count < 1 || count > 4) return none();
  const int device = slots->get_device();
  if (!dense(slots, device, at::kInt, 2, 4) || !dense(parents, device, at::kInt, 2, 4) ||
      parents->sizes() != slots->sizes())
    return none();
  void* bases[4];
  int64_t sizes[4];
  int layers[4];
  int64_t rows = 0;
  for (Py_ssize_t i = 0; i < count; ++i) {
    const at::Tensor* p = tensor(PySequence_Fast_GET_ITEM(a[0], i), &ok);
    if (!ok || p == nullptr || !p->is_cuda() || p->get_device() != device || p->dim() < 2 ||
        !p->is_contiguous() || (i > 0 && p->size(1) != rows))
      return none();
    rows = p->size(1);
    bases[i] = p->data_ptr();
    layers[i] = (int)p->size(0);
    sizes[i] = p->stride(1) * p->element_size();
  }
  const at::Tensor out = at::empty(slots->sizes(), slots->options());
  const int rc = sc_reorder_rows(bases, sizes, layers, (int)count, (int)rows, data<int32_t>(slots),
                                 data<int32_t>(parents), data<int32_t>(&out), (int)slots->size(0),
                                 (int)slots->size(1), stream_of(device));
  return rc != 0 ? none() : THPVariable_Wrap(out);
} catch (const std::exception&) {
  return none();
}

// shared_prefix_attention(q, pool, table, ctx_len, scale, out, lse_out, groups, prefix_split,
//                         tail_split, scratch): out
// groups: (batch, q_heads, kv_heads, head_dim, device, ntiles, max_prefix_pages, first_page,
// tiles, members, home stream, its tables); the splits are (pages, count); scratch the five
// addresses of the parts.
PyObject* shared_prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n) try {
  if (n != 11 || !PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 12) return none();
  for (int i = 8; i < 11; ++i)
    if (!PyTuple_Check(a[i]) || PyTuple_GET_SIZE(a[i]) != (i < 10 ? 2 : 5)) return none();
  bool ok = true;
  const at::Tensor *q = tensor(a[0], &ok), *pool = tensor(a[1], &ok), *table = tensor(a[2], &ok),
                   *ctx = tensor(a[3], &ok), *out = tensor(a[5], &ok), *lse = tensor(a[6], &ok);
  const double scale = PyFloat_AsDouble(a[4]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  const long long B = item(a[7], 0, &ok), hq = item(a[7], 1, &ok), hkv = item(a[7], 2, &ok),
                  dim = item(a[7], 3, &ok);
  const int device = (int)item(a[7], 4, &ok), ntiles = (int)item(a[7], 5, &ok);
  const long long longest = item(a[7], 6, &ok), home = item(a[7], 10, &ok);
  long long at[3], part[5];
  for (int i = 0; i < 3; ++i) at[i] = item(a[7], 7 + i, &ok);
  for (int i = 0; i < 5; ++i) part[i] = item(a[10], i, &ok);
  const int pre_pps = (int)item(a[8], 0, &ok), pre_splits = (int)item(a[8], 1, &ok);
  const int pps = (int)item(a[9], 0, &ok), splits = (int)item(a[9], 1, &ok);
  if (!ok || ntiles < 1 || !dense(q, device, at::kBFloat16, 3, 16) ||
      !dense(pool, device, at::kBFloat16, 5, 16) || !dense(table, device, at::kInt, 2, 4) ||
      !dense(ctx, device, at::kInt, 1, 4))
    return none();
  if (q->size(0) != B || q->size(1) != hq || q->size(2) != dim || pool->size(1) != hkv ||
      pool->size(2) != 2 || pool->size(4) != dim || table->size(0) != B || ctx->size(0) != B ||
      longest > table->size(1))
    return none();
  if (out != nullptr && (!dense(out, device, at::kBFloat16, 3, 16) || out->sizes() != q->sizes()))
    return none();
  if (lse != nullptr && (!dense(lse, device, at::kFloat, 1, 4) || lse->size(0) != B * hq)) return none();
  const at::Tensor fresh = out != nullptr ? *out : at::empty(q->sizes(), q->options());
  const int rc = sc_shared_prefix_attention(
      data<sc_bf16>(q), data<sc_bf16>(pool), pool->size(0), data<int32_t>(table),
      data<int32_t>(ctx), reinterpret_cast<const int32_t*>(at[0]),
      reinterpret_cast<const int32_t*>(at[1]), reinterpret_cast<const int32_t*>(at[2]), ntiles,
      (int)B, (int)hq, (int)hkv, (int)dim, (int)pool->size(3), (int)table->size(1), pre_pps,
      pre_splits, pps, splits, (float)scale, reinterpret_cast<float*>(part[0]),
      reinterpret_cast<float*>(part[1]), reinterpret_cast<float*>(part[2]),
      reinterpret_cast<float*>(part[3]), reinterpret_cast<int32_t*>(part[4]), data<sc_bf16>(&fresh),
      data<float>(lse), stream_of(device, a[7], 11, home));
  return rc != 0 ? none() : THPVariable_Wrap(fresh);
} catch (const std::exception&) {
  return none();
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<rotary_append>("rotary_append"),
                         method<beam_select>("beam_select"),
                         method<reorder_rows>("reorder_rows"),
                         method<shared_prefix_attention>("shared_prefix_attention"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastpath", nullptr, -1, methods};

}  // namespace

// The module reaches into torch's C++ objects: with another torch than it was compiled for it
// must not be used, even where it links.
PyMODINIT_FUNC PyInit__fastpath() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", SC_TORCH_VERSION) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
