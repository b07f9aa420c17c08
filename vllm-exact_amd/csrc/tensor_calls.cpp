// The serving operators' calls on torch tensors: argument checks, pointers and strides, torch's current stream, and the C
// entry point, without a Python object for every stride. A call of 9 tensors spends 2 us here, where the same checks in
// Python and a ctypes call of 50 arguments took 15: a decode step makes such calls for every layer.
//
// The module holds no code of the kernels: bind() is given the addresses of the loaded library's entry points.
// Every function returns the entry point's status; what an argument check refuses is raised here.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <string>

#include "../../include/vllm_exact_amd.h"

namespace {

decltype(&vxa_prompt_attention) prompt_attention_fn;
decltype(&vxa_int8_cache_write) cache_write_fn;
decltype(&vxa_int8_cache_read) cache_read_fn;
decltype(&vxa_tree_decode_call_workspace) tree_workspace_fn;
decltype(&vxa_tree_decode) tree_decode_fn;

struct Refused {
  PyObject* kind;
  std::string text;
};
[[noreturn]] void refuse(const char* what, const char* text, PyObject* kind = PyExc_ValueError) {
  throw Refused{kind, std::string(what) + text};
}

// A tensor argument, or nothing for None where that is allowed.
const at::Tensor* tensor(const char* what, PyObject* o, bool optional = false) {
  if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
  if (optional && o == Py_None) return nullptr;
  refuse(what, ": expected a tensor", PyExc_TypeError);
}
double number(const char* what, PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, ": expected a number", PyExc_TypeError);
  }
  return v;
}
int64_t integer(const char* what, PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, ": expected an integer", PyExc_TypeError);
  }
  return v;
}

void check_gpu(const char* what, std::initializer_list<const at::Tensor*> tensors, const char* statement) {
  const at::Tensor* first = *tensors.begin();
  for (const at::Tensor* t : tensors)
    if (t && !t->is_cuda())
      refuse(what, (std::string(" runs the gfx950 HIP kernel and needs GPU tensors; use ") + statement + " for the CPU statement").c_str());
  for (const at::Tensor* t : tensors)
    if (t && t->device() != first->device()) refuse(what, ": all tensors must be on one GPU");
}
int dtype_enum(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return VXA_F32;
    case at::kBFloat16: return VXA_BF16;
    case at::kHalf: return VXA_F16;
    default: refuse("unsupported floating dtype ", c10::toString(t.scalar_type()));
  }
}
bool is16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
bool vector_of(const at::Tensor& t, at::ScalarType type, int64_t n) {
  return t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}
template <typename T = void>
T* ptr(const at::Tensor* t) {
  return t ? reinterpret_cast<T*>(t->data_ptr()) : nullptr;
}
int64_t stride(const at::Tensor* t, int i) { return t ? t->stride(i) : 0; }

// The interpreter lock, given back while this lives: also where an exception ends the scope.
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// fn(arguments, stream) with the tensors' device current and torch's current stream there. The arguments are pointers, strides and
// sizes, taken from the tensors by the caller while it holds the lock: a tensor without memory (torch.vmap's) throws there.
template <typename F, typename... A>
int on_device(const at::Tensor& t, F fn, A... arguments) {
  const c10::DeviceGuard guard(t.device());
  const vxa_stream_t stream = c10::hip::getCurrentHIPStream(t.device().index()).stream();
  const Unlocked unlocked;
  return fn(arguments..., stream);
}

struct Cache {
  const at::Tensor *key, *value, *key_scale, *value_scale;
};
// The cache's four views, of 8 bits.
void check_int8(const char* what, const Cache& c) {
  if (c.key->scalar_type() != at::kChar || c.value->scalar_type() != at::kChar) refuse(what, ": the cache must be int8", PyExc_NotImplementedError);
  if (c.key_scale->scalar_type() != at::kFloat || c.value_scale->scalar_type() != at::kFloat)
    refuse(what, ": the scales must be fp32", PyExc_NotImplementedError);
  if (c.key->dim() != 4 || c.value->sizes() != c.key->sizes() || c.key_scale->sizes() != c.key->sizes().slice(0, 3) ||
      c.value_scale->sizes() != c.key_scale->sizes())
    refuse(what, ": cache views are (num_blocks, block_size, KV, D), scales (num_blocks, block_size, KV)");
  if (c.key->stride(3) != 1 || c.value->stride(3) != 1) refuse(what, ": the head dimension must be contiguous");
}
void check_rows(const char* what, const at::Tensor& key, const at::Tensor& value, const at::Tensor& cache) {
  if (key.dim() != 3 || value.sizes() != key.sizes() || key.sizes().slice(1) != cache.sizes().slice(2) ||
      value.scalar_type() != key.scalar_type())
    refuse(what, ": key and value are (tokens, KV, D) of one type");
  if (key.stride(2) != 1 || value.stride(2) != 1) refuse(what, ": the head dimension must be contiguous");
}
void check_table(const char* what, const at::Tensor& t) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1))
    refuse(what, ": block_table must be int32 with contiguous rows");
}

int prompt_attention(PyObject* const* a) {
  const char* what = "prompt_attention";
  const at::Tensor &q = *tensor(what, a[0]), &k = *tensor(what, a[1]), &v = *tensor(what, a[2]), &cu = *tensor(what, a[3]);
  const double scale = number(what, a[4]);
  const at::Tensor& out = *tensor(what, a[5]);
  check_gpu(what, {&q, &k, &v, &cu, &out}, "prompt_attention_torch");
  if (!is16(q) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    refuse(what, ": query, key and value must be all bf16 or all fp16", PyExc_NotImplementedError);
  if (cu.scalar_type() != at::kInt || cu.dim() != 1 || !cu.is_contiguous() || cu.size(0) == 0)
    refuse(what, ": cu_seqlens must be a contiguous int32 vector of the n + 1 starts");
  if (q.dim() != 3 || k.dim() != 3 || v.sizes() != k.sizes() || out.sizes() != q.sizes() || k.size(0) != q.size(0) ||
      k.size(2) != q.size(2) || k.size(1) == 0 || q.size(1) % k.size(1) != 0)
    refuse(what, ": inconsistent shapes");
  for (const at::Tensor* t : {&q, &k, &v, &out})
    if (t->size(2) && t->stride(2) != 1) refuse(what, ": the head dimension must be contiguous");
  const int out_dtype = dtype_enum(out);
  if (q.size(0) == 0) return VXA_OK;
  return on_device(q, prompt_attention_fn, ptr(&q), q.stride(0), q.stride(1), ptr(&k), k.stride(0), k.stride(1), ptr(&v), v.stride(0),
                   v.stride(1), dtype_enum(q), ptr<int32_t>(&cu), cu.size(0) - 1, q.size(0), (float)scale, ptr(&out), out_dtype,
                   out.stride(0), out.stride(1), q.size(1), k.size(1), q.size(2));
}

int write_cache(PyObject* const* a) {
  const char* what = "write_cache";
  const at::Tensor &k = *tensor(what, a[0]), &v = *tensor(what, a[1]);
  const Cache c{tensor(what, a[2]), tensor(what, a[3]), tensor(what, a[4]), tensor(what, a[5])};
  const at::Tensor& slots = *tensor(what, a[6]);
  check_gpu(what, {&k, &v, c.key, c.value, c.key_scale, c.value_scale, &slots}, "quantize_torch");
  check_int8(what, c);
  check_rows(what, k, v, *c.key);
  if (!vector_of(slots, at::kLong, k.size(0))) refuse(what, ": slot_mapping must be a contiguous int64 vector, one slot for each token");
  const int dtype = dtype_enum(k);
  if (k.size(0) == 0) return VXA_OK;
  const at::Tensor &kc = *c.key, &vc = *c.value, &ks = *c.key_scale, &vs = *c.value_scale;
  return on_device(k, cache_write_fn, ptr(&k), k.stride(0), k.stride(1), ptr(&v), v.stride(0), v.stride(1), dtype, k.size(0), k.size(1),
                   k.size(2), ptr<int8_t>(&kc), kc.stride(0), kc.stride(1), kc.stride(2), ptr<int8_t>(&vc), vc.stride(0), vc.stride(1),
                   vc.stride(2), ptr<float>(&ks), ks.stride(0), ks.stride(1), ks.stride(2), ptr<float>(&vs), vs.stride(0), vs.stride(1),
                   vs.stride(2), kc.size(0), kc.size(1), ptr<int64_t>(&slots));
}

int read_cache(PyObject* const* a) {
  const char* what = "read_cache";
  const Cache c{tensor(what, a[0]), tensor(what, a[1]), tensor(what, a[2]), tensor(what, a[3])};
  const at::Tensor &bt = *tensor(what, a[4]), &cu = *tensor(what, a[5]), &k = *tensor(what, a[6]), &v = *tensor(what, a[7]);
  const at::Tensor* first = tensor(what, a[8], true);
  check_gpu(what, {c.key, c.value, c.key_scale, c.value_scale, &bt, &cu, &k, &v, first}, "dequantize_torch");
  check_int8(what, c);
  check_rows(what, k, v, *c.key);
  check_table(what, bt);
  const int64_t n = bt.size(0);
  if (!vector_of(cu, at::kInt, n + 1)) refuse(what, ": cu_seqlens must be a contiguous int32 vector of the n + 1 starts");
  if (first && !vector_of(*first, at::kInt, n)) refuse(what, ": first must be a contiguous int32 vector, one token for each sequence");
  const int dtype = dtype_enum(k);
  if (k.size(0) == 0 || n == 0) return VXA_OK;
  const at::Tensor &kc = *c.key, &vc = *c.value, &ks = *c.key_scale, &vs = *c.value_scale;
  return on_device(k, cache_read_fn, ptr<int8_t>(&kc), kc.stride(0), kc.stride(1), kc.stride(2), ptr<int8_t>(&vc), vc.stride(0),
                   vc.stride(1), vc.stride(2), ptr<float>(&ks), ks.stride(0), ks.stride(1), ks.stride(2), ptr<float>(&vs), vs.stride(0),
                   vs.stride(1), vs.stride(2), kc.size(0), kc.size(1), ptr<int32_t>(&bt), bt.stride(0), bt.size(1), ptr<int32_t>(&cu),
                   ptr<int32_t>(first), n, k.size(0), k.size(1), k.size(2), ptr(&k), k.stride(0), k.stride(1), ptr(&v), v.stride(0),
                   v.stride(1), dtype);
}

int tree_decode(PyObject* const* a) {
  const char* what = "tree_decode";
  const at::Tensor& q = *tensor(what, a[0]);
  const Cache c{tensor(what, a[1]), tensor(what, a[2]), tensor(what, a[11], true), tensor(what, a[12], true)};
  const at::Tensor &bt = *tensor(what, a[3]), &sl = *tensor(what, a[4]), &qsl = *tensor(what, a[5]);
  const at::Tensor* mask = tensor(what, a[6], true);
  const double scale = number(what, a[7]);
  const at::Tensor& out = *tensor(what, a[8]);
  const int64_t max_nodes = integer(what, a[9]), max_len = integer(what, a[10]);
  check_gpu(what, {&q, c.key, c.value, &bt, &sl, &qsl, &out, mask, c.key_scale, c.value_scale}, "tree_decode_torch");
  if (!is16(q)) refuse(what, ": query must be bf16 or fp16", PyExc_NotImplementedError);
  if ((c.key_scale == nullptr) != (c.value_scale == nullptr)) refuse(what, ": key_scale and value_scale come together");
  const at::Tensor &kc = *c.key, &vc = *c.value;
  if (c.key_scale)
    check_int8(what, c);
  else if (kc.scalar_type() != q.scalar_type() || vc.scalar_type() != q.scalar_type())
    refuse(what, ": the cache must have the query's type, or be int8 with scales", PyExc_NotImplementedError);
  if (q.dim() != 3 || kc.dim() != 4 || vc.sizes() != kc.sizes() || out.sizes() != q.sizes() || kc.size(3) != q.size(2) ||
      kc.size(2) == 0 || q.size(1) % kc.size(2) != 0)
    refuse(what, ": inconsistent shapes");
  if (q.stride(2) != 1 || kc.stride(3) != 1 || vc.stride(3) != 1 || out.stride(2) != 1)
    refuse(what, ": the head dimension must be contiguous");
  check_table(what, bt);
  const int64_t n = bt.size(0), T = q.size(0), H = q.size(1), KV = kc.size(2), D = q.size(2);
  if (!vector_of(sl, at::kInt, n) || !vector_of(qsl, at::kInt, n + 1))
    refuse(what, ": seq_lens and query_start_loc must be contiguous int32 vectors, one length for each block-table row and the n + 1 starts");
  if (mask && !vector_of(*mask, at::kLong, T)) refuse(what, ": tree_mask must be a contiguous int64 vector, one mask for each node");
  if (max_nodes < 0 || max_len < 0) refuse(what, ": max_nodes and max_seq_len must be >= 0");
  if (max_nodes > 64)
    refuse(what, (": at most 64 nodes a request, got " + std::to_string(max_nodes)).c_str(), PyExc_NotImplementedError);
  const int out_dtype = dtype_enum(out);
  if (T == 0 || n == 0 || max_nodes == 0) return VXA_OK;
  size_t bytes = 0;
  const int rc = tree_workspace_fn(n, T, H, KV, D, max_nodes, max_len, &bytes);
  if (rc != VXA_OK) return rc;
  at::Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes / 4}, q.options().dtype(at::kFloat));
  const at::Tensor *ks = c.key_scale, *vs = c.value_scale;
  return on_device(q, tree_decode_fn, ptr(&q), q.stride(0), q.stride(1), dtype_enum(q), ptr(&kc), kc.stride(0), kc.stride(1),
                   kc.stride(2), ptr(&vc), vc.stride(0), vc.stride(1), vc.stride(2), ptr<float>(ks), stride(ks, 0), stride(ks, 1),
                   stride(ks, 2), ptr<float>(vs), stride(vs, 0), stride(vs, 1), stride(vs, 2), kc.size(0), kc.size(1), ptr<int32_t>(&bt),
                   bt.stride(0), bt.size(1), ptr<int32_t>(&sl), ptr<int32_t>(&qsl), ptr<int64_t>(mask), (float)scale, ptr(&out),
                   out_dtype, out.stride(0), out.stride(1), n, T, H, KV, D, max_nodes, max_len, bytes ? ptr(&ws) : nullptr, bytes);
}

// fn(arguments) as a Python function of `count` positional arguments; C++ exceptions end here, torch's as the Python exceptions
// that torch makes of them (OutOfMemoryError for a workspace that does not fit).
template <int (*fn)(PyObject* const*), int count>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t given) {
  if (given != count || !tree_decode_fn) {
    PyErr_SetString(PyExc_TypeError, given != count ? "wrong number of arguments" : "bind() has not been called");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  try {
    return PyLong_FromLong(fn(args));
  } catch (const Refused& r) {
    PyErr_SetString(r.kind, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind(prompt_attention, cache_write, cache_read, tree_workspace, tree_decode): the entry points' addresses.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t given) {
  void* at[5];
  if (given != 5) {
    PyErr_SetString(PyExc_TypeError, "bind() takes five addresses");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind(): null address");
      return nullptr;
    }
  }
  prompt_attention_fn = reinterpret_cast<decltype(prompt_attention_fn)>(at[0]);
  cache_write_fn = reinterpret_cast<decltype(cache_write_fn)>(at[1]);
  cache_read_fn = reinterpret_cast<decltype(cache_read_fn)>(at[2]);
  tree_workspace_fn = reinterpret_cast<decltype(tree_workspace_fn)>(at[3]);
  tree_decode_fn = reinterpret_cast<decltype(tree_decode_fn)>(at[4]);
  Py_RETURN_NONE;
}

#define VXA_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {VXA_METHOD("bind", bind),
                         VXA_METHOD("prompt_attention", (call<prompt_attention, 6>)),
                         VXA_METHOD("write_cache", (call<write_cache, 7>)),
                         VXA_METHOD("read_cache", (call<read_cache, 9>)),
                         VXA_METHOD("tree_decode", (call<tree_decode, 13>)),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_calls() { return PyModule_Create(&module); }
