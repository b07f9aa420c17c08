// The serving operators' calls on torch tensors: argument checks, pointers and strides, torch's current stream, and the C
// entry point, without a Python object for every stride. A call of 9 tensors spends 2 us here, where the same checks in
// Python and a ctypes call of 50 arguments took 15: a decode step makes such calls for every layer.
//
// The module holds no code of the kernels: bind() is given the addresses of the loaded library's entry points.
// Every function returns the entry point's status; what an argument check refuses is raised here.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <string>
#include <vector>

#include "../../include/vllm_exact_amd.h"

namespace {

decltype(&vxa_prompt_attention) prompt_attention_fn;
decltype(&vxa_int8_cache_write) cache_write_fn;
decltype(&vxa_int8_cache_read) cache_read_fn;
decltype(&vxa_tree_decode_call_workspace) tree_workspace_fn;
decltype(&vxa_tree_decode) tree_decode_fn;
decltype(&vxa_linear_prompt_workspace) linear_workspace_fn;
decltype(&vxa_linear_prompt) linear_prompt_fn;
decltype(&vxa_linear_step) linear_step_fn;
decltype(&vxa_beam_select_workspace) beam_workspace_fn;
decltype(&vxa_beam_select) beam_select_fn;
decltype(&vxa_pages_copy) pages_copy_fn;
decltype(&vxa_pages_fork_workspace) fork_workspace_fn;
decltype(&vxa_pages_fork) pages_fork_fn;
decltype(&vxa_pages_resize_workspace) resize_workspace_fn;
decltype(&vxa_pages_resize) pages_resize_fn;
decltype(&vxa_pages_keep) pages_keep_fn;

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

// A tensor's memory: runs of `bytes` from `start` on, at all sums of the dims' strides. (Strides are not negative.)
struct Memory {
  struct Dim {
    int64_t size, stride;  // bytes
  };
  int64_t start, bytes;
  c10::SmallVector<Dim, 6> dims;  // the widest first
  explicit Memory(const at::Tensor& t) : start((int64_t)(intptr_t)t.const_data_ptr()), bytes((int64_t)t.element_size()) {
    const int64_t item = bytes;
    for (int64_t i = 0; i < t.dim(); ++i)
      if (t.size(i) > 1) dims.push_back({t.size(i), t.stride(i) * item});
    std::sort(dims.begin(), dims.end(), [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
    for (; !dims.empty() && dims.back().stride <= bytes; dims.pop_back()) bytes += (dims.back().size - 1) * dims.back().stride;
  }
  int64_t extent(size_t from = 0) const {  // from the first byte to the one behind the last, of the dims from `from` on
    int64_t n = bytes;
    for (size_t i = from; i < dims.size(); ++i) n += (dims[i].size - 1) * dims[i].stride;
    return n;
  }
};
// Whether b's runs, `apart` bytes behind a's, meet them, without the widest i dims of a and j of b. Of the widest left the places are
// tried at which what is left of both meets: two, where rows and heads lie within each other. Layouts that take more than
// `steps` trials count as meeting.
bool meet(const Memory& a, size_t i, const Memory& b, size_t j, int64_t apart, int& steps) {
  if (--steps < 0) return true;
  const int64_t x = a.extent(i), y = b.extent(j);
  if (apart >= x || -apart >= y) return false;
  if (i == a.dims.size() && j == b.dims.size()) return true;
  const int64_t sa = i < a.dims.size() ? a.dims[i].stride : -1, sb = j < b.dims.size() ? b.dims[j].stride : -1, s = std::max(sa, sb);
  const int64_t most = sa == s ? a.dims[i].size - 1 : 0, least = sb == s ? 1 - b.dims[j].size : 0;  // places of a less those of b
  i += sa == s, j += sb == s;
  const int64_t p = a.extent(i), q = b.extent(j);
  auto up = [](int64_t n, int64_t d) { return n >= 0 ? (n + d - 1) / d : -(-n / d); };  // n / d rounded up
  for (int64_t k = std::max(least, up(apart - p + 1, s)); k <= most && k * s < apart + q; ++k)
    if (meet(a, i, b, j, apart - k * s, steps)) return true;
  return false;
}
struct Range {  // from the first byte to behind the last
  int64_t start, end;
  explicit Range(const at::Tensor& t) : start((int64_t)(intptr_t)t.const_data_ptr()), end(start) {
    if (t.numel() == 0) return;
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    end = start + (last + 1) * (int64_t)t.element_size();
  }
  bool apart(const Range& o) const { return start == end || o.start == o.end || end <= o.start || o.end <= start; }
};
// Whether two views of the same strides are rows beside each other, as keys and values in one buffer: a quick answer for most.
bool side_by_side(const at::Tensor& a, const at::Tensor& b) {
  const int64_t dims = a.dim(), size = a.element_size();
  if (dims < 2 || b.dim() != dims || b.element_size() != size) return false;
  int64_t step = INT64_MAX;  // all differences between the starts of two rows of one view are multiples of it
  for (int64_t i = 0; i + 1 < dims; ++i) {
    if (a.stride(i) != b.stride(i) || a.stride(i) == 0) return false;
    step = std::min(step, a.stride(i));
  }
  for (int64_t i = 0; i + 1 < dims; ++i)
    if (a.stride(i) % step != 0) return false;
  const int64_t x = (a.size(dims - 1) - 1) * a.stride(dims - 1) + 1, y = (b.size(dims - 1) - 1) * b.stride(dims - 1) + 1;  // a row's elements
  const int64_t bytes = (int64_t)(intptr_t)b.const_data_ptr() - (int64_t)(intptr_t)a.const_data_ptr(), apart = bytes / size;
  const int64_t behind = (apart % step + step) % step;
  return bytes % size == 0 && behind >= x && step - behind >= y;
}
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  if (Range(a).apart(Range(b)) || side_by_side(a, b)) return false;
  const Memory x(a), y(b);
  int steps = 1 << 14;
  return meet(x, 0, y, 0, y.start - x.start, steps);
}
// Outputs that other workgroups' inputs, or other outputs, lie in.
void check_apart(const char* what, const char* name, const at::Tensor& out, std::initializer_list<const at::Tensor*> others) {
  const Range range(out);
  for (const at::Tensor* t : others)
    if (t && !range.apart(Range(*t)) && overlap(out, *t)) refuse(what, (std::string(": ") + name + " must not be, or overlap, another argument").c_str());
}

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

// What linear_prompt and linear_step share; `states` may be null.
struct Linear {
  const at::Tensor &q, &k, &v, &decay, &out;
  double scale;
  const at::Tensor *state, *read, *write;
};
void check_linear(const char* what, const Linear& x, int64_t n, const at::Tensor* cu) {
  check_gpu(what, {&x.q, &x.k, &x.v, cu, &x.decay, &x.out, x.state, x.read, x.write}, "linear_attention_torch");
  if (!is16(x.q) || x.k.scalar_type() != x.q.scalar_type() || x.v.scalar_type() != x.q.scalar_type())
    refuse(what, ": query, key and value must be all bf16 or all fp16", PyExc_NotImplementedError);
  if (x.q.dim() != 3 || x.k.dim() != 3 || x.v.sizes() != x.k.sizes() || x.out.sizes() != x.q.sizes() || x.k.size(0) != x.q.size(0) ||
      x.k.size(2) != x.q.size(2) || x.k.size(1) == 0 || x.q.size(1) == 0 || x.q.size(1) % x.k.size(1) != 0)
    refuse(what, ": inconsistent shapes");
  for (const at::Tensor* t : {&x.q, &x.k, &x.v, &x.out})
    if (t->size(2) && t->stride(2) != 1) refuse(what, ": the head dimension must be contiguous");
  const int64_t H = x.q.size(1), D = x.q.size(2);
  if (!vector_of(x.decay, at::kFloat, H)) refuse(what, ": log_decay must be a contiguous fp32 vector, one number for each head");
  if ((x.read || x.write) && !x.state) refuse(what, ": slots need a pool of states");
  if (x.state) {
    const at::Tensor& s = *x.state;
    if (s.scalar_type() != at::kFloat) refuse(what, ": states must be fp32", PyExc_NotImplementedError);
    if (s.dim() != 4 || s.size(1) != H || s.size(2) != D || s.size(3) != D || s.stride(3) != 1 || s.stride(2) != D)
      refuse(what, ": states are (slots, H, D, D), each matrix contiguous");
    if (x.write && s.numel()) {  // a workgroup writes each matrix
      const bool slots_inside = s.stride(0) < s.stride(1);
      const int64_t size = D * D, inner = s.size(slots_inside ? 0 : 1), inner_stride = s.stride(slots_inside ? 0 : 1), wide = s.stride(slots_inside ? 1 : 0);
      if ((inner > 1 && inner_stride < size) || (s.size(slots_inside ? 1 : 0) > 1 && wide < (inner - 1) * inner_stride + size))
        refuse(what, ": states must not overlap each other");
      check_apart(what, "state", s, {&x.q, &x.k, &x.v, cu, &x.decay, x.read, x.write});
    }
  }
  for (const at::Tensor* t : {x.read, x.write})
    if (t && !vector_of(*t, at::kInt, n)) refuse(what, ": slots must be contiguous int32 vectors, one for each sequence");
  // Workgroups read rows whose outputs others have written.
  check_apart(what, "out", x.out, {&x.q, &x.k, &x.v, cu, &x.decay, x.state, x.read, x.write});
}

int linear_prompt(PyObject* const* a) {
  const char* what = "linear_prompt";
  const at::Tensor& cu = *tensor(what, a[3]);
  const Linear x{*tensor(what, a[0]),   *tensor(what, a[1]),       *tensor(what, a[2]),       *tensor(what, a[4]),      *tensor(what, a[6]),
                 number(what, a[5]), tensor(what, a[7], true), tensor(what, a[8], true), tensor(what, a[9], true)};
  if (cu.scalar_type() != at::kInt || cu.dim() != 1 || !cu.is_contiguous() || cu.size(0) == 0)
    refuse(what, ": cu_seqlens must be a contiguous int32 vector of the n + 1 starts");
  const int64_t n = cu.size(0) - 1;
  check_linear(what, x, n, &cu);
  const int out_dtype = dtype_enum(x.out);
  const int64_t T = x.q.size(0), H = x.q.size(1), D = x.q.size(2);
  if (n == 0) return VXA_OK;
  size_t bytes = 0;
  const int rc = linear_workspace_fn(T, H, D, &bytes);
  if (rc != VXA_OK) return rc;
  at::Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes / 4}, x.q.options().dtype(at::kFloat));
  return on_device(x.q, linear_prompt_fn, ptr(&x.q), x.q.stride(0), x.q.stride(1), ptr(&x.k), x.k.stride(0), x.k.stride(1), ptr(&x.v),
                   x.v.stride(0), x.v.stride(1), dtype_enum(x.q), ptr<int32_t>(&cu), n, T, ptr<float>(&x.decay), (float)x.scale, ptr(&x.out),
                   out_dtype, x.out.stride(0), x.out.stride(1), ptr<float>(x.state), x.state ? x.state->size(0) : 0, stride(x.state, 0),
                   stride(x.state, 1), ptr<int32_t>(x.read), ptr<int32_t>(x.write), H, x.k.size(1), D, bytes ? ptr(&ws) : nullptr, bytes);
}

int linear_step(PyObject* const* a) {
  const char* what = "linear_step";
  const Linear x{*tensor(what, a[0]),   *tensor(what, a[1]), *tensor(what, a[2]),       *tensor(what, a[3]),      *tensor(what, a[5]),
                 number(what, a[4]), tensor(what, a[6]),  tensor(what, a[7], true), tensor(what, a[8], true)};
  check_linear(what, x, x.q.dim() ? x.q.size(0) : 0, nullptr);
  const int out_dtype = dtype_enum(x.out);
  const int64_t n = x.q.size(0);
  if (n == 0) return VXA_OK;
  return on_device(x.q, linear_step_fn, ptr(&x.q), x.q.stride(0), x.q.stride(1), ptr(&x.k), x.k.stride(0), x.k.stride(1), ptr(&x.v),
                   x.v.stride(0), x.v.stride(1), dtype_enum(x.q), n, ptr<float>(&x.decay), (float)x.scale, ptr(&x.out), out_dtype,
                   x.out.stride(0), x.out.stride(1), ptr<float>(x.state), x.state->size(0), x.state->stride(0), x.state->stride(1),
                   ptr<int32_t>(x.read), ptr<int32_t>(x.write), x.q.size(1), x.k.size(1), x.q.size(2));
}

int beam_select(PyObject* const* a) {
  const char* what = "beam_select";
  const at::Tensor &x = *tensor(what, a[0]), &scores = *tensor(what, a[1]);
  const int64_t beams = integer(what, a[2]);
  const at::Tensor &best = *tensor(what, a[3]), &parents = *tensor(what, a[4]), &tokens = *tensor(what, a[5]);
  check_gpu(what, {&x, &scores, &best, &parents, &tokens}, "beam_select_torch");
  const int dtype = dtype_enum(x);
  if (beams <= 0 || x.dim() != 2 || x.size(0) % beams != 0) refuse(what, ": logits are (requests * beams, vocabulary)");
  if (x.size(1) > 1 && x.stride(1) != 1) refuse(what, ": the vocabulary must be contiguous");
  const int64_t n = x.size(0) / beams, V = x.size(1);
  if (!vector_of(scores, at::kFloat, x.size(0))) refuse(what, ": scores must be a contiguous fp32 vector, one for each row of logits");
  if (best.scalar_type() != at::kFloat || parents.scalar_type() != at::kInt || tokens.scalar_type() != at::kLong || best.dim() != 2 ||
      best.size(0) != n || best.size(1) == 0 || parents.sizes() != best.sizes() || tokens.sizes() != best.sizes() || !best.is_contiguous() ||
      !parents.is_contiguous() || !tokens.is_contiguous())
    refuse(what, ": out_scores (fp32), out_parents (int32) and out_tokens (int64) are contiguous (requests, count)");
  // A request's workgroup reads its scores before it writes as many in their place; with another count they would be others'.
  const bool in_place = best.const_data_ptr() == scores.const_data_ptr() && best.numel() == scores.numel();
  check_apart(what, "out_scores", best, {&x, in_place ? nullptr : &scores, &parents, &tokens});
  check_apart(what, "out_parents", parents, {&x, &scores, &tokens});
  check_apart(what, "out_tokens", tokens, {&x, &scores});
  if (n == 0) return VXA_OK;
  size_t bytes = 0;
  const int rc = beam_workspace_fn(n, beams, V, best.size(1), &bytes);
  if (rc != VXA_OK) return rc;
  const at::Tensor ws = at::empty({(int64_t)bytes / 4}, x.options().dtype(at::kFloat));
  return on_device(x, beam_select_fn, ptr(&x), x.stride(0), dtype, ptr<float>(&scores), n, beams, V, best.size(1), ptr<float>(&best),
                   ptr<int32_t>(&parents), ptr<int64_t>(&tokens), ptr(&ws), bytes);
}

// The tensors of a cache, views (num_blocks, block_size, KV, D) or (num_blocks, block_size, KV), as the library takes them.
struct Caches {
  std::vector<vxa_cache_view> views;
  int64_t num_blocks = 0;
};
// apart: refused if they have memory in common, which is then moved twice.
Caches caches_of(const char* what, PyObject* o, int64_t page, const at::Tensor& beside, bool apart = false) {
  PyObject* const list = PySequence_Fast(o, "");
  if (!list) {
    PyErr_Clear();
    refuse(what, ": caches must be a list of tensors", PyExc_TypeError);
  }
  const THPObjectPtr kept(list);
  Caches c;
  std::vector<std::pair<Range, const at::Tensor*>> ranges;
  c.num_blocks = -1;
  c.views.reserve(PySequence_Fast_GET_SIZE(list));
  if (apart) ranges.reserve(PySequence_Fast_GET_SIZE(list));
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(list); ++i) {
    const at::Tensor& t = *tensor(what, PySequence_Fast_GET_ITEM(list, i));
    check_gpu(what, {&beside, &t}, "the torch statements of pages.py");
    if ((t.dim() != 3 && t.dim() != 4) || t.size(1) != page || (t.dim() == 4 && t.size(3) > 1 && t.stride(3) != 1))
      refuse(what, ": caches are views (num_blocks, block_size, KV, D) or (num_blocks, block_size, KV), D contiguous");
    if (c.num_blocks >= 0 && t.size(0) != c.num_blocks) refuse(what, ": all caches must have the same blocks");
    c.num_blocks = t.size(0);
    const int64_t size = t.element_size();
    if (apart && t.numel()) {
      for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1 && t.stride(d) == 0) refuse(what, ": caches must not be expanded views");
      const Range range(t);
      for (size_t j = 0; j < ranges.size(); ++j)
        if (!range.apart(ranges[j].first) && overlap(t, *ranges[j].second)) refuse(what, ": caches must not have memory in common");
      ranges.emplace_back(range, &t);
    }
    if (t.numel())
      c.views.push_back({t.data_ptr(), t.stride(0) * size, t.stride(1) * size, t.stride(2) * size, t.size(2), (t.dim() == 4 ? t.size(3) : 1) * size});
  }
  return c;
}
int64_t block_size(const char* what, PyObject* o) {
  const int64_t page = integer(what, o);
  if (page <= 0) refuse(what, ": block_size must be positive");
  return page;
}
void check_counts(const char* what, const at::Tensor& refs, const at::Tensor& out) {
  for (const at::Tensor* t : {&refs, &out})
    if (!vector_of(*t, at::kInt, refs.dim() ? refs.size(0) : 0)) refuse(what, ": ref_count must be a contiguous int32 vector, one count for each block");
}
void check_tables(const char* what, const at::Tensor& table, const at::Tensor& out) {
  check_table(what, table);
  check_table(what, out);
  if (out.size(1) != table.size(1)) refuse(what, ": the tables must have the same columns");
  if (out.size(0) > 1 && out.stride(0) < out.size(1)) refuse(what, ": the new table's rows must not overlap");
}
// Counts in their own place, or apart.
void check_new_counts(const char* what, const at::Tensor& refs, const at::Tensor& out, std::initializer_list<const at::Tensor*> others) {
  if (out.const_data_ptr() != refs.const_data_ptr()) check_apart(what, "out_ref_count", out, {&refs});
  check_apart(what, "out_ref_count", out, others);
}

int copy_pages(PyObject* const* a) {
  const char* what = "copy_pages";
  const int64_t page = block_size(what, a[1]);
  const at::Tensor &source = *tensor(what, a[2]), &target = *tensor(what, a[3]);
  check_gpu(what, {&source, &target}, "the torch statements of pages.py");
  const Caches c = caches_of(what, a[0], page, source);
  const int64_t n = source.dim() == 1 ? source.size(0) : -1;
  if (!vector_of(source, at::kInt, n) || !vector_of(target, at::kInt, n)) refuse(what, ": source and target must be contiguous int32 vectors of one length");
  if (n == 0 || c.views.empty()) return VXA_OK;
  return on_device(source, pages_copy_fn, c.views.data(), (int64_t)c.views.size(), c.num_blocks, page, ptr<int32_t>(&source), ptr<int32_t>(&target), n);
}

int fork_pages(PyObject* const* a) {
  const char* what = "fork_pages";
  const at::Tensor &bt = *tensor(what, a[1]), &sl = *tensor(what, a[2]), &parents = *tensor(what, a[3]), &refs = *tensor(what, a[4]);
  const int64_t page = block_size(what, a[5]);
  const at::Tensor &out = *tensor(what, a[6]), &out_lens = *tensor(what, a[7]), &out_refs = *tensor(what, a[8]), &missing = *tensor(what, a[9]);
  check_gpu(what, {&bt, &sl, &parents, &refs, &out, &out_lens, &out_refs, &missing}, "fork_pages_torch");
  const Caches c = caches_of(what, a[0], page, bt);
  check_tables(what, bt, out);
  check_counts(what, refs, out_refs);
  if (c.num_blocks >= 0 && c.num_blocks != refs.size(0)) refuse(what, ": ref_count must have a count for each block of the caches");
  const int64_t rows = bt.size(0), many = out.size(0);
  if (!vector_of(sl, at::kInt, rows) || !vector_of(parents, at::kInt, many) || !vector_of(out_lens, at::kInt, many))
    refuse(what, ": seq_lens, parents and out_lens must be contiguous int32 vectors, one number for each row of their table");
  if (!vector_of(missing, at::kInt, 1)) refuse(what, ": missing must be one int32 number");
  size_t bytes = 0;
  const int rc = fork_workspace_fn(rows, many, &bytes);
  if (rc != VXA_OK) return rc;
  // Rows read each other's pages and lengths while others are written.
  check_apart(what, "out_table", out, {&bt, &sl, &parents, &refs, &out_lens, &out_refs, &missing});
  check_apart(what, "out_lens", out_lens, {&bt, &sl, &parents, &refs, &out_refs, &missing});
  check_new_counts(what, refs, out_refs, {&bt, &sl, &parents, &missing});
  at::Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes / 4}, bt.options());
  return on_device(bt, pages_fork_fn, c.views.data(), (int64_t)c.views.size(), ptr<int32_t>(&bt), bt.stride(0), bt.size(1), ptr<int32_t>(&sl), rows,
                   ptr<int32_t>(&parents), many, ptr<int32_t>(&refs), refs.size(0), page, ptr<int32_t>(&out), out.stride(0),
                   ptr<int32_t>(&out_lens), ptr<int32_t>(&out_refs), ptr<int32_t>(&missing), bytes ? ptr(&ws) : nullptr, bytes);
}

int resize_pages(PyObject* const* a) {
  const char* what = "resize_pages";
  const at::Tensor &bt = *tensor(what, a[0]), &sl = *tensor(what, a[1]), &lens = *tensor(what, a[2]), &refs = *tensor(what, a[3]);
  const int64_t page = block_size(what, a[4]);
  const at::Tensor &out = *tensor(what, a[5]), &out_refs = *tensor(what, a[6]), &missing = *tensor(what, a[7]);
  check_gpu(what, {&bt, &sl, &lens, &refs, &out, &out_refs, &missing}, "resize_pages_torch");
  check_tables(what, bt, out);
  check_counts(what, refs, out_refs);
  const int64_t rows = bt.size(0);
  if (out.size(0) != rows) refuse(what, ": the tables must have the same rows");
  if (!vector_of(sl, at::kInt, rows) || !vector_of(lens, at::kInt, rows))
    refuse(what, ": seq_lens and new_lens must be contiguous int32 vectors, one length for each row");
  if (!vector_of(missing, at::kInt, 1)) refuse(what, ": missing must be one int32 number");
  size_t bytes = 0;
  const int rc = resize_workspace_fn(rows, refs.size(0), &bytes);
  if (rc != VXA_OK) return rc;
  const bool in_place = out.const_data_ptr() == bt.const_data_ptr() && (rows <= 1 || out.stride(0) == bt.stride(0));
  check_apart(what, "out_table", out, {in_place ? nullptr : &bt, &sl, &lens, &refs, &out_refs, &missing});
  check_new_counts(what, refs, out_refs, {&bt, &sl, &lens, &missing});
  const at::Tensor ws = at::empty({(int64_t)bytes / 4}, bt.options());
  return on_device(bt, pages_resize_fn, ptr<int32_t>(&bt), bt.stride(0), bt.size(1), ptr<int32_t>(&sl), ptr<int32_t>(&lens), rows,
                   ptr<int32_t>(&refs), refs.size(0), page, ptr<int32_t>(&out), out.stride(0), ptr<int32_t>(&out_refs), ptr<int32_t>(&missing),
                   ptr(&ws), bytes);
}

// Whether two tensors have memory in common, for tests.
PyObject* overlap_of(PyObject*, PyObject* const* args, Py_ssize_t given) {
  HANDLE_TH_ERRORS
  if (given != 2 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "overlap() takes two tensors");
    return nullptr;
  }
  return PyBool_FromLong(overlap(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1])));
  END_HANDLE_TH_ERRORS
}

int keep_drafted(PyObject* const* a) {
  const char* what = "keep_drafted";
  const at::Tensor &bt = *tensor(what, a[1]), &sl = *tensor(what, a[2]), &qsl = *tensor(what, a[3]), &keep = *tensor(what, a[4]);
  const int64_t page = block_size(what, a[5]);
  const at::Tensor& out_lens = *tensor(what, a[6]);
  check_gpu(what, {&bt, &sl, &qsl, &keep, &out_lens}, "keep_drafted_torch");
  const Caches c = caches_of(what, a[0], page, bt, true);
  check_table(what, bt);
  const int64_t n = bt.size(0);
  if (!vector_of(sl, at::kInt, n) || !vector_of(qsl, at::kInt, n + 1) || !vector_of(out_lens, at::kInt, n))
    refuse(what, ": seq_lens, query_start_loc and out_lens must be contiguous int32 vectors, one length for each block-table row and the n + 1 starts");
  if (!vector_of(keep, at::kLong, n)) refuse(what, ": keep must be a contiguous int64 vector, one mask for each request");
  check_apart(what, "out_lens", out_lens, {&bt, &sl, &qsl, &keep});
  if (n == 0) return VXA_OK;
  return on_device(bt, pages_keep_fn, c.views.data(), (int64_t)c.views.size(), ptr<int32_t>(&bt), bt.stride(0), bt.size(1), ptr<int32_t>(&sl),
                   ptr<int32_t>(&qsl), ptr<int64_t>(&keep), n, std::max<int64_t>(c.num_blocks, 0), page, ptr<int32_t>(&out_lens));
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

// bind(addresses): the entry points', in the order of _native.py's _CALLED.
template <typename F>
void take(F& fn, PyObject* address) {
  fn = reinterpret_cast<F>(PyLong_AsVoidPtr(address));
}
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t given) {
  constexpr int kEntries = 16;
  if (given != kEntries) {
    PyErr_SetString(PyExc_TypeError, "bind() takes sixteen addresses");
    return nullptr;
  }
  for (int i = 0; i < kEntries; ++i)
    if (!PyLong_AsVoidPtr(args[i])) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind(): null address");
      return nullptr;
    }
  PyObject* const* next = args;
  take(prompt_attention_fn, *next++), take(cache_write_fn, *next++), take(cache_read_fn, *next++), take(tree_workspace_fn, *next++);
  take(tree_decode_fn, *next++), take(linear_workspace_fn, *next++), take(linear_prompt_fn, *next++), take(linear_step_fn, *next++);
  take(beam_workspace_fn, *next++), take(beam_select_fn, *next++), take(pages_copy_fn, *next++), take(fork_workspace_fn, *next++);
  take(pages_fork_fn, *next++), take(resize_workspace_fn, *next++), take(pages_resize_fn, *next++), take(pages_keep_fn, *next++);
  Py_RETURN_NONE;
}

#define VXA_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {VXA_METHOD("bind", bind),
                         VXA_METHOD("overlap", overlap_of),
                         VXA_METHOD("prompt_attention", (call<prompt_attention, 6>)),
                         VXA_METHOD("write_cache", (call<write_cache, 7>)),
                         VXA_METHOD("read_cache", (call<read_cache, 9>)),
                         VXA_METHOD("tree_decode", (call<tree_decode, 13>)),
                         VXA_METHOD("linear_prompt", (call<linear_prompt, 10>)),
                         VXA_METHOD("linear_step", (call<linear_step, 9>)),
                         VXA_METHOD("beam_select", (call<beam_select, 6>)),
                         VXA_METHOD("copy_pages", (call<copy_pages, 4>)),
                         VXA_METHOD("fork_pages", (call<fork_pages, 10>)),
                         VXA_METHOD("resize_pages", (call<resize_pages, 8>)),
                         VXA_METHOD("keep_drafted", (call<keep_drafted, 7>)),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_calls() { return PyModule_Create(&module); }
