// Python binding of the operators around a key/value cache in pages (vla_ops.py documents them): checks of the tensors,
// outputs and workspaces from torch's allocator, the current stream, then the C entry point.  The smallest calls take three to ten
// microseconds on the GPU; here the host needs 5 to 10 for each, of which the launch is 3, and through ctypes it needed 11 to 19.
#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <climits>
#include <cmath>
#include <string>

#include "../../include/vla_b200.h"

namespace {

PyObject* capi;          // the module _capi: its VlaError and check()
PyObject* error_type;

struct Refusal {
  std::string text;
};
struct Raised {};        // the Python error is set
std::string text(const char* s) { return s; }
std::string text(int64_t n) { return std::to_string(n); }
std::string text(at::ScalarType type) { return at::toString(type); }
std::string text(c10::Device device) { return device.str(); }
std::string text(at::IntArrayRef sizes) {
  std::string s = "(";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + ")";
}
std::string text(const at::Tensor& t) { return text(t.scalar_type()) + " " + text(t.sizes()) + " on " + text(t.device()); }
template <typename... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
  throw Refusal{"vla_ops: " + (text(parts) + ...)};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, " must be a tensor");
  return THPVariable_Unpack(o);
}
int number(int64_t n, const char* name) {
  if (n > INT_MAX || n < INT_MIN) refuse(name, " is too large: ", n);
  return (int)n;
}
int number(PyObject* o, const char* name) {
  const long long n = PyLong_AsLongLong(o);
  if (n == -1 && PyErr_Occurred()) throw Raised{};
  return number((int64_t)n, name);
}
float scale_of(PyObject* o, int64_t dim) {
  if (o == Py_None) return (float)(1.0 / std::sqrt((double)dim));
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw Raised{};
  return (float)x;
}
// the stride of a dimension of one element, which may be anything, is never used
int64_t step(const at::Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; }
bool rows_contiguous(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) <= 1; }

// An int32 tensor of `dim` dimensions on `device` with contiguous rows
const at::Tensor& whole(PyObject* o, const char* name, c10::Device device, int dim = 1) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.dim() != dim || t.device() != device || !rows_contiguous(t))
    refuse(name, " must be int32 with ", (int64_t)dim, " dimension(s), contiguous rows, on ", device, "; got ", t);
  return t;
}
const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }

// Neither a gradient nor a tangent of an argument may be lost on the way
void no_gradient(const at::Tensor& t, const char* name) {
  if (t.requires_grad() && c10::GradMode::is_enabled()) refuse(name, " requires a gradient; this operator has no backward pass");
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()) refuse(name, " has a tangent; this operator has no forward-mode gradient");
}
// What an operator has written: autograd's saved copies of it are out of date.  Tensors of inference mode keep no count.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A 16-bit tensor of `dim` dimensions on `device` whose last one is contiguous
const at::Tensor& rows(PyObject* o, const char* name, c10::Device device, at::ScalarType type, int dim) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type || t.dim() != dim || t.device() != device || !rows_contiguous(t))
    refuse(name, " must be ", type, " with ", (int64_t)dim, " dimensions, the last one contiguous, on ", device, "; got ", t);
  no_gradient(t, name);
  return t;
}
int type_code(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return VLA_BF16;
  if (t.scalar_type() == at::kHalf) return VLA_F16;
  refuse(name, " must be bfloat16 or float16, got ", t.scalar_type());
}
const at::Tensor& on_gpu(PyObject* o, const char* name) {
  const at::Tensor& t = tensor(o, name);
  if (!t.is_cuda()) refuse(name, " must be on a GPU; there is no CPU path");
  return t;
}

struct Cache {
  const at::Tensor *k, *v, *ks, *vs;
};
Cache cache_of(PyObject* o, c10::Device device) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse("cache must be a KvCache");
  const Cache c{&tensor(PyTuple_GET_ITEM(o, 0), "cache.k"), &tensor(PyTuple_GET_ITEM(o, 1), "cache.v"),
                &tensor(PyTuple_GET_ITEM(o, 2), "cache.k_scale"), &tensor(PyTuple_GET_ITEM(o, 3), "cache.v_scale")};
  auto part = [&](const at::Tensor& t, at::ScalarType type, int dim) {
    return t.scalar_type() == type && t.dim() == dim && t.device() == device && t.is_contiguous() &&
           (dim == 4 ? t.sizes() == c.k->sizes() : t.size(0) == c.k->size(0) && t.size(1) == c.k->size(1));
  };
  if (!(part(*c.k, at::kFloat8_e4m3fn, 4) && part(*c.v, at::kFloat8_e4m3fn, 4) && part(*c.ks, at::kFloat, 2) && part(*c.vs, at::kFloat, 2)))
    refuse("a cache is float8_e4m3fn codes [blocks, kv_heads, block_size, head_dim] twice and float32 scales [blocks, kv_heads] twice, "
           "all contiguous and on ", device, "; got ", *c.k, ", ", *c.v, ", ", *c.ks, ", ", *c.vs);
  no_gradient(*c.k, "cache.k");
  no_gradient(*c.v, "cache.v");
  no_gradient(*c.ks, "cache.k_scale");
  no_gradient(*c.vs, "cache.v_scale");
  return c;
}

// The C entry point on the current stream of the tensors' device
template <typename Desc>
void enqueue(int (*fn)(const Desc*, void*), const Desc& d, c10::Device device) {
  const c10::cuda::CUDAGuard guard(device);
  const int rc = fn(&d, c10::cuda::getCurrentCUDAStream(device.index()).stream());
  if (rc) {
    THPObjectPtr none(PyObject_CallMethod(capi, "check", "i", rc));
    if (!none) throw Raised{};
  }
}

// Whether two tensors have an element in common, of which nothing is known only where their layouts do not fit each other.
bool apart(const at::Tensor& a, const at::Tensor& b) {
  if (!a.numel() || !b.numel()) return true;
  // bytes from the first element to behind the last one, of the dimensions whose stride is below `s` bytes
  auto extent = [](const at::Tensor& t, int64_t s) {
    int64_t n = t.element_size();
    for (int64_t i = 0; i < t.dim(); ++i)
      if (t.size(i) > 1 && t.stride(i) * (int64_t)t.element_size() < s) n += (t.size(i) - 1) * t.stride(i) * t.element_size();
    return n;
  };
  const int64_t at_a = (int64_t)a.const_data_ptr(), at_b = (int64_t)b.const_data_ptr();
  if (at_a + extent(a, INT64_MAX) <= at_b || at_b + extent(b, INT64_MAX) <= at_a) return true;
  // parts of rows of s bytes: slices of one buffer
  for (int64_t i = 0; i < a.dim(); ++i) {
    const int64_t s = a.stride(i) * a.element_size();
    if (a.size(i) < 2 || s <= 0) continue;
    bool rows = true;
    for (const at::Tensor* t : {&a, &b})
      for (int64_t k = 0; k < t->dim(); ++k)
        if (t->size(k) > 1 && t->stride(k) * (int64_t)t->element_size() >= s && t->stride(k) * (int64_t)t->element_size() % s) rows = false;
    const int64_t from = ((at_b - at_a) % s + s) % s;
    if (rows && extent(a, s) <= from && from + extent(b, s) <= s) return true;
  }
  return false;
}
bool same_place(const at::Tensor& a, const at::Tensor& b) {
  if (a.const_data_ptr() != b.const_data_ptr()) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

// out, or a new tensor like q.  It may be q itself: a row of q has been read by all that read it when it is written.
at::Tensor output(PyObject* o, const at::Tensor& q) {
  if (o == Py_None) return at::empty(q.sizes(), q.options());
  const at::Tensor& t = rows(o, "out", q.device(), q.scalar_type(), (int)q.dim());
  if (t.sizes() != q.sizes()) refuse("out must have the shape of q");
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.stride(i) == 0 && t.size(i) > 1) refuse("out is expanded: several of its elements are one place in memory");
  if (!same_place(t, q) && !apart(t, q)) refuse("out overlaps q without being q");
  return t;
}

PyObject* block_plan(PyObject* const* a) {      // context_lens, new_lens, block_table, free_blocks, block_size, total_new, first_free
  const at::Tensor& context = on_gpu(a[0], "context_lens");
  const c10::Device dev = context.device();
  whole(a[0], "context_lens", dev);
  const at::Tensor& fresh = whole(a[1], "new_lens", dev);
  const at::Tensor& table = whole(a[2], "block_table", dev, 2);
  const at::Tensor& free_ids = whole(a[3], "free_blocks", dev);
  const int32_t* first = nullptr;
  if (a[6] != Py_None) {
    const at::Tensor& t = whole(a[6], "first_free", dev);
    if (t.numel() != 1) refuse("first_free must have one element");
    first = ints(t);
  }
  const int64_t n = context.size(0), total = number(a[5], "total_new");
  if (fresh.size(0) != n || table.size(0) != n) refuse("context_lens, new_lens and block_table do not fit each other");
  if (total < 0) refuse("total_new is negative");
  vla_block_plan_desc d{};
  d.context_lens = ints(context); d.new_lens = ints(fresh); d.n_seqs = number(n, "context_lens");
  d.block_table = static_cast<int32_t*>(table.data_ptr()); d.width = number(table.size(1), "block_table");
  d.table_stride = n > 1 ? table.stride(0) : table.size(1);
  d.free_blocks = ints(free_ids); d.n_free = number(free_ids.size(0), "free_blocks"); d.first_free = first;
  d.block_size = number(a[4], "block_size"); d.total_new = (int)total;
  const int64_t room = (total + 3) / 4 * 4;     // one allocation, of which slots and positions start on 16 bytes
  const at::Tensor out = at::empty({2 * room + 2 * n + 4}, context.options());
  const int64_t start[5] = {0, room, 2 * room, 2 * room + n + 1, 2 * room + 2 * n + 1}, length[5] = {total, total, n + 1, n, 3};
  int32_t* const base = static_cast<int32_t*>(out.data_ptr());
  d.slots = base; d.positions = base + start[1]; d.cu_new = base + start[2]; d.seq_lens = base + start[3]; d.counts = base + start[4];
  enqueue(vla_op_block_plan, d, dev);
  written(table);
  const at::AutoDispatchBelowADInplaceOrView plain;     // integers: views that autograd need not know of
  THPObjectPtr result(PyTuple_New(5));
  if (!result) throw Raised{};
  for (int i = 0; i < 5; ++i) {
    PyObject* part = THPVariable_Wrap(out.slice(0, start[i], start[i] + length[i]));
    if (!part) throw Raised{};
    PyTuple_SET_ITEM(result.get(), i, part);
  }
  return result.release();
}

PyObject* cache_append(PyObject* const* a) {    // k, v, cache, slots
  const at::Tensor& k = on_gpu(a[0], "k");
  const c10::Device dev = k.device();
  vla_cache_append_desc d{};
  d.dtype = type_code(k, "k");
  rows(a[0], "k", dev, k.scalar_type(), 3);
  const at::Tensor& v = rows(a[1], "v", dev, k.scalar_type(), 3);
  const Cache c = cache_of(a[2], dev);
  const at::Tensor& slots = whole(a[3], "slots", dev);
  if (k.sizes() != v.sizes() || k.size(1) != c.k->size(1) || k.size(2) != c.k->size(3) || slots.size(0) != k.size(0))
    refuse("k ", k.sizes(), ", v ", v.sizes(), " and slots ", slots.sizes(), " do not fit the cache ", c.k->sizes());
  d.k = k.const_data_ptr(); d.v = v.const_data_ptr(); d.slots = ints(slots); d.tokens = number(k.size(0), "k");
  d.k_tok_stride = step(k, 0); d.k_head_stride = step(k, 1); d.v_tok_stride = step(v, 0); d.v_head_stride = step(v, 1);
  d.k_codes = c.k->data_ptr(); d.v_codes = c.v->data_ptr();
  d.k_scale = static_cast<float*>(c.ks->data_ptr()); d.v_scale = static_cast<float*>(c.vs->data_ptr());
  d.num_blocks = number(c.k->size(0), "cache"); d.kv_heads = number(c.k->size(1), "cache");
  d.block_size = number(c.k->size(2), "cache"); d.head_dim = number(c.k->size(3), "cache");
  enqueue(vla_op_cache_append, d, dev);
  for (const at::Tensor* t : {c.k, c.v, c.ks, c.vs}) written(*t);
  Py_RETURN_NONE;
}

PyObject* paged_attention(PyObject* const* a) { // q, cache, block_table, seq_lens, scale, out
  const at::Tensor& q = on_gpu(a[0], "q");
  const c10::Device dev = q.device();
  vla_paged_attn_desc d{};
  d.dtype = type_code(q, "q");
  rows(a[0], "q", dev, q.scalar_type(), 4);
  const Cache c = cache_of(a[1], dev);
  const at::Tensor& table = whole(a[2], "block_table", dev, 2);
  const at::Tensor& lens = whole(a[3], "seq_lens", dev);
  if (q.size(3) != c.k->size(3) || table.size(0) != q.size(0) || lens.size(0) != q.size(0))
    refuse("q ", q.sizes(), ", block_table ", table.sizes(), ", seq_lens ", lens.sizes(), " and cache ", c.k->sizes(), " do not fit each other");
  const at::Tensor out = output(a[5], q);
  d.q = q.const_data_ptr(); d.o = out.data_ptr();
  d.q_seq_stride = step(q, 0); d.q_tok_stride = step(q, 1); d.q_head_stride = step(q, 2);
  d.o_seq_stride = step(out, 0); d.o_tok_stride = step(out, 1); d.o_head_stride = step(out, 2);
  d.k_codes = c.k->const_data_ptr(); d.v_codes = c.v->const_data_ptr();
  d.k_scale = static_cast<const float*>(c.ks->const_data_ptr()); d.v_scale = static_cast<const float*>(c.vs->const_data_ptr());
  d.block_table = ints(table); d.width = number(table.size(1), "block_table"); d.table_stride = q.size(0) > 1 ? table.stride(0) : table.size(1);
  d.seq_lens = ints(lens);
  d.n_seqs = number(q.size(0), "q"); d.n_q = number(q.size(1), "q"); d.heads = number(q.size(2), "q");
  d.kv_heads = number(c.k->size(1), "cache"); d.head_dim = number(q.size(3), "q");
  d.num_blocks = number(c.k->size(0), "cache"); d.block_size = number(c.k->size(2), "cache");
  d.scale = scale_of(a[4], q.size(3));
  // the workspace is this call's own; the allocator orders its reuse on the stream
  at::Tensor space;
  {
    const c10::cuda::CUDAGuard guard(dev);      // its size follows from the sizes and the device's number of SMs
    if (vla_op_paged_attention_workspace(&d, &d.workspace_bytes) == 0 && d.workspace_bytes) {
      space = at::empty({(int64_t)d.workspace_bytes}, q.options().dtype(at::kByte));
      d.workspace = space.data_ptr();
    }
  }
  enqueue(vla_op_paged_attention, d, dev);      // refuses what the size was refused for, too
  if (a[5] != Py_None) written(out);
  return THPVariable_Wrap(out);
}

PyObject* prompt_attention(PyObject* const* a) {        // q, k, v, cu_q, cu_k, causal, scale, out
  const at::Tensor& q = on_gpu(a[0], "q");
  const c10::Device dev = q.device();
  vla_prompt_attn_desc d{};
  d.dtype = type_code(q, "q");
  rows(a[0], "q", dev, q.scalar_type(), 3);
  const at::Tensor& k = rows(a[1], "k", dev, q.scalar_type(), 3);
  const at::Tensor& v = rows(a[2], "v", dev, q.scalar_type(), 3);
  const at::Tensor& cu_q = whole(a[3], "cu_q", dev);
  const at::Tensor& cu_k = a[4] == Py_None ? cu_q : whole(a[4], "cu_k", dev);
  if (k.sizes() != v.sizes() || k.size(2) != q.size(2) || cu_q.size(0) != cu_k.size(0) || cu_q.size(0) < 1)
    refuse("q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes(), ", cu_q ", cu_q.sizes(), " and cu_k ", cu_k.sizes(), " do not fit each other");
  const int causal = PyObject_IsTrue(a[5]);
  if (causal < 0) throw Raised{};
  const at::Tensor out = output(a[7], q);
  if (a[7] != Py_None && !apart(out, k)) refuse("out overlaps k");
  if (a[7] != Py_None && !apart(out, v)) refuse("out overlaps v");
  d.q = q.const_data_ptr(); d.k = k.const_data_ptr(); d.v = v.const_data_ptr(); d.o = out.data_ptr();
  d.cu_q = ints(cu_q); d.cu_k = ints(cu_k);
  d.n_seqs = number(cu_q.size(0) - 1, "cu_q"); d.tokens_q = number(q.size(0), "q"); d.tokens_k = number(k.size(0), "k");
  d.heads = number(q.size(1), "q"); d.kv_heads = number(k.size(1), "k"); d.head_dim = number(q.size(2), "q");
  d.q_tok_stride = step(q, 0); d.q_head_stride = step(q, 1); d.k_tok_stride = step(k, 0); d.k_head_stride = step(k, 1);
  d.v_tok_stride = step(v, 0); d.v_head_stride = step(v, 1); d.o_tok_stride = step(out, 0); d.o_head_stride = step(out, 1);
  d.causal = causal; d.scale = scale_of(a[6], q.size(2));
  enqueue(vla_op_prompt_attention, d, dev);
  if (a[7] != Py_None) written(out);
  return THPVariable_Wrap(out);
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refusal& r) {
    PyErr_SetString(error_type, r.text.c_str());
    return nullptr;
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<block_plan, 7>("block_plan"), method<cache_append, 4>("cache_append"),
                         method<paged_attention, 6>("paged_attention"), method<prompt_attention, 8>("prompt_attention"), {}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_vla_ops", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__vla_ops() {
  if (!(capi = PyImport_ImportModule("_capi"))) return nullptr;
  if (!(error_type = PyObject_GetAttrString(capi, "VlaError"))) return nullptr;
  return PyModule_Create(&module);
}
