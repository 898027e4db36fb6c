// Python binding of the serving operators: argument checks, outputs and workspaces in C++, so that a
// call of a few microseconds on the GPU is not held up by the host.  The functions take positional
// arguments from the wrappers in serving.py, which say what they mean; the launches are the C entry
// points of include/tj_b200.h, taken from the library that runtime.py loads.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <map>
#include <mutex>
#include <sstream>

#include "../../../include/tj_b200.h"

namespace {

struct Api {
  decltype(&tj_b200_rotary) rotary;
  decltype(&tj_b200_cache_write) write;
  decltype(&tj_b200_cache_read) read;
  decltype(&tj_b200_paged_attention) attention;
  decltype(&tj_b200_paged_attention_workspace) attention_workspace;
  decltype(&tj_b200_narrow_indices) narrow;
  decltype(&tj_b200_last_error) last_error;
} api;
PyObject* runtime_error = nullptr;  // runtime.RuntimeError_
PyObject* out_of_memory = nullptr;  // torch.OutOfMemoryError

// A Python exception to be raised when the entry returns.
struct Fault {
  PyObject* type;
  std::string what;
  int code = 0;
};
[[noreturn]] void fail(PyObject* type, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void fail(PyObject* type, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw Fault{type, buf};
}
#define BAD(...) fail(PyExc_ValueError, __VA_ARGS__)

// Arguments whose conversion Python refuses (its exception is set already: `type` is NULL, `code` 0)
bool truth(PyObject* o) {
  const int t = PyObject_IsTrue(o);
  if (t < 0) throw Fault{nullptr, "", 0};
  return t;
}
const char* text(PyObject* o) {
  if (!PyUnicode_Check(o)) return "";
  const char* s = PyUnicode_AsUTF8(o);
  if (!s) throw Fault{nullptr, "", 0};
  return s;
}

void launched(int rc) {
  if (rc != TJ_OK) throw Fault{nullptr, api.last_error(), rc};
}

std::string shape_text(const at::Tensor& t) {
  std::ostringstream s;
  s << "(";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << (t.dim() == 1 ? ",)" : ")");
  return s.str();
}
const char* dtype_text(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kChar: return "torch.int8";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    case at::kDouble: return "torch.float64";
    case at::kFloat8_e4m3fn: return "torch.float8_e4m3fn";
    default: return c10::toString(t);
  }
}
int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return TJ_F32;
    case at::kHalf: return TJ_F16;
    case at::kBFloat16: return TJ_BF16;
    case at::kChar: return TJ_I8;
    case at::kFloat8_e4m3fn: return TJ_E4M3;
    default: return -1;
  }
}

using Types = std::initializer_list<at::ScalarType>;
constexpr Types ROWS = {at::kFloat, at::kHalf, at::kBFloat16};
constexpr Types INDEX = {at::kInt, at::kLong};

const at::Tensor& tensor(PyObject* o, const char* name, int64_t dim, Types types, int device = -1) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, "%s: expected a torch.Tensor, got %s", name, Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.dim() != dim) BAD("%s: expected %lld dimensions, got shape %s", name, static_cast<long long>(dim), shape_text(t).c_str());
  bool known = false;
  for (const at::ScalarType s : types) known |= s == t.scalar_type();
  if (!known) {
    std::string list;
    for (const at::ScalarType s : types) list += (list.empty() ? "" : ", ") + std::string(dtype_text(s));
    BAD("%s: dtype %s is not supported (one of %s)", name, dtype_text(t.scalar_type()), list.c_str());
  }
  if (!t.is_cuda() || (device >= 0 && t.get_device() != device))
    BAD("%s: tensor is on %s, not on %s", name, t.device().str().c_str(),
        device >= 0 ? ("cuda:" + std::to_string(device)).c_str() : "a CUDA device");
  return t;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// 64-bit indices as 32-bit ones, those that do not fit still out of range
at::Tensor narrowed(const at::Tensor& t) {
  const at::Tensor to = at::empty(t.sizes(), t.options().dtype(at::kInt));
  const bool vector = t.dim() == 1;
  const c10::cuda::CUDAGuard guard(t.device());
  launched(api.narrow(t.data_ptr<int64_t>(), vector ? 1 : t.size(0), t.size(t.dim() - 1), vector ? 0 : t.stride(0), t.stride(t.dim() - 1),
                      to.data_ptr<int32_t>(), stream_of(t.get_device())));
  return to;
}

// a vector of 32-bit indices, contiguous
at::Tensor indices(PyObject* o, const char* name, int device, int64_t size) {
  const at::Tensor& t = tensor(o, name, 1, INDEX, device);
  if (size >= 0 && t.size(0) != size)
    BAD("%s: expected %lld entries, got %lld", name, static_cast<long long>(size), static_cast<long long>(t.size(0)));
  return t.scalar_type() == at::kLong ? narrowed(t) : t.contiguous();
}

bool rows_fit(const at::Tensor& t) {
  const int64_t unit = 16 / t.element_size();
  return t.stride(2) == 1 && t.stride(0) % unit == 0 && t.stride(1) % unit == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
// rows that the kernels can read 16 bytes at a time: the tensor itself, or a copy
at::Tensor rows(const at::Tensor& t) { return t.numel() == 0 || rows_fit(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Whether autograd would follow what is made of t.  The entries then return NotImplemented, for the wrappers to put the
// call into the graph.
bool followed(const at::Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }
PyObject* to_the_graph(PyObject* out) {
  if (out != Py_None) BAD("out: not with inputs that require gradients; call it under torch.no_grad()");
  return Py_NewRef(Py_NotImplemented);
}

// Torch counts a tensor's changes, by which autograd knows that a value it has kept is no longer there.
void changed(c10::TensorImpl* t) {
  if (t && !t->is_inference()) t->bump_version();
}

at::Tensor out_rows(PyObject* o, const char* name, const at::Tensor& like) {
  const at::Tensor& t = tensor(o, name, 3, {like.scalar_type()}, like.get_device());
  if (t.sizes() != like.sizes()) BAD("%s: expected shape %s, got %s", name, shape_text(like).c_str(), shape_text(t).c_str());
  if (t.numel() && !rows_fit(t)) BAD("%s: rows must be contiguous and start on 16-byte boundaries", name);
  if (followed(t)) BAD("%s: requires gradients; call it under torch.no_grad()", name);
  changed(t.unsafeGetTensorImpl());
  return t;
}

void head_dim(int64_t dim) {
  if (dim % 8 || dim <= 0 || dim > 512) BAD("head dim %lld is not a multiple of 8 from 8 to 512", static_cast<long long>(dim));
}

// What PagedCache keeps of its tensors, which it holds and which cannot be replaced.
struct CacheInfo {
  tj_kv_cache c;
  int64_t device;
  c10::TensorImpl* tensors[4];  // k, v, their scales or NULL
};
const CacheInfo& cache_info(PyObject* o) {
  if (!PyBytes_Check(o) || PyBytes_GET_SIZE(o) != sizeof(CacheInfo)) fail(PyExc_TypeError, "cache: not a PagedCache's description");
  const CacheInfo& i = *reinterpret_cast<const CacheInfo*>(PyBytes_AS_STRING(o));
  // a tensor may have been given other memory since (t.data = ..., module.to()), and the old may be someone else's
  const void* held[4] = {i.c.k, i.c.v, i.c.k_scale, i.c.v_scale};
  for (int n = 0; n < 4; ++n)
    if (i.tensors[n] && i.tensors[n]->data() != held[n]) BAD("cache: its tensors have other memory than when the PagedCache was made");
  return i;
}

PyObject* describe(PyObject* const* a) {
  const at::Tensor& k = tensor(a[0], "k", 4, {at::kHalf, at::kBFloat16, at::kChar, at::kFloat8_e4m3fn});
  const int dev = k.get_device();
  const at::Tensor& v = tensor(a[1], "v", 4, {k.scalar_type()}, dev);
  if (v.sizes() != k.sizes() || v.strides() != k.strides()) BAD("k and v must have the same shape and strides");
  const int64_t size = k.element_size(), unit = size == 1 ? 8 : 16;
  head_dim(k.size(3));
  if (k.stride(3) != 1 || k.stride(0) * size % unit || k.stride(1) * size % unit || k.stride(2) * size % unit ||
      (reinterpret_cast<uintptr_t>(k.data_ptr()) | reinterpret_cast<uintptr_t>(v.data_ptr())) % 16)
    BAD("cache rows must be contiguous and start on %lld-byte boundaries", static_cast<long long>(unit));
  CacheInfo i{};
  if (size == 1) {
    for (int n = 0; n < 2; ++n) {
      const char* name = n ? "v_scale" : "k_scale";
      if (a[2 + n] == Py_None) BAD("a %s cache needs %s", dtype_text(k.scalar_type()), name);
      const at::Tensor& s = tensor(a[2 + n], name, 3, {at::kFloat}, dev);
      if (s.sizes() != k.sizes().slice(0, 3))
        BAD("%s: expected shape (%lld, %lld, %lld), got %s", name, static_cast<long long>(k.size(0)), static_cast<long long>(k.size(1)),
            static_cast<long long>(k.size(2)), shape_text(s).c_str());
      (n ? i.c.v_scale : i.c.k_scale) = s.data_ptr<float>();
      if (n && s.strides() != THPVariable_Unpack(a[2]).strides()) BAD("k_scale and v_scale must have the same strides");
      i.c.scale_page = s.stride(0);
      i.c.scale_slot = s.stride(1);
      i.c.scale_head = s.stride(2);
    }
  } else if (a[2] != Py_None || a[3] != Py_None) {
    BAD("a %s cache has no scales", dtype_text(k.scalar_type()));
  }
  i.c.k = k.data_ptr();
  i.c.v = v.data_ptr();
  i.c.pages = k.size(0);
  i.c.page_size = k.size(1);
  i.c.heads = k.size(2);
  i.c.dim = k.size(3);
  i.c.page_stride = k.stride(0);
  i.c.slot_stride = k.stride(1);
  i.c.head_stride = k.stride(2);
  i.c.dtype = code_of(k.scalar_type());
  i.device = dev;
  for (int n = 0; n < 4; ++n) i.tensors[n] = a[n] == Py_None ? nullptr : THPVariable_Unpack(a[n]).unsafeGetTensorImpl();
  return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&i), sizeof(i));
}

// table and positions into the arguments; the tensors that hold them
struct Turn {
  at::Tensor table, positions;
};
Turn turn(tj_rows& r, PyObject* positions, PyObject* table, PyObject* layout, int device) {
  Turn t;
  t.table = tensor(table, "table", 2, {at::kFloat}, device);
  if (followed(t.table)) BAD("table: no gradient is computed for it");
  const char* how = text(layout);
  r.interleaved = strcmp(how, "interleaved") == 0;
  if (!r.interleaved && strcmp(how, "half")) BAD("layout must be 'half' or 'interleaved', not '%s'", how);
  r.rot = t.table.size(1);
  r.table_rows = t.table.size(0);
  if (r.rot % 2 || r.rot <= 0 || r.rot > r.dim || r.table_rows == 0)
    BAD("table: %lld columns do not turn rows of %lld", static_cast<long long>(r.rot), static_cast<long long>(r.dim));
  if (!t.table.is_contiguous() || reinterpret_cast<uintptr_t>(t.table.data_ptr()) % 16) t.table = t.table.clone(at::MemoryFormat::Contiguous);
  t.positions = indices(positions, "positions", device, r.tokens);
  r.table = t.table.data_ptr<float>();
  r.positions = t.positions.data_ptr<int32_t>();
  return t;
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject* x = THPVariable_Wrap(a);
  PyObject* y = b.defined() ? THPVariable_Wrap(b) : Py_NewRef(Py_None);
  PyObject* t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, x);
  PyTuple_SET_ITEM(t, 1, y);
  return t;
}

// q, k, positions, table, layout, inverse, out
PyObject* rotary(PyObject* const* a) {
  const at::Tensor& q = tensor(a[0], "q", 3, ROWS);
  const int dev = q.get_device();
  tj_rows r{};
  r.tokens = q.size(0);
  r.q_heads = q.size(1);
  r.dim = q.size(2);
  head_dim(r.dim);
  r.dtype = code_of(q.scalar_type());
  const Turn held = turn(r, a[2], a[3], a[4], dev);
  r.inverse = truth(a[5]);
  const bool keys = a[1] != Py_None;
  at::Tensor k, q2, k2;
  if (keys) {
    k = tensor(a[1], "k", 3, {q.scalar_type()}, dev);
    if (k.size(0) != r.tokens || k.size(2) != r.dim) BAD("k: shape %s does not go with q's %s", shape_text(k).c_str(), shape_text(q).c_str());
    r.kv_heads = k.size(1);
  }
  if (followed(q) || (keys && followed(k))) return to_the_graph(a[6]);
  if (a[6] == Py_None) {
    q2 = at::empty(q.sizes(), q.options());
    if (keys) k2 = at::empty(k.sizes(), k.options());
  } else {
    if (!PyTuple_Check(a[6]) || PyTuple_GET_SIZE(a[6]) != 2) fail(PyExc_TypeError, "out: expected a pair");
    q2 = out_rows(PyTuple_GET_ITEM(a[6], 0), "out[0]", q);
    if (keys) k2 = out_rows(PyTuple_GET_ITEM(a[6], 1), "out[1]", k);
  }
  const at::Tensor qr = rows(q), kr = keys ? rows(k) : at::Tensor();
  r.q = qr.data_ptr();
  r.q_out = q2.data_ptr();
  r.q_token = qr.stride(0);
  r.q_head = qr.stride(1);
  r.qo_token = q2.stride(0);
  r.qo_head = q2.stride(1);
  if (keys && k.numel()) {
    r.k = kr.data_ptr();
    r.k_out = k2.data_ptr();
    r.k_token = kr.stride(0);
    r.k_head = kr.stride(1);
    r.ko_token = k2.stride(0);
    r.ko_head = k2.stride(1);
  }
  if (q.numel() || k.defined()) {
    if (!q.numel()) r.q = nullptr;
    if (r.q || r.k) {
      const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
      launched(api.rotary(&r, stream_of(dev)));
    }
  }
  return pair(q2, k2);
}

// cache, q, k, v, slots, positions, table, layout, out
PyObject* write(PyObject* const* a) {
  const CacheInfo& cache = cache_info(a[0]);
  const int dev = static_cast<int>(cache.device);
  const at::Tensor& k = tensor(a[2], "k", 3, ROWS, dev);
  const at::Tensor& v = tensor(a[3], "v", 3, {k.scalar_type()}, dev);
  tj_rows r{};
  r.cache = cache.c;
  r.tokens = k.size(0);
  r.kv_heads = k.size(1);
  r.dim = k.size(2);
  r.dtype = code_of(k.scalar_type());
  if (v.sizes() != k.sizes() || r.kv_heads != cache.c.heads || r.dim != cache.c.dim)
    BAD("k %s and v %s do not go with a cache of %lld heads of %lld", shape_text(k).c_str(), shape_text(v).c_str(),
        static_cast<long long>(cache.c.heads), static_cast<long long>(cache.c.dim));
  const at::Tensor slots = indices(a[4], "slots", dev, r.tokens);
  r.slots = slots.data_ptr<int32_t>();
  Turn held;
  at::Tensor qr, q2;
  if (a[6] != Py_None) {
    held = turn(r, a[5], a[6], a[7], dev);
    if (a[1] != Py_None) {
      const at::Tensor& q = tensor(a[1], "q", 3, {k.scalar_type()}, dev);
      if (q.size(0) != r.tokens || q.size(2) != r.dim) BAD("q: shape %s does not go with k's %s", shape_text(q).c_str(), shape_text(k).c_str());
      if (followed(q)) return to_the_graph(a[8]);
      q2 = a[8] == Py_None ? at::empty(q.sizes(), q.options()) : out_rows(a[8], "out", q);
      qr = rows(q);
      if (q.numel()) {
        r.q_heads = q.size(1);
        r.q = qr.data_ptr();
        r.q_out = q2.data_ptr();
        r.q_token = qr.stride(0);
        r.q_head = qr.stride(1);
        r.qo_token = q2.stride(0);
        r.qo_head = q2.stride(1);
      }
    }
  }
  if (r.tokens) {
    for (c10::TensorImpl* t : cache.tensors) {
      if (t && t->requires_grad() && at::GradMode::is_enabled()) BAD("cache: requires gradients; write it under torch.no_grad()");
      changed(t);
    }
    const at::Tensor kr = rows(k), vr = rows(v);
    r.k = kr.data_ptr();
    r.v = vr.data_ptr();
    r.k_token = kr.stride(0);
    r.k_head = kr.stride(1);
    r.v_token = vr.stride(0);
    r.v_head = vr.stride(1);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    launched(api.write(&r, stream_of(dev)));
  }
  if (!q2.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(q2);
}

// cache, slots, dtype
PyObject* read(PyObject* const* a) {
  const CacheInfo& cache = cache_info(a[0]);
  const int dev = static_cast<int>(cache.device);
  const char* how = text(a[2]);
  at::ScalarType kind;
  if (!strcmp(how, "bf16"))
    kind = at::kBFloat16;
  else if (!strcmp(how, "f16"))
    kind = at::kHalf;
  else if (!strcmp(how, "f32"))
    kind = at::kFloat;
  else
    BAD("dtype must be f32, f16 or bf16, not '%s'", how);
  const at::Tensor slots = indices(a[1], "slots", dev, -1);
  const auto options = slots.options().dtype(kind);
  const at::Tensor k = at::empty({slots.size(0), cache.c.heads, cache.c.dim}, options), v = at::empty(k.sizes(), options);
  if (slots.size(0)) {
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    launched(api.read(&cache.c, slots.data_ptr<int32_t>(), slots.size(0), k.data_ptr(), v.data_ptr(), code_of(kind), stream_of(dev)));
  }
  return pair(k, v);
}

// A call's workspace and its counters (zero between calls), kept for each stream: calls on one stream
// follow one another, calls on two must not share them.
struct Workspace {
  at::Tensor bytes, counters;
};
std::map<std::pair<int, void*>, Workspace> workspaces;
std::mutex workspaces_lock;

Workspace workspace(int dev, void* stream, int64_t size, int64_t count, const at::TensorOptions& like) {
  const auto make = [&](int64_t s, int64_t c) {
    return Workspace{at::empty({s}, like.dtype(at::kByte)), at::zeros({c}, like.dtype(at::kInt))};
  };
  cudaStreamCaptureStatus state = cudaStreamCaptureStatusNone;
  cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &state);
  // a graph's own: its zeroing is part of the graph, its memory belongs to the graph's pool
  if (state != cudaStreamCaptureStatusNone) return make(size, count);
  const std::lock_guard<std::mutex> hold(workspaces_lock);
  Workspace& w = workspaces[{dev, stream}];
  if (!w.bytes.defined() || w.bytes.size(0) < size || w.counters.size(0) < count)
    w = make(w.bytes.defined() ? std::max(size, w.bytes.size(0)) : size, w.bytes.defined() ? std::max(count, w.counters.size(0)) : count);
  return w;
}
PyObject* forget(PyObject* const*) {
  const std::lock_guard<std::mutex> hold(workspaces_lock);
  workspaces.clear();
  Py_RETURN_NONE;
}

// cache, q, page_table, kv_lens, q_starts, max_new, scale, causal, window, return_lse, out
PyObject* attention(PyObject* const* a) {
  const CacheInfo& cache = cache_info(a[0]);
  const int dev = static_cast<int>(cache.device);
  const at::Tensor& q = tensor(a[1], "q", 3, {at::kHalf, at::kBFloat16}, dev);
  tj_paged_attention p{};
  p.cache = cache.c;
  p.dtype = code_of(q.scalar_type());
  p.tokens = q.size(0);
  p.q_heads = q.size(1);
  const int64_t dim = cache.c.dim;
  if (q.size(2) != dim || p.q_heads % cache.c.heads || p.q_heads == 0)
    BAD("q: shape %s does not go with a cache of %lld heads of %lld", shape_text(q).c_str(), static_cast<long long>(cache.c.heads), static_cast<long long>(dim));
  if (dim != 64 && dim != 128) BAD("head dim must be 64 or 128, not %lld", static_cast<long long>(dim));
  if ((cache.c.dtype == TJ_F16 || cache.c.dtype == TJ_BF16) && cache.c.dtype != p.dtype)
    BAD("q is %s and the cache %s: a 16-bit cache must have q's dtype", dtype_text(q.scalar_type()), cache.c.dtype == TJ_F16 ? "torch.float16" : "torch.bfloat16");
  at::Tensor table = tensor(a[2], "page_table", 2, INDEX, dev);
  if (table.scalar_type() == at::kLong)
    table = narrowed(table);
  else if (table.stride(1) != 1)
    table = table.contiguous();
  p.batch = table.size(0);
  p.table_width = table.size(1);
  p.table_row = table.stride(0);
  if (p.table_width == 0 && p.batch) BAD("page_table: no columns");
  p.page_table = table.data_ptr<int32_t>();
  const at::Tensor lens = indices(a[3], "kv_lens", dev, p.batch);
  p.kv_lens = lens.data_ptr<int32_t>();
  at::Tensor starts;
  if (a[4] != Py_None) {
    starts = indices(a[4], "q_starts", dev, p.batch + 1);
    p.q_starts = starts.data_ptr<int32_t>();
  } else if (p.tokens != p.batch) {
    BAD("without q_starts there is one token to a sequence: %lld tokens, %lld sequences", static_cast<long long>(p.tokens), static_cast<long long>(p.batch));
  }
  p.max_new = a[5] != Py_None ? PyLong_AsLongLong(a[5]) : p.q_starts ? INT64_MAX : 1;
  p.window = PyLong_AsLongLong(a[8]);
  p.scale = a[6] != Py_None ? PyFloat_AsDouble(a[6]) : 1.0 / std::sqrt(static_cast<double>(dim));
  p.causal = truth(a[7]);
  if (PyErr_Occurred()) return nullptr;
  if (p.max_new < 1 || p.window < 0) BAD("max_new must be positive and window not negative");
  if (!(p.scale > 0.0) || !std::isfinite(p.scale)) BAD("scale must be positive");
  if (followed(q)) return to_the_graph(a[10]);
  const at::Tensor out = a[10] == Py_None ? at::empty(q.sizes(), q.options()) : out_rows(a[10], "out", q);
  at::Tensor lse;
  if (truth(a[9])) {
    lse = at::empty({p.tokens, p.q_heads}, q.options().dtype(at::kFloat));
    p.lse = lse.data_ptr<float>();
  }
  if (p.tokens && p.batch) {
    const at::Tensor qr = rows(q);
    p.q = qr.data_ptr();
    p.out = out.data_ptr();
    p.q_token = qr.stride(0);
    p.q_head = qr.stride(1);
    p.out_token = out.stride(0);
    p.out_head = out.stride(1);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    void* stream = stream_of(dev);
    launched(api.attention_workspace(&p, &p.workspace_bytes, &p.counters_count));
    const Workspace w = workspace(dev, stream, p.workspace_bytes, p.counters_count, q.options());
    p.workspace = w.bytes.data_ptr();
    p.counters = w.counters.data_ptr<int32_t>();
    launched(api.attention(&p, stream));
  }
  return lse.defined() ? pair(out, lse) : THPVariable_Wrap(out);
}

// library path, runtime.RuntimeError_, torch.OutOfMemoryError
PyObject* init(PyObject* const* a) {
  const char* path = PyUnicode_AsUTF8(a[0]);
  if (!path) return nullptr;
  void* lib = dlopen(path, RTLD_NOW);
  if (!lib) fail(PyExc_ImportError, "%s", dlerror());
  const auto get = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(lib, name));
    if (!f) fail(PyExc_ImportError, "%s has no %s", path, name);
  };
  get(api.rotary, "tj_b200_rotary");
  get(api.write, "tj_b200_cache_write");
  get(api.read, "tj_b200_cache_read");
  get(api.attention, "tj_b200_paged_attention");
  get(api.attention_workspace, "tj_b200_paged_attention_workspace");
  get(api.narrow, "tj_b200_narrow_indices");
  get(api.last_error, "tj_b200_last_error");
  Py_XDECREF(runtime_error);
  runtime_error = Py_NewRef(a[1]);
  Py_XDECREF(out_of_memory);
  out_of_memory = Py_NewRef(a[2]);
  Py_RETURN_NONE;
}

// Nothing of C++ passes into Python: faults and torch's own errors become exceptions.
template <PyObject* (*F)(PyObject* const*), int N> PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Fault& f) {
    if (f.type) {
      PyErr_SetString(f.type, f.what.c_str());
    } else if (f.code != 0) {
      PyObject* e = PyObject_CallFunction(runtime_error, "is", f.code, f.what.c_str());
      if (e) {
        PyErr_SetObject(runtime_error, e);
        Py_DECREF(e);
      }
    }
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(out_of_memory ? out_of_memory : PyExc_MemoryError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "serving: unknown C++ exception");
  }
  return nullptr;
}

#define ENTRY(f, n) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(init, 3),  ENTRY(describe, 4), ENTRY(rotary, 7), ENTRY(write, 9),
                         ENTRY(read, 3),  ENTRY(attention, 11), ENTRY(forget, 0), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving() { return PyModule_Create(&module); }
