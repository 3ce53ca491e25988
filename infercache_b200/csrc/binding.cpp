// Python binding of the paged serving tick: argument checks, output and
// workspace tensors and the C-ABI call, without an interpreter in between (a
// decode tick makes several of these calls per layer, each a few microseconds
// of GPU work).  It adds nothing to the C ABI of include/infercache.h, which it
// calls; paged_ops.py and logits.py wrap it and document the operators.
//
// Errors: ValueError for bad tensors; a non-zero ic_status goes to
// _lib.raise_for, which every other binding uses too.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <cmath>
#include <limits>
#include <sstream>
#include <string>

#include "../../include/infercache.h"

namespace {

using at::Tensor;

constexpr int PAGE = 16;
PyObject* g_require = nullptr;  // _lib.require_device
PyObject* g_raise = nullptr;    // _lib.raise_for
bool g_device_ok[64] = {};

// Thrown once a Python exception is set.
struct Raised {};

[[noreturn]] void bad(const char* name, const std::string& why) {
  PyErr_Format(PyExc_ValueError, "%s: %s", name, why.c_str());
  throw Raised();
}

std::string shape_text(at::IntArrayRef s) {
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  o << ")";
  return o.str();
}

const Tensor& tensor(PyObject* o, const char* name, const char* what) {
  if (!THPVariable_Check(o)) bad(name, std::string(what) + " must be a tensor");
  return THPVariable_Unpack(o);
}
bool none(PyObject* o) { return o == Py_None; }

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised();
  return v != 0;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}

// The device of a CUDA tensor, once known to be an sm_100 GPU.
c10::Device device_of(const char* name, const Tensor& t) {
  if (!t.is_cuda()) bad(name, "runs on CUDA tensors only");
  const c10::Device d = t.device();
  const int i = d.index();
  if (i < 0 || i >= 64 || !g_device_ok[i]) {
    THPObjectPtr wrapped(THPVariable_Wrap(t));
    THPObjectPtr device(wrapped ? PyObject_GetAttrString(wrapped.get(), "device") : nullptr);
    THPObjectPtr r(device ? PyObject_CallFunctionObjArgs(g_require, device.get(), nullptr) : nullptr);
    if (!r) throw Raised();
    if (i >= 0 && i < 64) g_device_ok[i] = true;
  }
  return d;
}

void check_status(int rc, const char* name) {
  if (rc == IC_OK) return;
  PyObject* r = PyObject_CallFunction(g_raise, "is", rc, name);
  if (r) {  // raise_for returned: it does so only for IC_OK
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, name);
  }
  throw Raised();
}

int float_code(const char* name, at::ScalarType t) {
  switch (t) {
    case at::kFloat: return IC_F32;
    case at::kHalf: return IC_F16;
    case at::kBFloat16: return IC_BF16;
    default: bad(name, std::string("unsupported dtype ") + c10::toString(t) + "; use float32, float16 or bfloat16");
  }
}

// Data pointer of an int32 tensor that a kernel reads or writes in place.
int32_t* state(const char* name, const char* what, const Tensor& t, c10::Device dev, at::IntArrayRef shape) {
  if (t.scalar_type() != at::kInt || t.device() != dev || !t.is_contiguous() || t.sizes() != shape)
    bad(name, std::string(what) + " must be a contiguous int32 tensor of shape " + shape_text(shape) + " on " + dev.str() +
                  ", got " + c10::toString(t.scalar_type()) + " " + shape_text(t.sizes()) + " on " + t.device().str());
  return static_cast<int32_t*>(t.data_ptr());
}
int32_t* status_word(const char* name, PyObject* o, c10::Device dev) {
  return none(o) ? nullptr : state(name, "status", tensor(o, name, "status"), dev, {1});
}

// An int32 copy of an int32 / int64 tensor (the tensor itself when it needs none).
// Values that 32 bits do not hold become the nearest that they do: outside every
// pool and vocabulary, and past every length, as the value itself is.
Tensor ints(const char* name, const char* what, const Tensor& t, c10::Device dev, at::IntArrayRef shape) {
  bool ok = (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.device() == dev &&
            t.dim() == static_cast<int64_t>(shape.size());
  for (size_t i = 0; ok && i < shape.size(); ++i) ok = shape[i] < 0 || t.size(i) == shape[i];
  if (!ok)
    bad(name, std::string(what) + " must be an int32 or int64 tensor of shape " + shape_text(shape) + " (-1: any) on " +
                  dev.str() + ", got " + c10::toString(t.scalar_type()) + " " + shape_text(t.sizes()) + " on " + t.device().str());
  if (t.scalar_type() == at::kInt) return t.contiguous();
  using limits = std::numeric_limits<int32_t>;
  return t.clamp(limits::min(), limits::max()).to(at::kInt).contiguous();
}

// Whether every row (last dimension) starts on a 16-byte boundary and is contiguous.
bool rows16(const Tensor& t) {
  const int64_t e = t.element_size(), d = t.dim();
  if (t.stride(d - 1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < d; ++i)
    if (t.size(i) > 1 && t.stride(i) * e % 16) return false;
  return true;
}
bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Whether the bytes from a tensor's first element to its last meet another's.
bool meet(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto end = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return reinterpret_cast<uintptr_t>(t.data_ptr()) + (last + 1) * t.element_size();
  };
  return reinterpret_cast<uintptr_t>(a.data_ptr()) < end(b) && reinterpret_cast<uintptr_t>(b.data_ptr()) < end(a);
}

// Whether rows [S, V] of `a` and `b` (contiguous, `stride` bytes apart in both) have
// none of their bytes in common, though they may alternate.
bool rows_apart(const Tensor& a, const Tensor& b, int64_t stride) {
  const auto pa = reinterpret_cast<uintptr_t>(a.data_ptr()), pb = reinterpret_cast<uintptr_t>(b.data_ptr());
  const Tensor &first = pa <= pb ? a : b, &second = pa <= pb ? b : a;
  const int64_t shift = static_cast<int64_t>(pa <= pb ? pb - pa : pa - pb) % stride;
  return shift >= first.size(1) * first.element_size() && shift + second.size(1) * second.element_size() <= stride;
}

// An uninitialised contiguous tensor on `dev` (made current by the caller).
Tensor fresh(at::IntArrayRef shape, at::ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(shape, type, dev, std::nullopt);
}

// `shape` elements of a one-dimensional tensor from `offset` on, as a tensor of
// its own over the same memory.
Tensor part_of(const Tensor& base, int64_t offset, int64_t shape) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), base.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({shape});
  return t;
}

struct Cache {
  c10::Device dev{c10::kCPU};
  int64_t dims, L, H, n, D;
  int code;
  const Tensor *k, *v, *ks, *vs;
};

Cache cache_of(const char* name, PyObject* const* a) {
  Cache c;
  c.k = &tensor(a[0], name, "k_cache");
  c.v = &tensor(a[1], name, "v_cache");
  c.ks = &tensor(a[2], name, "k_scale");
  c.vs = &tensor(a[3], name, "v_scale");
  c.dev = device_of(name, *c.k);
  const auto type = c.k->scalar_type();
  if (type != at::kFloat8_e4m3fn && type != at::kChar)
    bad(name, std::string("the cache must be float8_e4m3fn or int8, got ") + c10::toString(type));
  c.code = type == at::kChar ? IC_I8 : IC_E4M3;
  c.dims = c.k->dim();
  if (c.dims != 3 && c.dims != 4) bad(name, "the cache must be [H, pool_tokens, D] or [L, H, pool_tokens, D]");
  c.L = c.dims == 4 ? c.k->size(0) : 1;
  c.H = c.k->size(c.dims - 3);
  c.n = c.k->size(c.dims - 2);
  c.D = c.k->size(c.dims - 1);
  if (c.n < PAGE || c.n % PAGE) bad(name, "pool_tokens must be a positive multiple of 16, got " + std::to_string(c.n));
  if (c.v->scalar_type() != type || c.v->sizes() != c.k->sizes() || c.v->device() != c.dev || !c.k->is_contiguous() ||
      !c.v->is_contiguous())
    bad(name, "k_cache and v_cache must be contiguous and alike in shape, dtype and device");
  for (const Tensor* s : {c.ks, c.vs}) {
    bool ok = s->scalar_type() == at::kFloat && s->dim() == c.dims - 1 && s->device() == c.dev && s->is_contiguous() &&
              s->size(c.dims - 2) == c.n / PAGE;
    for (int64_t i = 0; ok && i < c.dims - 2; ++i) ok = s->size(i) == c.k->size(i);
    if (!ok) bad(name, "scales must be contiguous float32 tensors, the cache's shape without D and with pool_tokens / 16, on " + c.dev.str());
  }
  return c;
}

Tensor slots_of(const char* name, PyObject* o, c10::Device dev) {
  return ints(name, "slots", tensor(o, name, "slots"), dev, {-1});
}

ic_page_q8_args q8_args(const Cache& c, const ic_page_q8_rows* rows, int buf_dtype, int32_t* status) {
  ic_page_q8_args a = {};
  a.pool.k = c.k->data_ptr();
  a.pool.v = c.v->data_ptr();
  a.pool.pool_tokens = c.n;
  a.pool.num_layers = static_cast<int32_t>(c.L);
  a.pool.num_kv_heads = static_cast<int32_t>(c.H);
  a.pool.head_dim = static_cast<int32_t>(c.D);
  a.pool.dtype = c.code;
  a.k_scale = static_cast<float*>(c.ks->data_ptr());
  a.v_scale = static_cast<float*>(c.vs->data_ptr());
  a.rows = rows;
  a.dev_status = status;
  a.count = 1;
  a.layer_end = a.pool.num_layers;
  a.buf_dtype = buf_dtype;
  return a;
}

template <typename Fn>
PyObject* guarded(Fn fn) {
  HANDLE_TH_ERRORS
  try {
    return fn();
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

bool arity(const char* name, Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, n);
  return false;
}

// lens, counts, block_table, free_pages, free_count, total, commit, status
//   -> (q_start, slots, positions, lens, free_count)
PyObject* py_page_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  static const char* name = "page_plan";
  if (!arity(name, n, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor &lens = tensor(a[0], name, "lens"), &counts = tensor(a[1], name, "counts");
    const Tensor &table = tensor(a[2], name, "block_table"), &pages = tensor(a[3], name, "free_pages");
    const Tensor& count = tensor(a[4], name, "free_count");
    const c10::Device dev = device_of(name, lens);
    if (lens.dim() != 1 || table.dim() != 2 || pages.dim() != 1)
      bad(name, "lens must be [S], block_table [S, width] and free_pages [P]");
    const int64_t S = lens.size(0), W = table.size(1), P = pages.size(0), total = integer(a[5]);
    if (total < 0 || total > 0x7fffffff) bad(name, "total must be in [0, 2^31), got " + std::to_string(total));
    const bool commit = truth(a[6]);
    ic_page_plan_args x = {};
    int32_t* lens_p = state(name, "lens", lens, dev, {S});
    int32_t* count_p = state(name, "free_count", count, dev, {1});
    x.lens = lens_p;
    x.counts = state(name, "counts", counts, dev, {S});
    x.block_table = state(name, "block_table", table, dev, {S, W});
    x.free_pages = state(name, "free_pages", pages, dev, {P});
    x.free_count = count_p;
    x.dev_status = status_word(name, a[7], dev);
    c10::cuda::CUDAGuard guard(dev);
    // the small results and the workspace share an allocation
    const Tensor small = fresh({4 * S + 3}, at::kInt, dev);
    Tensor slots = fresh({total}, at::kInt, dev), positions = fresh({total}, at::kLong, dev);
    Tensor q_start = part_of(small, 0, S + 1);
    Tensor lens_out = commit ? lens : part_of(small, S + 1, S), count_out = commit ? count : part_of(small, 2 * S + 1, 1);
    x.q_start = static_cast<int32_t*>(q_start.data_ptr());
    x.slots = static_cast<int32_t*>(slots.data_ptr());
    x.positions = static_cast<int64_t*>(positions.data_ptr());
    x.lens_out = static_cast<int32_t*>(lens_out.data_ptr());
    x.free_count_out = static_cast<int32_t*>(count_out.data_ptr());
    x.workspace = static_cast<int32_t*>(small.data_ptr()) + 2 * S + 2;
    x.num_sessions = static_cast<int32_t>(S);
    x.width = static_cast<int32_t>(std::min<int64_t>(W, 0x7fffffff));
    x.total = static_cast<int32_t>(total);
    x.free_capacity = static_cast<int32_t>(std::min<int64_t>(P, 0x7fffffff));
    check_status(ic_page_plan(&x, at::cuda::getCurrentCUDAStream(dev.index()).stream()), "ic_page_plan");
    return PyTuple_Pack(5, THPObjectPtr(THPVariable_Wrap(q_start)).get(), THPObjectPtr(THPVariable_Wrap(slots)).get(),
                        THPObjectPtr(THPVariable_Wrap(positions)).get(), THPObjectPtr(THPVariable_Wrap(lens_out)).get(),
                        THPObjectPtr(THPVariable_Wrap(count_out)).get());
  });
}

// lens, keep, block_table, free_pages, free_count, status
PyObject* py_page_release(PyObject*, PyObject* const* a, Py_ssize_t n) {
  static const char* name = "page_release";
  if (!arity(name, n, 6)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor &lens = tensor(a[0], name, "lens"), &table = tensor(a[2], name, "block_table");
    const Tensor& pages = tensor(a[3], name, "free_pages");
    const c10::Device dev = device_of(name, lens);
    if (lens.dim() != 1 || table.dim() != 2 || pages.dim() != 1)
      bad(name, "lens must be [S], block_table [S, width] and free_pages [P]");
    const int64_t S = lens.size(0), W = table.size(1), P = pages.size(0);
    ic_page_release_args x = {};
    x.lens = state(name, "lens", lens, dev, {S});
    x.keep = state(name, "keep", tensor(a[1], name, "keep"), dev, {S});
    x.block_table = state(name, "block_table", table, dev, {S, W});
    x.free_pages = state(name, "free_pages", pages, dev, {P});
    x.free_count = state(name, "free_count", tensor(a[4], name, "free_count"), dev, {1});
    x.dev_status = status_word(name, a[5], dev);
    x.num_sessions = static_cast<int32_t>(S);
    x.width = static_cast<int32_t>(std::min<int64_t>(W, 0x7fffffff));
    x.free_capacity = static_cast<int32_t>(std::min<int64_t>(P, 0x7fffffff));
    c10::cuda::CUDAGuard guard(dev);
    check_status(ic_page_release(&x, at::cuda::getCurrentCUDAStream(dev.index()).stream()), "ic_page_release");
    Py_RETURN_NONE;
  });
}

// k, v, k_cache, v_cache, k_scale, v_scale, slots, status
PyObject* py_page_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  static const char* name = "page_write";
  if (!arity(name, n, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Cache c = cache_of(name, a + 2);
    Tensor k = tensor(a[0], name, "k"), v = tensor(a[1], name, "v");
    const int64_t d = c.dims;
    if (k.dim() != d || v.sizes() != k.sizes() || k.size(d - 2) != c.H || k.size(d - 1) != c.D ||
        (d == 4 && k.size(0) != c.L))
      bad(name, std::string("k and v must be ") + (d == 4 ? "[L, N, H, D]" : "[N, H, D]") + " for a cache " +
                    shape_text(c.k->sizes()) + ", got " + shape_text(k.sizes()) + " and " + shape_text(v.sizes()));
    if (k.scalar_type() != v.scalar_type() || k.device() != c.dev || v.device() != c.dev)
      bad(name, "k and v must share the cache's device and a dtype");
    if (meet(*c.k, *c.v) || meet(*c.ks, *c.vs)) bad(name, "k_cache and v_cache, and their scales, must not overlap");
    const int dt = float_code(name, k.scalar_type());
    const int64_t N = k.size(d - 3);
    Tensor slots = slots_of(name, a[6], c.dev);
    if (slots.size(0) != N) bad(name, std::to_string(N) + " tokens but " + std::to_string(slots.size(0)) + " slots");
    int32_t* status = status_word(name, a[7], c.dev);
    if (N == 0 || c.L == 0 || c.H == 0) Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(c.dev);
    if (k.strides() != v.strides() || !rows16(k) || !rows16(v)) {
      k = k.clone(at::MemoryFormat::Contiguous);
      v = v.clone(at::MemoryFormat::Contiguous);
    }
    ic_page_q8_rows rows = {};
    rows.slots = static_cast<int32_t*>(slots.data_ptr());
    rows.k_buf = k.data_ptr();
    rows.v_buf = v.data_ptr();
    rows.n_tokens = N;
    rows.stride_l = d == 4 && c.L > 1 ? k.stride(0) : 0;
    rows.stride_t = N > 1 ? k.stride(d - 3) : 0;
    rows.stride_h = c.H > 1 ? k.stride(d - 2) : 0;
    const ic_page_q8_args x = q8_args(c, &rows, dt, status);
    check_status(ic_page_write_q8(&x, at::cuda::getCurrentCUDAStream(c.dev.index()).stream()), "ic_page_write_q8");
    Py_RETURN_NONE;
  });
}

// k_cache, v_cache, k_scale, v_scale, slots, dtype code, out_k, out_v -> (k, v)
PyObject* py_page_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  static const char* name = "page_read";
  if (!arity(name, n, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Cache c = cache_of(name, a);
    Tensor slots = slots_of(name, a[4], c.dev);
    const int64_t N = slots.size(0);
    at::DimVector shape;
    if (c.dims == 4) shape.push_back(c.L);
    shape.push_back(c.H);
    shape.push_back(N);
    shape.push_back(c.D);
    c10::cuda::CUDAGuard guard(c.dev);
    Tensor k, v;
    if (none(a[6])) {
      const int64_t code = integer(a[5]);
      const auto type = code == IC_F32 ? at::kFloat : code == IC_F16 ? at::kHalf : at::kBFloat16;
      k = fresh(shape, type, c.dev);
      v = fresh(shape, type, c.dev);
    } else {
      k = tensor(a[6], name, "out");
      v = tensor(a[7], name, "out");
      for (const Tensor* t : {&k, &v})
        if (t->sizes() != at::IntArrayRef(shape) || t->scalar_type() != k.scalar_type() || t->device() != c.dev ||
            !t->is_contiguous() || !aligned16(*t))
          bad(name, "out must be two contiguous, 16-byte aligned " + shape_text(shape) + " tensors on " + c.dev.str());
      if (meet(k, v)) bad(name, "out's tensors must not overlap");
    }
    const int dt = float_code(name, k.scalar_type());
    if (N > 0 && c.L > 0 && c.H > 0) {
      ic_page_q8_rows rows = {};
      rows.slots = static_cast<int32_t*>(slots.data_ptr());
      rows.k_buf = k.data_ptr();
      rows.v_buf = v.data_ptr();
      rows.n_tokens = N;
      rows.stride_l = c.H * N * c.D;
      rows.stride_h = N * c.D;
      rows.stride_t = c.D;
      const ic_page_q8_args x = q8_args(c, &rows, dt, nullptr);
      check_status(ic_page_read_q8(&x, at::cuda::getCurrentCUDAStream(c.dev.index()).stream()), "ic_page_read_q8");
    }
    return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(k)).get(), THPObjectPtr(THPVariable_Wrap(v)).get());
  });
}

// q, k_cache, v_cache, k_scale, v_scale, block_table, lens, q_start, scale or
// None, max_count or None, out or None, return_lse, status -> out or (out, lse)
PyObject* py_paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  static const char* name = "paged_attention";
  if (!arity(name, n, 13)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Cache c = cache_of(name, a + 1);
    if (c.dims != 3) bad(name, "the cache must be one layer's, [H, pool_tokens, D]");
    Tensor q = tensor(a[0], name, "q");
    if (q.dim() != 3 || q.size(2) != c.D || c.H == 0 || q.size(1) == 0 || q.size(1) % c.H)
      bad(name, "q must be [N, Hq, " + std::to_string(c.D) + "] with Hq a multiple of " + std::to_string(c.H) + ", got " +
                    shape_text(q.sizes()));
    const auto type = q.scalar_type();
    if ((type != at::kHalf && type != at::kBFloat16) || q.device() != c.dev)
      bad(name, "q must be float16 or bfloat16 on " + c.dev.str() + ", got " + c10::toString(type) + " on " + q.device().str());
    const Tensor &table = tensor(a[5], name, "block_table"), &lens = tensor(a[6], name, "lens");
    const Tensor& q_start = tensor(a[7], name, "q_start");
    if (table.dim() != 2) bad(name, "block_table must be [S, width]");
    const int64_t S = table.size(0), W = table.size(1), N = q.size(0), Hq = q.size(1);
    ic_paged_attn_args x = {};
    x.block_table = state(name, "block_table", table, c.dev, {S, W});
    x.lens = state(name, "lens", lens, c.dev, {S});
    x.q_start = state(name, "q_start", q_start, c.dev, {S + 1});
    x.dev_status = status_word(name, a[12], c.dev);
    x.scale = static_cast<float>(none(a[8]) ? 1.0 / std::sqrt(static_cast<double>(c.D)) : number(a[8]));
    const int64_t max_count = none(a[9]) ? N : std::max<int64_t>(0, std::min<int64_t>(integer(a[9]), N));
    c10::cuda::CUDAGuard guard(c.dev);
    Tensor out, lse;
    if (none(a[10])) {
      out = fresh(q.sizes(), type, c.dev);
    } else {
      out = tensor(a[10], name, "out");
      if (out.sizes() != q.sizes() || out.scalar_type() != type || out.device() != c.dev || !out.is_contiguous() ||
          !aligned16(out))
        bad(name, "out must be a contiguous, 16-byte aligned tensor like q");
      // a row of q is read by those alone that write the same row of out, before they do
      if (meet(q, out) && (q.data_ptr() != out.data_ptr() || !q.is_contiguous())) bad(name, "out must be q or not overlap it");
    }
    const bool want_lse = truth(a[11]);
    if (want_lse) lse = fresh({N, Hq}, at::kFloat, c.dev);
    if (N > 0 && S > 0) {
      if (!rows16(q)) q = q.clone(at::MemoryFormat::Contiguous);
      x.q = q.data_ptr();
      x.out = out.data_ptr();
      x.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
      x.k = c.k->data_ptr();
      x.v = c.v->data_ptr();
      x.k_scale = static_cast<float*>(c.ks->data_ptr());
      x.v_scale = static_cast<float*>(c.vs->data_ptr());
      x.pool_tokens = c.n;
      x.q_stride_t = N > 1 ? q.stride(0) : 0;
      x.q_stride_h = Hq > 1 ? q.stride(1) : 0;
      x.num_sessions = static_cast<int32_t>(std::min<int64_t>(S, 0x7fffffff));
      x.table_width = static_cast<int32_t>(std::min<int64_t>(W, 0x7fffffff));
      x.num_q_tokens = static_cast<int32_t>(std::min<int64_t>(N, 0x7fffffff));
      x.max_count = static_cast<int32_t>(std::min<int64_t>(max_count, 0x7fffffff));
      x.num_q_heads = static_cast<int32_t>(Hq);
      x.num_kv_heads = static_cast<int32_t>(c.H);
      x.head_dim = static_cast<int32_t>(c.D);
      x.q_dtype = type == at::kHalf ? IC_F16 : IC_BF16;
      x.code_dtype = c.code;
      // on the current stream, for this call alone: captured graphs and calls
      // on other streams have their own
      Tensor work;
      x.workspace_bytes = ic_paged_attention_workspace(&x);
      if (x.workspace_bytes > 0) {
        work = fresh({x.workspace_bytes}, at::kByte, c.dev);
        x.workspace = work.data_ptr();
      }
      check_status(ic_paged_attention(&x, at::cuda::getCurrentCUDAStream(c.dev.index()).stream()), "ic_paged_attention");
    }
    if (!want_lse) return THPVariable_Wrap(out);
    return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(out)).get(), THPObjectPtr(THPVariable_Wrap(lse)).get());
  });
}

// a penalty: a number for every row, or a [S] tensor
Tensor per_row(const char* name, const char* what, PyObject* o, float& all, int64_t S, c10::Device dev) {
  if (none(o)) return Tensor();
  if (!THPVariable_Check(o)) {
    all = static_cast<float>(number(o));
    return Tensor();
  }
  const Tensor& t = THPVariable_Unpack(o);
  if (t.dim() != 1 || t.size(0) != S || t.device() != dev)
    bad(name, std::string(what) + " must be a number or a [" + std::to_string(S) + "] tensor on " + dev.str());
  return t.to(at::kFloat).contiguous();
}

// logits, tokens, token_lens, prompt_lens, repetition, presence, frequency,
// bias_ids, bias_values, bias_lens, mask, out -> out
PyObject* py_process_logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  static const char* name = "process_logits";
  if (!arity(name, n, 12)) return nullptr;
  return guarded([&]() -> PyObject* {
    Tensor x = tensor(a[0], name, "logits");
    const c10::Device dev = device_of(name, x);
    if (x.dim() != 2) bad(name, "logits must be [S, V], got " + shape_text(x.sizes()));
    const int64_t S = x.size(0), V = x.size(1);
    ic_logits_args r = {};
    r.dtype = float_code(name, x.scalar_type());
    if (none(a[1]) && !(none(a[2]) && none(a[3]))) bad(name, "token_lens and prompt_lens need tokens");
    if (none(a[1]) && !(none(a[4]) && none(a[5]) && none(a[6]))) bad(name, "penalties need tokens");
    if (none(a[7]) != none(a[8]) || (none(a[7]) && !none(a[9]))) bad(name, "bias_ids and bias_values come together");
    c10::cuda::CUDAGuard guard(dev);
    if (x.stride(1) != 1 || (S > 1 && x.stride(0) < V)) x = x.contiguous();
    Tensor out;
    if (none(a[11])) {
      out = fresh({S, V}, at::kFloat, dev);
    } else {
      out = tensor(a[11], name, "out");
      if (out.scalar_type() != at::kFloat || out.sizes() != x.sizes() || out.device() != dev || out.stride(1) != 1 ||
          (S > 1 && out.stride(0) < V))
        bad(name, "out must be a float32 " + shape_text(x.sizes()) + " tensor with contiguous rows on " + dev.str());
      const bool alike = S == 1 || out.stride(0) * 4 == x.stride(0) * x.element_size();
      if (meet(x, out) && !(alike && x.scalar_type() == at::kFloat && x.data_ptr() == out.data_ptr()) &&
          !(alike && S > 1 && rows_apart(x, out, out.stride(0) * 4)))
        bad(name, "out must be logits or not overlap them");
    }
    Tensor tok, tl, pl, ids, vals, bl, mask;
    if (!none(a[1])) tok = ints(name, "tokens", tensor(a[1], name, "tokens"), dev, {S, -1});
    if (!none(a[2])) tl = ints(name, "token_lens", tensor(a[2], name, "token_lens"), dev, {S});
    if (!none(a[3])) pl = ints(name, "prompt_lens", tensor(a[3], name, "prompt_lens"), dev, {S});
    r.repetition_all = 1.f;
    r.presence_all = r.frequency_all = 0.f;
    const Tensor rep = per_row(name, "repetition", a[4], r.repetition_all, S, dev);
    const Tensor pres = per_row(name, "presence", a[5], r.presence_all, S, dev);
    const Tensor freq = per_row(name, "frequency", a[6], r.frequency_all, S, dev);
    // a number's reciprocal is taken in 64 bits, as torch divides by a number
    r.repetition_all_inv = none(a[4]) || THPVariable_Check(a[4]) ? 1.f : static_cast<float>(1.0 / number(a[4]));
    if (!none(a[7])) {
      ids = ints(name, "bias_ids", tensor(a[7], name, "bias_ids"), dev, {S, -1});
      const Tensor& b = tensor(a[8], name, "bias_values");
      if (b.sizes() != ids.sizes() || b.device() != dev) bad(name, "bias_values must be " + shape_text(ids.sizes()) + " on " + dev.str());
      vals = b.to(at::kFloat).contiguous();
    }
    if (!none(a[9])) bl = ints(name, "bias_lens", tensor(a[9], name, "bias_lens"), dev, {S});
    if (!none(a[10])) {
      const Tensor& m = tensor(a[10], name, "mask");
      if (m.scalar_type() != at::kInt || m.dim() != 2 || m.size(0) != S || m.size(1) < (V + 31) / 32 || m.device() != dev)
        bad(name, "mask must be int32 [" + std::to_string(S) + ", >= " + std::to_string((V + 31) / 32) + "] on " + dev.str());
      mask = m.contiguous();
    }
    if (S == 0 || V == 0) return THPVariable_Wrap(out);
    const auto i32 = [](const Tensor& t) { return t.defined() ? static_cast<const int32_t*>(t.data_ptr()) : nullptr; };
    const auto f32 = [](const Tensor& t) { return t.defined() ? static_cast<const float*>(t.data_ptr()) : nullptr; };
    r.logits = x.data_ptr();
    r.out = static_cast<float*>(out.data_ptr());
    r.logits_stride = std::max(x.stride(0), V);
    r.out_stride = std::max(out.stride(0), V);
    r.max_tokens = tok.defined() ? static_cast<int32_t>(tok.size(1)) : 0;
    r.bias_width = ids.defined() ? static_cast<int32_t>(ids.size(1)) : 0;
    r.tokens = r.max_tokens ? i32(tok) : nullptr;
    r.token_lens = i32(tl);
    r.prompt_lens = i32(pl);
    r.repetition = f32(rep);
    r.presence = f32(pres);
    r.frequency = f32(freq);
    r.bias_ids = r.bias_width ? i32(ids) : nullptr;
    r.bias_values = f32(vals);
    r.bias_lens = i32(bl);
    r.mask = i32(mask);
    r.tokens_stride = r.max_tokens;
    r.bias_stride = r.bias_width;
    r.mask_stride = mask.defined() ? mask.size(1) : 0;
    r.rows = static_cast<int32_t>(std::min<int64_t>(S, 0x7fffffff));
    if (V > 0x7fffffff) bad(name, "the vocabulary must be below 2^31");
    r.vocab = static_cast<int32_t>(V);
    check_status(ic_process_logits(&r, at::cuda::getCurrentCUDAStream(dev.index()).stream()), "ic_process_logits");
    return THPVariable_Wrap(out);
  });
}

// require_device, raise_for: the Python side's device check and status mapping
PyObject* py_setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity("setup", n, 2)) return nullptr;
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  Py_XSETREF(g_require, a[0]);
  Py_XSETREF(g_raise, a[1]);
  Py_RETURN_NONE;
}

#define IC_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {IC_METHOD(setup),      IC_METHOD(page_plan), IC_METHOD(page_release),
                         IC_METHOD(page_write), IC_METHOD(page_read), IC_METHOD(paged_attention),
                         IC_METHOD(process_logits), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) {
  PyObject* m = PyModule_Create(&module);
  // torch's C++ interface differs from version to version: the loader compares
  if (m && PyModule_AddStringConstant(m, "torch_version", IC_TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
