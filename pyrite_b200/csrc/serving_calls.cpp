// serving_calls.cpp -- the serving entry points as Python calls them: every check of
// the tensors, the current stream and the launch in one native call.
//
// The kernels behind these calls take 2 to 20 us, so the host's share counts: with
// the checks in Python and the arguments through ctypes a call took 8 to 10 us of
// host time, here about 3 us, most of it the launch itself (append of 16 rows: 10.3 and
// 3.4 us a call).  The functions of
// libpyrite_b200.so are bound by address (bind), so this module and the ctypes
// signatures use one copy of the library.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <initializer_list>
#include <string>

#include "../../include/pyrite_b200.h"

namespace {

decltype(&pyrite_cuda_page_tables) page_tables_fn;
decltype(&pyrite_cuda_qk_rope_kv_paged) append_fn;
decltype(&pyrite_cuda_kv_store_paged) store_fn;
decltype(&pyrite_cuda_attention_paged_workspace_size) workspace_fn;
decltype(&pyrite_cuda_attention_paged) attention_fn;
decltype(&pyrite_cuda_sample_rows) sample_fn;

struct Entry {
  const char* name;
  void** fn;
};
const Entry kEntries[] = {
    {"pyrite_cuda_page_tables", reinterpret_cast<void**>(&page_tables_fn)},
    {"pyrite_cuda_qk_rope_kv_paged", reinterpret_cast<void**>(&append_fn)},
    {"pyrite_cuda_kv_store_paged", reinterpret_cast<void**>(&store_fn)},
    {"pyrite_cuda_attention_paged_workspace_size", reinterpret_cast<void**>(&workspace_fn)},
    {"pyrite_cuda_attention_paged", reinterpret_cast<void**>(&attention_fn)},
    {"pyrite_cuda_sample_rows", reinterpret_cast<void**>(&sample_fn)},
};

const int64_t kHeadDim = 128;
using at::ScalarType;

// ---- arguments --------------------------------------------------------------------------
std::string seen(const at::Tensor& t) {
  std::string s = std::string(", got ") + c10::toString(t.scalar_type()) + " (";
  for (int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.size(d));
  return s + ") on " + t.device().str();
}
const at::Tensor& tensor(PyObject* o, const char* what) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor* optional(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
// An int of the C interface: what does not fit is refused there as a shape.
int as_int(int64_t v) { return v < INT32_MIN ? INT32_MIN : v > INT32_MAX ? INT32_MIN : (int)v; }
c10::Device cuda_device(const at::Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda(), what, " must be a CUDA tensor");
  return t.device();
}
void need(const at::Tensor& t, const char* what, ScalarType type, std::initializer_list<int64_t> shape, c10::Device dev) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.device() == dev && t.sizes().equals(at::IntArrayRef(shape)) &&
                        t.is_contiguous(),
                    what, " must be a contiguous ", c10::toString(type), " tensor of shape ", at::IntArrayRef(shape),
                    " on ", dev.str(), seen(t));
}
int64_t need_list(const at::Tensor& t, const char* what, ScalarType type, c10::Device dev) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.device() == dev && t.dim() == 1 && t.is_contiguous(), what,
                    " must be a contiguous ", c10::toString(type), " vector on ", dev.str(), seen(t));
  return t.size(0);
}
// A float32 matrix with unit stride along its rows; its row stride.  rows, cols < 0: any.
int64_t need_rows(const at::Tensor& t, const char* what, int64_t rows, int64_t cols, c10::Device dev) {
  const bool ok = t.scalar_type() == ScalarType::Float && t.device() == dev && t.dim() == 2 &&
                  (rows < 0 || t.size(0) == rows) && (cols < 0 || t.size(1) == cols) &&
                  (t.stride(1) == 1 || t.size(1) == 1);
  TORCH_CHECK_VALUE(ok, what, " must be a float32 matrix of ", rows < 0 ? "any" : std::to_string(rows), " x ",
                    cols < 0 ? "any" : std::to_string(cols), " with contiguous rows on ", dev.str(), seen(t));
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

struct Pool {
  void *k, *v;
  int type, n_pages, n_kv_heads, page_size;
};
Pool need_pool(PyObject* k_arg, PyObject* v_arg, c10::Device dev) {
  const at::Tensor &k = tensor(k_arg, "pool.k"), &v = tensor(v_arg, "pool.v");
  const ScalarType t = k.scalar_type();
  TORCH_CHECK_VALUE(k.device() == dev && v.device() == dev, "the pool lies on another device");
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes().equals(v.sizes()) && v.scalar_type() == t && k.is_contiguous() &&
                        v.is_contiguous() && k.size(3) == kHeadDim &&
                        (t == ScalarType::Float || t == ScalarType::Half || t == ScalarType::BFloat16),
                    "the pool's k and v must be contiguous tensors of one shape (n_pages, n_kv_heads, page_size, 128) and "
                    "one type, float32, float16 or bfloat16");
  return Pool{k.data_ptr(), v.data_ptr(), t == ScalarType::Float ? 0 : t == ScalarType::Half ? 1 : 30,
              as_int(k.size(0)), as_int(k.size(1)), as_int(k.size(2))};
}
void count_args(Py_ssize_t got, Py_ssize_t want) { TORCH_CHECK_VALUE(got == want, want, " arguments expected"); }

struct Unlocked {  // without the interpreter's lock, also past an exception
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
// The launch on the device's current stream.
template <typename Fn> int launch(c10::Device dev, Fn fn) {
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Unlocked unlocked;
  return fn(stream);
}
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// ---- the calls: None or the outputs; an error code of the library as an int -----------------
PyObject* page_tables(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count_args(n_args, 13);
  const ScalarType i32 = ScalarType::Int;
  const at::Tensor &lens = tensor(a[0], "lens"), &fresh = tensor(a[1], "new_tokens"), &free = tensor(a[3], "free_pages"),
                   &used = tensor(a[4], "used"), &table = tensor(a[5], "table"), &used_out = tensor(a[6], "used_out"),
                   &slots = tensor(a[7], "out.slots"), &positions = tensor(a[8], "out.positions"),
                   &kv_lens = tensor(a[9], "out.kv_lens"), &starts = tensor(a[10], "out.starts"),
                   &ticket = tensor(a[11], "out.ticket");
  const c10::Device dev = cuda_device(lens, "lens");
  const int64_t n = need_list(lens, "lens", i32, dev), capacity = need_list(slots, "out.slots", i32, dev);
  const int64_t n_free = need_list(free, "free_pages", i32, dev);
  need(fresh, "new_tokens", i32, {n}, dev);
  need(used, "used", i32, {1}, dev);
  need(used_out, "used_out", i32, {1}, dev);
  need(positions, "out.positions", i32, {capacity}, dev);
  need(kv_lens, "out.kv_lens", i32, {n}, dev);
  need(starts, "out.starts", i32, {n + 1}, dev);
  need(ticket, "out.ticket", i32, {1}, dev);
  TORCH_CHECK_VALUE(table.scalar_type() == i32 && table.device() == dev && table.dim() == 2 && table.size(0) == n &&
                        (table.stride(1) == 1 || table.size(1) == 1),
                    "table must be an int32 matrix of one row per request, rows contiguous, on the lens' device");
  TORCH_CHECK_VALUE(n == 0 || (kv_lens.data_ptr() != lens.data_ptr() && kv_lens.data_ptr() != fresh.data_ptr()),
                    "out.kv_lens must not be lens or new_tokens itself");
  const int64_t page_size = integer(a[2]), row_stride = integer(a[12]), width = table.size(1);
  const c10::cuda::CUDAGuard guard(dev);
  const int code = launch(dev, [&](void* st) {
    return page_tables_fn(lens.data_ptr<int>(), fresh.data_ptr<int>(), as_int(n), as_int(page_size), free.data_ptr<int>(),
                          as_int(n_free), used.data_ptr<int>(), used_out.data_ptr<int>(), table.data_ptr<int>(),
                          n > 1 ? table.stride(0) : width, as_int(width), as_int(row_stride), slots.data_ptr<int>(),
                          positions.data_ptr<int>(), as_int(capacity), starts.data_ptr<int>(), kv_lens.data_ptr<int>(),
                          reinterpret_cast<unsigned*>(ticket.data_ptr<int>()), st);
  });
  return PyLong_FromLong(code);
  END_HANDLE_TH_ERRORS
}

PyObject* append_kv(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count_args(n_args, 12);
  const at::Tensor &qkv = tensor(a[0], "qkv"), &slots = tensor(a[3], "slots"), &positions = tensor(a[4], "positions"),
                   &rope = tensor(a[5], "rope");
  const int64_t n_heads = integer(a[6]), first = integer(a[10]);
  const at::Tensor *qn = optional(a[7], "q_norm"), *kn = optional(a[8], "k_norm"), *q_out = optional(a[11], "q_out");
  const double eps = PyFloat_AsDouble(a[9]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  const c10::Device dev = cuda_device(qkv, "qkv");
  const Pool p = need_pool(a[1], a[2], dev);
  TORCH_CHECK_VALUE(n_heads > 0 && n_heads <= 1024, "n_heads must be 1 to 1024");
  const int64_t q_dim = n_heads * kHeadDim;
  const int64_t ld = need_rows(qkv, "qkv", -1, q_dim + 2 * p.n_kv_heads * kHeadDim, dev), rows = qkv.size(0);
  TORCH_CHECK_VALUE(rows > 0 && first >= 0 && first <= INT32_MAX,
                    "qkv must have at least one row, and first lie in 0 .. 2^31 - 1");
  need(slots, "slots", ScalarType::Int, {rows}, dev);
  need(positions, "positions", ScalarType::Int, {rows}, dev);
  need(rope, "rope", ScalarType::Double, {rope.dim() ? rope.size(0) : 0, kHeadDim / 2, 2}, dev);
  if (qn) need(*qn, "q_norm", ScalarType::Float, {kHeadDim}, dev);
  if (kn) need(*kn, "k_norm", ScalarType::Float, {kHeadDim}, dev);
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor made;
  if (!q_out) made = at::empty({rows, q_dim}, at::TensorOptions().dtype(ScalarType::Float).device(dev));
  const at::Tensor& q = q_out ? *q_out : made;
  const int64_t ldq = need_rows(q, "q_out", rows, q_dim, dev);
  const int code = launch(dev, [&](void* st) {
    return append_fn(qkv.data_ptr<float>(), ld, qn ? qn->data_ptr<float>() : nullptr, kn ? kn->data_ptr<float>() : nullptr,
                     (int)n_heads, p.n_kv_heads, (int)kHeadDim, eps, (int)first, positions.data_ptr<int>(),
                     slots.data_ptr<int>(), as_int(rows), rope.data_ptr(), as_int(rope.size(0)), q.data_ptr<float>(), ldq,
                     p.k, p.v, p.type, p.n_pages, p.page_size, st);
  });
  if (code != 0) return PyLong_FromLong(code);
  return q_out ? same(a[11]) : THPVariable_Wrap(made);
  END_HANDLE_TH_ERRORS
}

PyObject* store_kv(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count_args(n_args, 5);
  const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &slots = tensor(a[4], "slots");
  const c10::Device dev = cuda_device(k, "k");
  const Pool p = need_pool(a[2], a[3], dev);
  const int64_t ld = need_rows(k, "k", -1, p.n_kv_heads * kHeadDim, dev), rows = k.size(0);
  TORCH_CHECK_VALUE(need_rows(v, "v", rows, p.n_kv_heads * kHeadDim, dev) == ld, "k and v must have one row stride");
  need(slots, "slots", ScalarType::Int, {rows}, dev);
  if (rows == 0) return PyLong_FromLong(0);
  const c10::cuda::CUDAGuard guard(dev);
  return PyLong_FromLong(launch(dev, [&](void* st) {
    return store_fn(k.data_ptr<float>(), v.data_ptr<float>(), ld, slots.data_ptr<int>(), as_int(rows), p.n_kv_heads,
                    (int)kHeadDim, p.k, p.v, p.type, p.n_pages, p.page_size, st);
  }));
  END_HANDLE_TH_ERRORS
}

PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count_args(n_args, 9);
  const ScalarType i32 = ScalarType::Int;
  const at::Tensor &q = tensor(a[0], "q"), &table = tensor(a[3], "table"), &kv_lens = tensor(a[4], "kv_lens");
  const at::Tensor *pages = optional(a[5], "prefix_pages"), *out = optional(a[7], "out"), *ws = optional(a[8], "workspace");
  const int64_t prefix = integer(a[6]);
  const c10::Device dev = cuda_device(q, "q");
  const Pool p = need_pool(a[1], a[2], dev);
  const int64_t ldq = need_rows(q, "q", -1, -1, dev), rows = q.size(0), cols = q.size(1);
  TORCH_CHECK_VALUE(rows > 0 && cols > 0 && p.n_kv_heads > 0 && cols % (kHeadDim * p.n_kv_heads) == 0,
                    "q must be rows of n_heads * 128 values, n_heads a multiple of the pool's KV heads");
  need(kv_lens, "kv_lens", i32, {rows}, dev);
  const int64_t dims = table.dim();
  TORCH_CHECK_VALUE(table.scalar_type() == i32 && table.device() == dev && (dims == 1 || dims == 2) &&
                        (table.stride(-1) == 1 || table.size(-1) == 1) && (dims == 1 || table.size(0) == rows),
                    "table must be int32, one row per row of q (or one list for all), rows contiguous");
  const int64_t width = table.size(-1), stride = dims == 1 ? 0 : rows > 1 ? table.stride(0) : width;
  TORCH_CHECK_VALUE(prefix >= 0 && (prefix == 0 || pages), "a prefix needs its pages and a length of at least 0");
  if (prefix > 0)
    TORCH_CHECK_VALUE(need_list(*pages, "prefix_pages", i32, dev) * p.page_size >= prefix,
                      "prefix_pages hold fewer than prefix_len tokens");
  const int64_t heads = cols / kHeadDim;
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor made, scratch;
  if (!out) made = at::empty({rows, cols}, at::TensorOptions().dtype(ScalarType::Float).device(dev));
  const at::Tensor& o = out ? *out : made;
  const int64_t ldo = need_rows(o, "out", rows, cols, dev);
  if (!ws) {
    const size_t size = workspace_fn(as_int(rows), as_int(heads), p.n_kv_heads, as_int(prefix), p.type);
    TORCH_CHECK_VALUE(size > 0, "no attention of these sizes (1..4096 rows, heads a multiple of the KV heads, 128 values each)");
    scratch = at::empty({(int64_t)size}, at::TensorOptions().dtype(ScalarType::Byte).device(dev));
  } else {
    TORCH_CHECK_VALUE(ws->scalar_type() == ScalarType::Byte && ws->device() == dev && ws->is_contiguous(),
                      "workspace must be a contiguous uint8 tensor on q's device");
  }
  const at::Tensor& w = ws ? *ws : scratch;
  const int code = launch(dev, [&](void* st) {
    return attention_fn(q.data_ptr<float>(), ldq, p.k, p.v, p.type, p.n_pages, p.page_size,
                        prefix > 0 ? pages->data_ptr<int>() : nullptr, as_int(prefix), table.data_ptr<int>(), stride,
                        as_int(width), kv_lens.data_ptr<int>(), as_int(rows), as_int(heads), p.n_kv_heads, (int)kHeadDim,
                        o.data_ptr<float>(), ldo, w.data_ptr(), (size_t)w.numel(), st);
  });
  if (code != 0) return PyLong_FromLong(code);
  return out ? same(a[7]) : THPVariable_Wrap(made);
  END_HANDLE_TH_ERRORS
}

PyObject* sample_rows(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count_args(n_args, 8);
  const ScalarType f32 = ScalarType::Float;
  const at::Tensor &logits = tensor(a[0], "logits"), &u = tensor(a[1], "uniforms"), &temp = tensor(a[2], "temperature");
  const at::Tensor *top_k = optional(a[3], "top_k"), *top_p = optional(a[4], "top_p"), *min_p = optional(a[5], "min_p"),
                   *out = optional(a[6], "out"), *probs = optional(a[7], "probs");
  const c10::Device dev = cuda_device(logits, "logits");
  const int64_t ld = need_rows(logits, "logits", -1, -1, dev), rows = logits.size(0), n = logits.size(1);
  TORCH_CHECK_VALUE(rows > 0 && n > 0, "logits must have at least one row and one column");
  need(u, "uniforms", f32, {rows}, dev);
  need(temp, "temperature", f32, {rows}, dev);
  if (top_k) need(*top_k, "top_k", ScalarType::Int, {rows}, dev);
  if (top_p) need(*top_p, "top_p", f32, {rows}, dev);
  if (min_p) need(*min_p, "min_p", f32, {rows}, dev);
  if (out) need(*out, "out", ScalarType::Int, {rows}, dev);
  if (probs) need(*probs, "probs", f32, {rows}, dev);
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor ids, share;
  if (!out) ids = at::empty({rows}, at::TensorOptions().dtype(ScalarType::Int).device(dev));
  if (!probs) share = at::empty({rows}, at::TensorOptions().dtype(f32).device(dev));
  const int code = launch(dev, [&](void* st) {
    return sample_fn(logits.data_ptr<float>(), ld, (size_t)n, (size_t)rows, u.data_ptr<float>(), temp.data_ptr<float>(),
                     top_k ? top_k->data_ptr<int>() : nullptr, top_p ? top_p->data_ptr<float>() : nullptr,
                     min_p ? min_p->data_ptr<float>() : nullptr, (out ? *out : ids).data_ptr<int>(),
                     (probs ? *probs : share).data_ptr<float>(), st);
  });
  if (code != 0) return PyLong_FromLong(code);
  PyObject* both = PyTuple_New(2);
  if (!both) return nullptr;
  PyTuple_SET_ITEM(both, 0, out ? same(a[6]) : THPVariable_Wrap(ids));
  PyTuple_SET_ITEM(both, 1, probs ? same(a[7]) : THPVariable_Wrap(share));
  return both;
  END_HANDLE_TH_ERRORS
}

// bind(name, address): a function of the library.
PyObject* bind(PyObject*, PyObject* args) {
  const char* name;
  unsigned long long at;
  if (!PyArg_ParseTuple(args, "sK", &name, &at)) return nullptr;
  for (const Entry& e : kEntries)
    if (std::strcmp(e.name, name) == 0) {
      *e.fn = reinterpret_cast<void*>(static_cast<uintptr_t>(at));
      Py_RETURN_NONE;
    }
  PyErr_Format(PyExc_KeyError, "%s", name);
  return nullptr;
}
// The names to bind before the first call.
PyObject* entries(PyObject*, PyObject*) {
  const Py_ssize_t n = sizeof(kEntries) / sizeof(kEntries[0]);
  PyObject* t = PyTuple_New(n);
  for (Py_ssize_t i = 0; t && i < n; ++i) {
    PyObject* s = PyUnicode_FromString(kEntries[i].name);
    if (!s) {
      Py_DECREF(t);
      return nullptr;
    }
    PyTuple_SET_ITEM(t, i, s);
  }
  return t;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {FAST(page_tables), FAST(append_kv), FAST(store_kv), FAST(attention), FAST(sample_rows),
                          {"bind", bind, METH_VARARGS, nullptr}, {"entries", entries, METH_NOARGS, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "serving_calls", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_serving_calls() { return PyModule_Create(&kModule); }
