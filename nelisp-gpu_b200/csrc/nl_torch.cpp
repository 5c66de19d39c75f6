// nl_torch.cpp -- the Python module nelisp_cuda._serving: the serving entry
// points for torch tensors.
//
// These are called once a layer a token, and their kernels run for 2 to 12 us at
// the smallest sizes: reading the tensors, checking them and packing the
// arguments in Python took as long (6 to 14 us a call).  Each function here
// checks its tensors, fills the C ABI's structure and calls the library that
// nelisp_cuda._lib has loaded (its entry points are bound by address); it
// returns the library's code.  A refusal is a ValueError.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <sstream>
#include <string>

#include "nelisp_cuda.h"

namespace {

using at::ScalarType;
using at::Tensor;

struct Refused {
  std::string text;
};
struct Raised {};                // a Python error is set

template <typename... A> [[noreturn]] void refuse(const A &...a) {
  std::ostringstream s;
  (s << ... << a);
  throw Refused{s.str()};
}

// The library's entry points, by address.
struct Api {
  decltype(&nl_qk_norm_rope_dev) norm_rope;
  decltype(&nl_qk_norm_rope_bwd_workspace_bytes) norm_rope_bwd_bytes;
  decltype(&nl_qk_norm_rope_bwd_dev) norm_rope_bwd;
  decltype(&nl_kv_append_dev) kv_append;
  decltype(&nl_kv_read_dev) kv_read;
  decltype(&nl_kv_move_dev) kv_move;
  decltype(&nl_tree_attn_workspace_bytes) tree_bytes;
  decltype(&nl_tree_attn_dev) tree;
  c10::DeviceIndex device;
} bound;
PyObject *binder;                // binds them, on the first call with a CUDA tensor

Api &api() {
  if (!bound.tree) {
    PyObject *r = binder ? PyObject_CallNoArgs(binder) : nullptr;
    if (!r && PyErr_Occurred()) throw Raised{};
    Py_XDECREF(r);
    if (!bound.tree) refuse("the library is not bound");
  }
  return bound;
}

// ---- arguments ------------------------------------------------------------------

const Tensor &tensor(PyObject *o) {
  if (!THPVariable_Check(o)) refuse("expected a tensor, not ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
// The kernels run on the library's device.
void on_device(const Tensor &t) {
  if (t.get_device() != api().device)
    refuse("a tensor on ", t.device(), ": the library's device is cuda:", (int)api().device);
}
const Tensor &flat(PyObject *o, ScalarType type) {
  const Tensor &t = tensor(o);
  if (t.scalar_type() != type || !t.is_cuda() || !t.is_contiguous())
    refuse("expected a contiguous CUDA tensor of ", type, ", not ", t.scalar_type(), " ", t.sizes(),
           " with strides ", t.strides(), " on ", t.device());
  on_device(t);
  return t;
}
int row_type(const Tensor &t) {
  if (t.scalar_type() == at::kFloat) return NL_F32;
  if (t.scalar_type() == at::kBFloat16) return NL_BF16;
  refuse("expected f32 or bf16 rows, not ", t.scalar_type());
}
// 2-D rows with unit inner stride.
const Tensor &rows(PyObject *o, ScalarType type) {
  const Tensor &t = tensor(o);
  if (t.scalar_type() != type || !t.is_cuda() || t.dim() != 2 ||
      (t.stride(1) != 1 && t.size(1) > 1))
    refuse("expected CUDA rows of ", type, " (2-D, unit inner stride), not ", t.scalar_type(), " ",
           t.sizes(), " with strides ", t.strides(), " on ", t.device());
  on_device(t);
  return t;
}
// Elements from a row to the next.  One row may have any stride (torch calls it
// contiguous all the same), and none is used.
uint64_t stride_of(const Tensor &t) {
  return t.size(0) > 1 ? (uint64_t)t.stride(0) : ((uint64_t)t.size(1) + 7) / 8 * 8;
}
uint32_t u32(int64_t v) {
  if (v < 0 || v > (int64_t)UINT32_MAX) refuse("a size of ", v, " does not fit 32 bits");
  return (uint32_t)v;
}
int64_t integer(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
float real(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return (float)v;
}
// The call, on the library's device and torch's current stream there.
template <typename A> int launch(int (*entry)(const A *, void *), const A &args) {
  const c10::cuda::CUDAGuard guard(api().device);
  return entry(&args, c10::cuda::getCurrentCUDAStream(api().device).stream());
}

// WORKSPACE as given, or of the caching allocator: it belongs to the current
// stream, so that calls on different streams never share one.
struct Workspace {
  c10::DataPtr held;
  void *at;
  size_t bytes;
  Workspace(PyObject *given, size_t need, const Tensor &like) {
    if (given != Py_None) {
      const Tensor &t = tensor(given);
      if (!t.is_cuda() || !t.is_contiguous()) refuse("workspace: a contiguous CUDA tensor");
      on_device(t);
      at = t.data_ptr();
      bytes = t.nbytes();
      return;
    }
    const c10::cuda::CUDAGuard guard(like.device());
    held = c10::GetAllocator(c10::kCUDA)->allocate(need);
    at = held.get();
    bytes = need;
  }
};

nl_kv_cache cache_of(PyObject *const *o, int64_t head_dim) {
  const Tensor &kc = flat(o[0], at::kByte), &vc = flat(o[2], at::kByte);
  const Tensor &kp = flat(o[1], at::kInt), &vp = flat(o[3], at::kInt);
  if (kc.dim() != 4 || vc.sizes() != kc.sizes() || kp.sizes() != kc.sizes().slice(0, 3) ||
      vp.sizes() != kp.sizes())
    refuse("cache codes of ", kc.sizes(), " and ", vc.sizes(), ", words of ", kp.sizes(), " and ",
           vp.sizes());
  const int64_t row = kc.size(3);
  if (head_dim <= 0 || (row != head_dim && 2 * row != head_dim))
    refuse("rows of ", row, " bytes for heads of ", head_dim);
  return {row == head_dim ? NL_KV_I8 : NL_KV_I4, u32(kc.size(1)), u32(head_dim), u32(kc.size(2)),
          u32(kc.size(0)), kc.data_ptr(), (uint32_t *)kp.data_ptr(), vc.data_ptr(),
          (uint32_t *)vp.data_ptr()};
}

// ---- Q/K norm + rotation ----------------------------------------------------------

// QKV, GQ, GK, CO, SI, POS and two tensors of rows, EPS and PAIRS: the fields
// that both directions have.
template <typename A>
void norm_rope_fields(A &x, PyObject *const *o, const Tensor &qkv, const Tensor &q, const Tensor &k,
                      PyObject *eps, PyObject *pairs) {
  const Tensor &gq = flat(o[1], at::kFloat), &gk = flat(o[2], at::kFloat);
  const Tensor &co = flat(o[3], at::kFloat), &si = flat(o[4], at::kFloat);
  const Tensor &pos = flat(o[5], at::kInt);
  const int64_t n = qkv.size(0), hd = gq.numel();
  if (hd == 0 || gk.numel() != hd) refuse("gains of different or no length");
  if (co.dim() != 2 || co.sizes() != si.sizes()) refuse("CO and SI: two tables of one 2-D shape");
  if (pos.numel() != n || q.size(0) != n || k.size(0) != n)
    refuse(n, " rows of QKV, ", pos.numel(), " positions, ", q.size(0), " and ", k.size(0),
           " rows");
  if (q.size(1) % hd || k.size(1) % hd || q.size(1) + k.size(1) > qkv.size(1))
    refuse("rows of ", qkv.size(1), " values do not hold heads of ", hd, ": ", q.size(1), " + ",
           k.size(1));
  if (PyUnicode_Check(pairs) && PyUnicode_CompareWithASCIIString(pairs, "half") == 0)
    x.pairs = NL_PAIRS_HALF;
  else if (PyUnicode_Check(pairs) && PyUnicode_CompareWithASCIIString(pairs, "adjacent") == 0)
    x.pairs = NL_PAIRS_ADJACENT;
  else
    refuse("pairs: 'half' or 'adjacent'");
  x.qkv = qkv.data_ptr();
  x.x_stride = stride_of(qkv);
  x.gq = (const float *)gq.data_ptr();
  x.gk = (const float *)gk.data_ptr();
  x.co = (const float *)co.data_ptr();
  x.si = (const float *)si.data_ptr();
  x.pos = (const int32_t *)pos.data_ptr();
  x.n = u32(n);
  x.heads = u32(q.size(1) / hd);
  x.kv_heads = u32(k.size(1) / hd);
  x.head_dim = u32(hd);
  x.rot_dim = u32(2 * co.size(1));
  x.rope_rows = u32(co.size(0));
  x.eps = real(eps);
}

// QKV GQ GK CO SI POS Q K eps pairs
int norm_rope(PyObject *const *o) {
  nl_qk_norm_rope_args x = {};
  const Tensor &first = tensor(o[0]);
  x.dtype = row_type(first);
  const ScalarType type = first.scalar_type();
  const Tensor &qkv = rows(o[0], type), &q = rows(o[6], type), &k = rows(o[7], type);
  norm_rope_fields(x, o, qkv, q, k, o[8], o[9]);
  x.q = q.data_ptr();
  x.q_stride = stride_of(q);
  x.k = k.data_ptr();
  x.k_stride = stride_of(k);
  return launch(api().norm_rope, x);
}

// QKV GQ GK CO SI POS DQ DK DQKV DGQ DGK eps pairs workspace
int norm_rope_bwd(PyObject *const *o) {
  nl_qk_norm_rope_bwd_args x = {};
  const Tensor &first = tensor(o[0]);
  x.dtype = row_type(first);
  const ScalarType type = first.scalar_type();
  const Tensor &qkv = rows(o[0], type), &dq = rows(o[6], type), &dk = rows(o[7], type);
  const Tensor &dqkv = rows(o[8], type);
  norm_rope_fields(x, o, qkv, dq, dk, o[11], o[12]);
  const Tensor &dgq = flat(o[9], at::kFloat), &dgk = flat(o[10], at::kFloat);
  if (dgq.numel() != x.head_dim || dgk.numel() != x.head_dim)
    refuse("DGQ and DGK: one value per gain");
  if (dqkv.size(0) != x.n || dqkv.size(1) < dq.size(1) + dk.size(1))
    refuse("DQKV of ", dqkv.sizes(), " for ", x.n, " rows");
  x.dq = dq.data_ptr();
  x.dq_stride = stride_of(dq);
  x.dk = dk.data_ptr();
  x.dk_stride = stride_of(dk);
  x.dqkv = dqkv.data_ptr();
  x.dx_stride = stride_of(dqkv);
  x.dgq = (float *)dgq.data_ptr();
  x.dgk = (float *)dgk.data_ptr();
  const Workspace ws(o[13], api().norm_rope_bwd_bytes(x.head_dim), qkv);
  x.workspace = ws.at;
  x.ws_bytes = ws.bytes;
  return launch(api().norm_rope_bwd, x);
}

// ---- the cache ------------------------------------------------------------------

nl_kv_rows_args rows_of(PyObject *ko, PyObject *vo, PyObject *slots, PyObject *const *cache) {
  nl_kv_rows_args x = {};
  const Tensor &first = tensor(ko);
  x.dtype = row_type(first);
  const ScalarType type = first.scalar_type();
  const Tensor &k = rows(ko, type), &v = rows(vo, type), &slot = flat(slots, at::kInt);
  const Tensor &kc = tensor(cache[0]);
  if (kc.dim() != 4) refuse("cache codes have 4 dimensions");
  const int64_t kvh = kc.size(1);
  if (v.sizes() != k.sizes() || slot.numel() != k.size(0) || kvh == 0 || k.size(1) % kvh)
    refuse("rows of ", k.sizes(), " and ", v.sizes(), ", ", slot.numel(), " slots, ", kvh,
           " key heads");
  x.cache = cache_of(cache, k.size(1) / kvh);
  x.n = u32(k.size(0));
  x.slot = (const int32_t *)slot.data_ptr();
  x.k = k.data_ptr();
  x.k_stride = stride_of(k);
  x.v = v.data_ptr();
  x.v_stride = stride_of(v);
  return x;
}

// K V SLOT KC KP VC VP
int kv_append(PyObject *const *o) {
  const nl_kv_rows_args x = rows_of(o[0], o[1], o[2], o + 3);
  return launch(api().kv_append, x);
}

// SLOT KC KP VC VP K V
int kv_read(PyObject *const *o) {
  const nl_kv_rows_args x = rows_of(o[5], o[6], o[0], o + 1);
  return launch(api().kv_read, x);
}

// SRC DST KC KP VC VP head_dim
int kv_move(PyObject *const *o) {
  const Tensor &src = flat(o[0], at::kInt), &dst = flat(o[1], at::kInt);
  if (src.dim() != 2 || src.sizes() != dst.sizes()) refuse("SRC and DST: [batch, count] each");
  const nl_kv_move_args x = {cache_of(o + 2, integer(o[6])), (const int32_t *)src.data_ptr(),
                             (const int32_t *)dst.data_ptr(), u32(src.size(0)), u32(src.size(1))};
  return launch(api().kv_move, x);
}

// ---- tree attention ---------------------------------------------------------------

// Q KC KP VC VP TABLE LEN MASK O head_dim scale lse workspace
int tree_attn(PyObject *const *o) {
  nl_tree_attn_args x = {};
  const Tensor &first = tensor(o[0]);
  x.dtype = row_type(first);
  const ScalarType type = first.scalar_type();
  const Tensor &q = rows(o[0], type), &out = rows(o[8], type);
  const Tensor &table = flat(o[5], at::kInt), &len = flat(o[6], at::kInt);
  const Tensor &mask = flat(o[7], at::kLong);
  const int64_t head_dim = integer(o[9]);
  x.cache = cache_of(o + 1, head_dim);
  if (mask.dim() != 2 || table.dim() != 2) refuse("MASK and TABLE have 2 dimensions");
  const int64_t batch = mask.size(0), nodes = mask.size(1), heads = q.size(1) / head_dim;
  if (len.numel() != batch || table.size(0) != batch || q.size(0) != batch * nodes ||
      out.sizes() != q.sizes() || q.size(1) != heads * head_dim)
    refuse("tree_attn: rows of ", q.sizes(), ", heads of ", head_dim, ", ", batch, " sequences of ",
           nodes, " nodes, ", len.numel(), " lengths, a table of ", table.sizes(), ", outputs of ",
           out.sizes());
  if (o[11] != Py_None) {
    const Tensor &lse = flat(o[11], at::kFloat);
    if (lse.dim() != 2 || lse.size(0) != q.size(0) || lse.size(1) != heads)
      refuse("lse: a value per row and head");
    x.lse = (float *)lse.data_ptr();
  }
  x.batch = u32(batch);
  x.nodes = u32(nodes);
  x.heads = u32(heads);
  x.max_blocks = u32(table.size(1));
  x.scale = o[10] == Py_None ? (float)(1.0 / std::sqrt((double)head_dim)) : real(o[10]);
  x.q = q.data_ptr();
  x.q_stride = stride_of(q);
  x.table = (const int32_t *)table.data_ptr();
  x.len = (const int32_t *)len.data_ptr();
  x.mask = (const uint64_t *)mask.data_ptr();
  x.o = out.data_ptr();
  x.o_stride = stride_of(out);
  const Workspace ws(o[12], api().tree_bytes(x.nodes, x.heads, x.cache.kv_heads, x.cache.head_dim),
                     q);
  x.workspace = ws.at;
  x.ws_bytes = ws.bytes;
  return launch(api().tree, x);
}

// ---- the module -----------------------------------------------------------------

template <int (*F)(PyObject *const *), int N>
PyObject *call(PyObject *, PyObject *const *args, Py_ssize_t n) {
  try {
    if (n != N) refuse("expected ", N, " arguments, not ", n);
    return PyLong_FromLong(F(args));
  } catch (const Refused &e) {
    PyErr_SetString(PyExc_ValueError, e.text.c_str());
  } catch (const Raised &) {
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// binder(f): f() is to call bind(device, addresses), in the order of Api's fields.
PyObject *set_binder(PyObject *, PyObject *f) {
  Py_INCREF(f);
  Py_XDECREF(binder);
  binder = f;
  Py_RETURN_NONE;
}
PyObject *bind(PyObject *, PyObject *args) {
  int device;
  unsigned long long a[8];
  if (!PyArg_ParseTuple(args, "i(KKKKKKKK)", &device, a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6,
                        a + 7))
    return nullptr;
  bound = {(decltype(bound.norm_rope))a[0], (decltype(bound.norm_rope_bwd_bytes))a[1],
           (decltype(bound.norm_rope_bwd))a[2], (decltype(bound.kv_append))a[3],
           (decltype(bound.kv_read))a[4], (decltype(bound.kv_move))a[5],
           (decltype(bound.tree_bytes))a[6], (decltype(bound.tree))a[7],
           (c10::DeviceIndex)device};
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"binder", set_binder, METH_O, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))call<norm_rope, 10>, METH_FASTCALL, nullptr},
    {"qk_norm_rope_bwd", (PyCFunction)(void (*)(void))call<norm_rope_bwd, 14>, METH_FASTCALL,
     nullptr},
    {"kv_append", (PyCFunction)(void (*)(void))call<kv_append, 7>, METH_FASTCALL, nullptr},
    {"kv_read", (PyCFunction)(void (*)(void))call<kv_read, 7>, METH_FASTCALL, nullptr},
    {"kv_move", (PyCFunction)(void (*)(void))call<kv_move, 7>, METH_FASTCALL, nullptr},
    {"tree_attn", (PyCFunction)(void (*)(void))call<tree_attn, 13>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving() { return PyModule_Create(&module); }
