// dk_native.cpp — decode_attention's call path as a CPython extension (module _dk_native), and
// paging's of a 4-bit cache's step: reads the tensors' sizes, strides and types through ATen,
// checks them, allocates the output and calls the C ABI. One call costs about as much as its launches; the same checks and
// argument marshalling in Python cost 8-10 us, more than a small call's kernels.
//
// decode() takes exactly the calls whose arguments are valid and plain (contiguous tables,
// 16-token pages, the current device, no capture, ordinary Python numbers); for every other
// call it returns None before doing anything, and attention.decode_attention's Python path
// runs it or raises its error.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cmath>
#include <cstdint>
#include <vector>

#include "dk_decode.h"

namespace {

decltype(&dk_decode_attention_ex) g_decode = nullptr;
decltype(&dk_decode_attention_kv) g_decode_kv = nullptr;
decltype(&dk_workspace_bytes) g_workspace_bytes = nullptr;
PyObject* g_get_device = nullptr;      // () -> current device index
PyObject* g_raw_stream = nullptr;      // (device index) -> hipStream_t of its current stream
PyObject* g_capturing = nullptr;       // () -> whether that stream is being captured
PyObject* g_scratch = nullptr;         // (tensor's device index, stream, bytes) -> uint8 tensor

// bind(ex, kv, workspace_bytes: addresses, get_device, raw_stream, capturing, scratch)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long ex, kv, ws;
  PyObject *dev, *stream, *cap, *scratch;
  if (!PyArg_ParseTuple(args, "KKKOOOO", &ex, &kv, &ws, &dev, &stream, &cap, &scratch))
    return nullptr;
  g_decode = reinterpret_cast<decltype(g_decode)>(ex);
  g_decode_kv = reinterpret_cast<decltype(g_decode_kv)>(kv);
  g_workspace_bytes = reinterpret_cast<decltype(g_workspace_bytes)>(ws);
  PyObject** slots[] = {&g_get_device, &g_raw_stream, &g_capturing, &g_scratch};
  PyObject* values[] = {dev, stream, cap, scratch};
  for (int i = 0; i < 4; ++i) {
    Py_INCREF(values[i]);
    Py_XSETREF(*slots[i], values[i]);
  }
  Py_RETURN_NONE;
}

bool int_arg(PyObject* o, int32_t* out) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &over);
  if (over || v < 0 || v > INT32_MAX) return false;
  *out = (int32_t)v;
  return true;
}

// None (given = false) or a finite float > 0
bool positive_arg(PyObject* o, bool* given, float* out) {
  *given = o != Py_None;
  if (!*given) return true;
  if (!PyFloat_CheckExact(o)) return false;
  const double v = PyFloat_AS_DOUBLE(o);
  *out = (float)v;
  return std::isfinite(v) && v > 0.0 && std::isfinite(*out) && *out > 0.f;
}

const at::Tensor* tensor_arg(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

bool table_ok(const at::Tensor& t, at::Device dev) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.device() == dev;
}

long long call_int(PyObject* fn, PyObject* arg) {   // -1 with an error set on failure
  PyObject* r = arg ? PyObject_CallOneArg(fn, arg) : PyObject_CallNoArgs(fn);
  if (!r) return -1;
  const long long v = PyLong_AsLongLong(r);
  Py_DECREF(r);
  return v;
}

// The arguments of decode_attention, by position.
enum Arg {
  kQ, kKv, kIndptr, kIndices, kLast, kSplit, kOut, kWorkspace, kQkPath, kWavesPerGroup,
  kWavesPerCU, kSchedule, kMaxPages, kSmScale, kKScale, kVScale, kLogitCap, kWindow, kSinks, kArgs
};

// The output tensor; an int (the C ABI's nonzero return); None for a call left to Python.
PyObject* decode_impl(PyObject* const* args) {
  if (c10::impl::TorchDispatchModeTLS::any_modes_set()) Py_RETURN_NONE;
  const at::Tensor* qp = tensor_arg(args[kQ]);
  const at::Tensor* ip = tensor_arg(args[kIndptr]);
  const at::Tensor* ix = tensor_arg(args[kIndices]);
  const at::Tensor* ll = tensor_arg(args[kLast]);
  if (!qp || !ip || !ix || !ll) Py_RETURN_NONE;
  const at::Tensor& q = *qp;
  const at::Tensor *k = nullptr, *v = nullptr;
  const bool pair = PyTuple_CheckExact(args[kKv]) && PyTuple_GET_SIZE(args[kKv]) == 2;
  if (pair) {
    k = tensor_arg(PyTuple_GET_ITEM(args[kKv], 0));
    v = tensor_arg(PyTuple_GET_ITEM(args[kKv], 1));
    if (!v) Py_RETURN_NONE;
  } else {
    k = tensor_arg(args[kKv]);
  }
  if (!k) Py_RETURN_NONE;

  const at::Device dev = q.device();
  const bool f16 = q.scalar_type() == at::kHalf, kv8 = k->scalar_type() == at::kFloat8_e4m3fn;
  // a 4-bit cache: uint8 (num_pages, num_kv_heads, 17 * head_dim)
  const bool kv4 = k->scalar_type() == at::kByte && !pair;
  if (!dev.is_cuda() || q.dim() != 3 || !(f16 || q.scalar_type() == at::kBFloat16) ||
      !(kv8 || kv4 || k->scalar_type() == q.scalar_type()) || k->device() != dev)
    Py_RETURN_NONE;
  const int kd = pair ? 4 : kv4 ? 3 : 5;
  if (k->dim() != kd || (kd == 5 && k->size(1) != 2)) Py_RETURN_NONE;
  const int64_t batch = q.size(0), hq = q.size(1), d = q.size(2);
  const int64_t page = kv4 ? 16 : k->size(kd - 3), hkv = k->size(kd - 2);
  if (page != 16 || batch <= 0 || hq <= 0 || hkv <= 0 || hq % hkv ||
      k->size(kd - 1) != (kv4 ? 17 * d : d) ||
      (d != 64 && d != 128 && d != 256) || batch > INT32_MAX || hq > INT32_MAX ||
      q.stride(2) != 1 || k->stride(kd - 1) != 1)
    Py_RETURN_NONE;
  if (pair && (v->sizes() != k->sizes() || v->strides() != k->strides() ||
               v->scalar_type() != k->scalar_type() || v->device() != dev))
    Py_RETURN_NONE;
  if (!table_ok(*ip, dev) || !table_ok(*ix, dev) || !table_ok(*ll, dev) ||
      ip->size(0) != batch + 1 || ll->size(0) != batch)
    Py_RETURN_NONE;

  int32_t split = 0;
  dk_options o{};
  if (args[kSplit] != Py_None && !int_arg(args[kSplit], &split)) Py_RETURN_NONE;
  if (!int_arg(args[kQkPath], &o.qk_path) || !int_arg(args[kWavesPerGroup], &o.waves_per_group) ||
      !int_arg(args[kWavesPerCU], &o.waves_per_cu) || !int_arg(args[kSchedule], &o.schedule) ||
      !int_arg(args[kMaxPages], &o.max_pages_per_seq))
    Py_RETURN_NONE;
  if (args[kWindow] != Py_None && !int_arg(args[kWindow], &o.window)) Py_RETURN_NONE;
  bool given = false;
  if (!positive_arg(args[kSmScale], &given, &o.sm_scale)) Py_RETURN_NONE;
  const bool no_cap = PyFloat_CheckExact(args[kLogitCap]) && PyFloat_AS_DOUBLE(args[kLogitCap]) == 0.0;
  if (!no_cap && !positive_arg(args[kLogitCap], &given, &o.logit_cap)) Py_RETURN_NONE;
  float scale[2] = {1.f, 1.f};
  for (int i = 0; i < 2; ++i) {
    if (!positive_arg(args[kKScale + i], &given, &scale[i])) Py_RETURN_NONE;
    if (!kv8 && given) Py_RETURN_NONE;   // Python decides (1.0) or refuses
  }
  if (kv8) {
    o.kv_dtype = DK_KV_FP8_E4M3;
    o.k_scale = scale[0];
    o.v_scale = scale[1];
  }
  if (kv4) o.kv_dtype = DK_KV_MXFP4;
  if (args[kSinks] != Py_None) {
    const at::Tensor* s = tensor_arg(args[kSinks]);
    if (!s || s->scalar_type() != at::kFloat || s->dim() != 1 || s->size(0) != hq ||
        !s->is_contiguous() || s->device() != dev)
      Py_RETURN_NONE;
    o.sinks = static_cast<const float*>(s->data_ptr());
  }
  at::Tensor out;
  if (args[kOut] != Py_None) {
    const at::Tensor* t = tensor_arg(args[kOut]);
    if (!t || t->sizes() != q.sizes() || t->scalar_type() != q.scalar_type() ||
        t->device() != dev || t->stride(2) != 1)
      Py_RETURN_NONE;
    out = *t;
  }
  const int64_t need = (int64_t)g_workspace_bytes((int32_t)batch, (int32_t)hq, (int32_t)hkv,
                                                  (int32_t)d, split);
  at::Tensor ws;
  if (need && args[kWorkspace] != Py_None) {
    const at::Tensor* t = tensor_arg(args[kWorkspace]);
    if (!t || t->device() != dev || t->numel() * (int64_t)t->element_size() < need)
      Py_RETURN_NONE;
    ws = *t;
  }

  const long long cur = call_int(g_get_device, nullptr);
  if (cur == -1 && PyErr_Occurred()) return nullptr;
  if (cur != dev.index()) Py_RETURN_NONE;
  PyObject* idx = PyLong_FromLong(dev.index());
  if (!idx) return nullptr;
  PyObject* stream = PyObject_CallOneArg(g_raw_stream, idx);
  if (!stream) {
    Py_DECREF(idx);
    return nullptr;
  }
  void* const raw = PyLong_AsVoidPtr(stream);
  size_t ws_bytes = ws.defined() ? (size_t)(ws.numel() * (int64_t)ws.element_size()) : 0;
  bool leave = false, failed = PyErr_Occurred() != nullptr;
  if (!failed && need && !ws.defined()) {
    // a captured call allocates its own scratch: left to Python
    PyObject* c = PyObject_CallNoArgs(g_capturing);
    failed = c == nullptr;
    leave = c != Py_False;
    Py_XDECREF(c);
    if (!failed && !leave) {
      PyObject* bytes = PyLong_FromLongLong(need);
      PyObject* w = bytes ? PyObject_CallFunctionObjArgs(g_scratch, idx, stream, bytes, nullptr)
                          : nullptr;
      failed = w == nullptr;
      if (w) ws = THPVariable_Unpack(w);
      Py_XDECREF(w);
      Py_XDECREF(bytes);
      ws_bytes = (size_t)need;   // not the buffer's size: see attention._launch
    }
  }
  Py_DECREF(idx);
  Py_DECREF(stream);
  if (failed) return nullptr;
  if (leave) Py_RETURN_NONE;

  if (!out.defined()) out = at::empty({batch, hq, d}, q.options());
  dk_strides s{};
  s.q_b = q.stride(0);
  s.q_h = q.stride(1);
  s.kv_p = k->stride(0);
  s.kv_r = pair || kv4 ? 0 : k->stride(1);
  s.kv_s = kv4 ? 0 : k->stride(kd - 3);
  s.kv_h = k->stride(kd - 2);
  s.o_b = out.stride(0);
  s.o_h = out.stride(1);
  const int32_t* tables[] = {static_cast<const int32_t*>(ip->data_ptr()),
                             static_cast<const int32_t*>(ix->data_ptr()),
                             static_cast<const int32_t*>(ll->data_ptr())};
  const void *qd = q.data_ptr(), *kd_ = k->data_ptr(), *vd = pair ? v->data_ptr() : nullptr;
  void *od = out.data_ptr(), *wd = ws.defined() ? ws.data_ptr() : nullptr;
  const int64_t pages = k->size(0), indices = ix->size(0);
  const int32_t dtype = f16 ? DK_F16 : DK_BF16;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = pair ? g_decode_kv(qd, kd_, vd, tables[0], tables[1], tables[2], od, wd, ws_bytes,
                          (int32_t)batch, (int32_t)hq, (int32_t)hkv, (int32_t)d, 16, pages,
                          indices, dtype, &s, split, &o, raw)
            : g_decode(qd, kd_, tables[0], tables[1], tables[2], od, wd, ws_bytes,
                       (int32_t)batch, (int32_t)hq, (int32_t)hkv, (int32_t)d, 16, pages, indices,
                       dtype, &s, split, &o, raw);
  Py_END_ALLOW_THREADS
  if (rc != DK_OK) return PyLong_FromLong(rc);
  if (args[kOut] != Py_None) {
    Py_INCREF(args[kOut]);
    return args[kOut];
  }
  return THPVariable_Wrap(std::move(out));
}

PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs || !g_decode) {
    PyErr_SetString(PyExc_TypeError, "_dk_native.decode: not bound, or a wrong argument count");
    return nullptr;
  }
  try {
    return decode_impl(args);
  } catch (const std::exception&) {
    // an ATen error (no storage, out of memory): the Python path meets and reports it
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
}

// ---- a 4-bit cache's step: block tables, rows written and read, prefill attention. Each takes
// plain calls (contiguous vectors, the current device, ordinary Python numbers) and returns None for
// the others, as decode() does; a nonzero C ABI return comes back as an int.

decltype(&dk_grow_block_tables) g_grow = nullptr;
decltype(&dk_kv4_write) g_kv4_write = nullptr;
decltype(&dk_kv4_read) g_kv4_read = nullptr;
decltype(&dk_extend_attention_kv4) g_extend = nullptr;
decltype(&dk_extend_kv4_workspace_bytes) g_extend_bytes = nullptr;

// bind_paging(grow_block_tables, kv4_write, kv4_read, extend_attention_kv4,
// extend_kv4_workspace_bytes: addresses), after bind()
PyObject* bind_paging(PyObject*, PyObject* args) {
  unsigned long long grow, write, read, extend, bytes;
  if (!PyArg_ParseTuple(args, "KKKKK", &grow, &write, &read, &extend, &bytes)) return nullptr;
  g_extend = reinterpret_cast<decltype(g_extend)>(extend);
  g_extend_bytes = reinterpret_cast<decltype(g_extend_bytes)>(bytes);
  g_grow = reinterpret_cast<decltype(g_grow)>(grow);
  g_kv4_write = reinterpret_cast<decltype(g_kv4_write)>(write);
  g_kv4_read = reinterpret_cast<decltype(g_kv4_read)>(read);
  Py_RETURN_NONE;
}

// A contiguous 1-D int32 or int64 tensor on dev, of n entries (any number for n < 0).
const at::Tensor* index_arg(PyObject* o, at::Device dev, int64_t n) {
  const at::Tensor* t = tensor_arg(o);
  return t && (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong) && t->dim() == 1 &&
                 t->is_contiguous() && t->device() == dev && (n < 0 || t->size(0) == n)
             ? t
             : nullptr;
}

// head_dim of a 4-bit cache on a GPU, 0 for another tensor
int64_t cache_dim(const at::Tensor* t) {
  if (!t || t->scalar_type() != at::kByte || t->dim() != 3 || !t->device().is_cuda() ||
      t->stride(2) != 1 || t->size(1) <= 0 || t->size(1) > INT32_MAX)
    return 0;
  const int64_t d = t->size(2) / 17;
  return t->size(2) % 17 == 0 && (d == 64 || d == 128 || d == 256) ? d : 0;
}

// The raw stream of dev where it is the current device: 1; another device: 0; -1: error set.
int stream_of(at::Device dev, void** raw) {
  const long long cur = call_int(g_get_device, nullptr);
  if (cur == -1 && PyErr_Occurred()) return -1;
  if (cur != dev.index()) return 0;
  PyObject* idx = PyLong_FromLong(dev.index());
  PyObject* s = idx ? PyObject_CallOneArg(g_raw_stream, idx) : nullptr;
  Py_XDECREF(idx);
  if (!s) return -1;
  *raw = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  return PyErr_Occurred() ? -1 : 1;
}

// A contiguous tensor over a part of `all`'s memory. Made directly: a view through the dispatcher
// costs the host 0.6 us, and a step's tables are six.
PyObject* part_of(const at::Tensor& all, int64_t offset, at::IntArrayRef sizes) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()),
                                                          all.key_set(), all.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return THPVariable_Wrap(std::move(t));
}

// (block_table, rows, cached_lens, new_lens, new_pages, num_tokens, capacity): the six tensors
PyObject* grow_impl(PyObject* const* args) {
  const at::Tensor* table = tensor_arg(args[0]);
  if (!table || table->scalar_type() != at::kInt || table->dim() != 2 ||
      !table->device().is_cuda() || (table->stride(1) != 1 && table->size(1) > 1) ||
      (table->stride(0) < table->size(1) && table->size(0) > 1))
    Py_RETURN_NONE;
  const at::Device dev = table->device();
  const at::Tensor* rows = index_arg(args[1], dev, -1);
  const int64_t batch = rows ? rows->size(0) : 0;
  if (batch <= 0 || batch >= INT32_MAX || table->size(1) > INT32_MAX) Py_RETURN_NONE;
  const at::Tensor* cached = index_arg(args[2], dev, batch);
  const at::Tensor* fresh = index_arg(args[3], dev, batch);
  const at::Tensor* pages = index_arg(args[4], dev, -1);
  int32_t tokens = 0, capacity = 0;
  if (!cached || !fresh || !pages || pages->scalar_type() != at::kInt ||
      !int_arg(args[5], &tokens) || !int_arg(args[6], &capacity))
    Py_RETURN_NONE;
  void* raw = nullptr;
  const int on = stream_of(dev, &raw);
  if (on < 0) return nullptr;
  if (!on) Py_RETURN_NONE;
  const int64_t sizes[6] = {batch + 1, capacity, batch, batch + 1, tokens, tokens};
  int64_t total = 0;
  for (int64_t n : sizes) total += n;
  const at::Tensor all = at::empty({total}, table->options());
  int32_t* base = static_cast<int32_t*>(all.data_ptr());
  int32_t* part[6];
  for (int i = 0; i < 6; ++i) {
    part[i] = base;
    base += sizes[i];
  }
  int rc;
  int32_t* const td = static_cast<int32_t*>(table->data_ptr());
  const void *rd = rows->data_ptr(), *cd = cached->data_ptr(), *nd = fresh->data_ptr();
  const int32_t* const pd = static_cast<const int32_t*>(pages->data_ptr());
  Py_BEGIN_ALLOW_THREADS
  rc = g_grow(td, table->stride(0), table->size(0), (int32_t)table->size(1), rd,
              rows->scalar_type() == at::kLong, cd, cached->scalar_type() == at::kLong, nd,
              fresh->scalar_type() == at::kLong, pd, pages->size(0), (int32_t)batch, part[0],
              part[1], capacity, part[2], part[3], part[4], part[5], tokens, raw);
  Py_END_ALLOW_THREADS
  if (rc != DK_OK) return PyLong_FromLong(rc);
  PyObject* out = PyTuple_New(6);
  int64_t at = 0;
  for (int i = 0; out && i < 6; ++i) {
    PyObject* t = part_of(all, at, {sizes[i]});
    at += sizes[i];
    if (!t) Py_CLEAR(out);
    else PyTuple_SET_ITEM(out, i, t);
  }
  return out;
}

// (k_new, v_new, cache, slots, q, inv_freq, positions, rope_style): 0, or the C ABI's return
PyObject* write_impl(PyObject* const* args) {
  const at::Tensor *k = tensor_arg(args[0]), *v = tensor_arg(args[1]), *c = tensor_arg(args[2]);
  const int64_t d = cache_dim(c);
  if (!k || !v || !d) Py_RETURN_NONE;
  const at::Device dev = c->device();
  const bool f16 = k->scalar_type() == at::kHalf;
  if (!(f16 || k->scalar_type() == at::kBFloat16) || k->dim() != 3 || k->device() != dev ||
      v->device() != dev || v->scalar_type() != k->scalar_type() || v->sizes() != k->sizes() ||
      v->strides() != k->strides() || k->stride(2) != 1 || k->size(0) <= 0 ||
      k->size(1) != c->size(1) || k->size(2) != d)
    Py_RETURN_NONE;
  const int64_t n = k->size(0);
  const at::Tensor* slots = index_arg(args[3], dev, n);
  if (!slots) Py_RETURN_NONE;
  const at::Tensor *q = nullptr, *freq = nullptr, *pos = nullptr;
  if (args[4] != Py_None) {
    q = tensor_arg(args[4]);
    if (!q || q->dim() != 3 || q->size(0) != n || q->size(2) != d || q->stride(2) != 1 ||
        q->scalar_type() != k->scalar_type() || q->device() != dev || q->size(1) > INT32_MAX)
      Py_RETURN_NONE;
  }
  if (args[5] != Py_None) {
    freq = tensor_arg(args[5]);
    if (!freq || freq->scalar_type() != at::kFloat || freq->numel() != d / 2 ||
        !freq->is_contiguous() || freq->device() != dev)
      Py_RETURN_NONE;
  }
  if (args[6] != Py_None && !(pos = index_arg(args[6], dev, n))) Py_RETURN_NONE;
  int32_t style = 0;
  if (!int_arg(args[7], &style) || style > 1 || (freq && !pos)) Py_RETURN_NONE;
  void* raw = nullptr;
  const int on = stream_of(dev, &raw);
  if (on < 0) return nullptr;
  if (!on) Py_RETURN_NONE;
  dk_strides s{};
  if (q) {
    s.q_b = q->stride(0);
    s.q_h = q->stride(1);
  }
  s.kv_p = c->stride(0);
  s.kv_h = c->stride(1);
  void *qd = q ? q->data_ptr() : nullptr, *cd = c->data_ptr();
  const void *kd = k->data_ptr(), *vd = v->data_ptr(), *sd = slots->data_ptr();
  const void* pd = pos ? pos->data_ptr() : nullptr;
  const float* fd = freq ? static_cast<const float*>(freq->data_ptr()) : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_kv4_write(qd, kd, vd, k->stride(0), k->stride(1), cd, sd,
                   slots->scalar_type() == at::kLong, pd, pos && pos->scalar_type() == at::kLong,
                   fd, style, n, q ? (int32_t)q->size(1) : 1, (int32_t)c->size(1), (int32_t)d,
                   c->size(0), f16 ? DK_F16 : DK_BF16, &s, raw);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// (cache, slots, dtype code): (k, v)
PyObject* read_impl(PyObject* const* args) {
  const at::Tensor* c = tensor_arg(args[0]);
  const int64_t d = cache_dim(c);
  int32_t dtype = 0;
  if (!d || !int_arg(args[2], &dtype) || (dtype != DK_F16 && dtype != DK_BF16)) Py_RETURN_NONE;
  const at::Device dev = c->device();
  const at::Tensor* slots = index_arg(args[1], dev, -1);
  if (!slots || slots->size(0) <= 0) Py_RETURN_NONE;
  void* raw = nullptr;
  const int on = stream_of(dev, &raw);
  if (on < 0) return nullptr;
  if (!on) Py_RETURN_NONE;
  const int64_t n = slots->size(0), hkv = c->size(1);
  const at::Tensor both =
      at::empty({2, n, hkv, d}, c->options().dtype(dtype == DK_F16 ? at::kHalf : at::kBFloat16));
  uint8_t* const kd = static_cast<uint8_t*>(both.data_ptr());
  uint8_t* const vd = kd + n * hkv * d * 2;
  const void *cd = c->data_ptr(), *sd = slots->data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_kv4_read(cd, c->stride(0), c->stride(1), sd, slots->scalar_type() == at::kLong, kd, vd,
                  hkv * d, d, n, (int32_t)hkv, (int32_t)d, c->size(0), dtype, raw);
  Py_END_ALLOW_THREADS
  if (rc != DK_OK) return PyLong_FromLong(rc);
  PyObject* k = part_of(both, 0, {n, hkv, d});
  PyObject* v = k ? part_of(both, n * hkv * d, {n, hkv, d}) : nullptr;
  PyObject* out = v ? PyTuple_Pack(2, k, v) : nullptr;
  Py_XDECREF(k);
  Py_XDECREF(v);
  return out;
}

// A list or tuple of n host integers as int32 (n < 0: any number); false: not that
bool ints_arg(PyObject* o, Py_ssize_t n, std::vector<int32_t>* out) {
  const bool list = PyList_CheckExact(o);
  if (!list && !PyTuple_CheckExact(o)) return false;
  const Py_ssize_t m = list ? PyList_GET_SIZE(o) : PyTuple_GET_SIZE(o);
  if (n >= 0 && m != n) return false;
  out->resize((size_t)m);
  for (Py_ssize_t i = 0; i < m; ++i)
    if (!int_arg(list ? PyList_GET_ITEM(o, i) : PyTuple_GET_ITEM(o, i), &(*out)[i])) return false;
  return true;
}

// (q, cache, block_table, rows, new_lens, all_lens, out, scale, logit_cap, window, sinks): the output
PyObject* extend_impl(PyObject* const* args) {
  const at::Tensor *q = tensor_arg(args[0]), *c = tensor_arg(args[1]), *t = tensor_arg(args[2]);
  const int64_t d = cache_dim(c);
  if (!q || !t || !d) Py_RETURN_NONE;
  const at::Device dev = c->device();
  const bool f16 = q->scalar_type() == at::kHalf;
  if (!(f16 || q->scalar_type() == at::kBFloat16) || q->dim() != 3 || q->device() != dev ||
      q->size(2) != d || q->stride(2) != 1 || q->size(1) <= 0 || q->size(1) % c->size(1) ||
      q->size(1) > INT32_MAX || t->scalar_type() != at::kInt || t->dim() != 2 || t->device() != dev ||
      (t->stride(1) != 1 && t->size(1) > 1) || t->size(1) > INT32_MAX)
    Py_RETURN_NONE;
  std::vector<int32_t> rows, news, alls;
  if (!ints_arg(args[3], -1, &rows) || !ints_arg(args[4], (Py_ssize_t)rows.size(), &news) ||
      !ints_arg(args[5], (Py_ssize_t)rows.size(), &alls) || rows.size() > INT32_MAX)
    Py_RETURN_NONE;
  at::Tensor out;
  if (args[6] != Py_None) {
    const at::Tensor* o = tensor_arg(args[6]);
    if (!o || o->sizes() != q->sizes() || o->scalar_type() != q->scalar_type() ||
        o->device() != dev || o->stride(2) != 1)
      Py_RETURN_NONE;
    out = *o;
  }
  bool given = false;
  float scale = 0.f, cap = 0.f;
  int32_t window = 0;
  const bool no_cap = PyFloat_CheckExact(args[8]) && PyFloat_AS_DOUBLE(args[8]) == 0.0;
  if (!positive_arg(args[7], &given, &scale)) Py_RETURN_NONE;
  if (!given) scale = (float)(1.0 / std::sqrt((double)d));
  if ((!no_cap && !positive_arg(args[8], &given, &cap)) ||
      (args[9] != Py_None && !int_arg(args[9], &window)))
    Py_RETURN_NONE;
  const float* sinks = nullptr;
  if (args[10] != Py_None) {
    const at::Tensor* x = tensor_arg(args[10]);
    if (!x || x->scalar_type() != at::kFloat || x->dim() != 1 || x->size(0) != q->size(1) ||
        !x->is_contiguous() || x->device() != dev)
      Py_RETURN_NONE;
    sinks = static_cast<const float*>(x->data_ptr());
  }
  void* raw = nullptr;
  const int on = stream_of(dev, &raw);
  if (on < 0) return nullptr;
  if (!on) Py_RETURN_NONE;
  const int32_t n = (int32_t)rows.size(), hq = (int32_t)q->size(1), hkv = (int32_t)c->size(1);
  const size_t need = g_extend_bytes(n, news.data(), alls.data(), hq, hkv, (int32_t)d, window);
  if (!out.defined()) out = at::empty(q->sizes(), q->options().memory_format(at::MemoryFormat::Contiguous));
  at::Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, c->options());
  dk_extend_strides s{};
  s.q_b = q->stride(0);
  s.q_h = q->stride(1);
  s.o_b = out.stride(0);
  s.o_h = out.stride(1);
  const void *qd = q->data_ptr(), *cd = c->data_ptr();
  void *od = out.data_ptr(), *wd = need ? ws.data_ptr() : nullptr;
  const int32_t* td = static_cast<const int32_t*>(t->data_ptr());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_extend(qd, cd, c->stride(0), c->stride(1), td, t->stride(0), t->size(0),
                (int32_t)t->size(1), rows.data(), news.data(), alls.data(), od, wd, need, n,
                q->size(0), hq, hkv, (int32_t)d, c->size(0), f16 ? DK_F16 : DK_BF16, &s, scale, cap,
                window, sinks, raw);
  Py_END_ALLOW_THREADS
  if (rc != DK_OK) return PyLong_FromLong(rc);
  if (args[6] != Py_None) {
    Py_INCREF(args[6]);
    return args[6];
  }
  return THPVariable_Wrap(std::move(out));
}

template <PyObject* (*Impl)(PyObject* const*), int N>
PyObject* paging_call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N || !g_grow || !g_get_device) {
    PyErr_SetString(PyExc_TypeError, "_dk_native: not bound, or a wrong argument count");
    return nullptr;
  }
  if (c10::impl::TorchDispatchModeTLS::any_modes_set()) Py_RETURN_NONE;
  try {
    return Impl(args);
  } catch (const std::exception&) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;   // as in decode()
  }
}

template <PyObject* (*Impl)(PyObject* const*), int N>
PyCFunction fast_call() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paging_call<Impl, N>));
}

PyMethodDef kMethods[] = {
    {"bind", bind, METH_VARARGS, "addresses and callables that decode() uses"},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL,
     "decode_attention's arguments by position: the output, a C ABI error code, or None"},
    {"bind_paging", bind_paging, METH_VARARGS, "addresses that paging's calls use"},
    {"grow_block_tables", fast_call<grow_impl, 7>(), METH_FASTCALL,
     "grow_block_tables' arguments but out: its six tensors, a C ABI error code, or None"},
    {"write_kv4", fast_call<write_impl, 8>(), METH_FASTCALL,
     "write_kv4's arguments: the C ABI's return, or None"},
    {"read_kv4", fast_call<read_impl, 3>(), METH_FASTCALL,
     "cache, slots, dtype code: (k, v), a C ABI error code, or None"},
    {"extend_attention_kv4", fast_call<extend_impl, 11>(), METH_FASTCALL,
     "extend_attention_kv4's arguments: the output, a C ABI error code, or None"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_dk_native", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

// BUILT_FOR: what this file was compiled against (the C ABI's version and struct sizes, torch,
// Python); attention.py binds it only where all of it is what runs.
PyMODINIT_FUNC PyInit__dk_native() {
  PyObject* m = PyModule_Create(&kModule);
  if (!m) return nullptr;
  PyObject* built = Py_BuildValue("(iiisii)", DK_ABI_VERSION, (int)sizeof(dk_options),
                                  (int)sizeof(dk_strides), TORCH_VERSION, PY_MAJOR_VERSION,
                                  PY_MINOR_VERSION);
  if (!built || PyModule_AddObject(m, "BUILT_FOR", built) != 0) {
    Py_XDECREF(built);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
