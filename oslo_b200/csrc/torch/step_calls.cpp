// The calls of one decoding step without Python's share of the work.
//
// A decoding step's kernels run for a few microseconds; reading forty attributes of a dozen tensors from Python takes ten (one call
// in a loop: storing a token 17 us through Python and 6 us through here, attention over 200 tokens 12 and 7 us, logits 11 and 5 us).  The
// functions here do what the Python functions of the same names do for the ordinary case (CUDA tensors of the current device,
// no gradient, nothing to copy or convert) and launch through the same C entry points of the kernel library, whose addresses
// bind() receives.  Whatever is not ordinary, a wrong argument among it, returns NotImplemented, and the Python function goes
// on to convert it or to say what is wrong with it.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../step_args.h"

namespace {

using at::Tensor;

int (*append_fn)(const OsloPagedAppendArgs*) = nullptr;
int (*attention_fn)(const OsloPagedAttentionArgs*) = nullptr;
long long (*workspace_fn)(const OsloPagedAttentionArgs*) = nullptr;
int (*logits_fn)(const OsloProcessLogitsArgs*) = nullptr;
constexpr int kDevices = 64;
int64_t status_words[kDevices] = {};

PyObject* other() { Py_RETURN_NOTIMPLEMENTED; }

int type_code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1; }
int64_t address(const Tensor& t) { return reinterpret_cast<int64_t>(t.data_ptr()); }
bool on(const Tensor& t, int device) { return t.is_cuda() && t.get_device() == device; }
// strided storage without a gradient that would be recorded or a forward derivative
bool plain(const Tensor& t, bool recording) {
  return t.layout() == at::kStrided && !(recording && t.requires_grad()) && !t._fw_grad(0).defined() && !t.is_neg();
}

struct Args {
  PyObject* const* args;
  bool has(int i) const { return args[i] != Py_None; }
  const Tensor* tensor(int i) const { return THPVariable_CheckExact(args[i]) ? &THPVariable_Unpack(args[i]) : nullptr; }
};

// 16-byte aligned heads with unit inner stride
bool aligned(const Tensor& t, int64_t step) {
  return t.stride(3) == 1 && (t.stride(0) | t.stride(1) | t.stride(2)) % step == 0 && address(t) % 16 == 0;
}
bool ints(const Tensor* t, int64_t b, int device) {
  return t && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == b && t->is_contiguous() && on(*t, device);
}
bool pages(const Tensor* k, const Tensor* v, const Tensor* table, int64_t b, int64_t hd, at::ScalarType type, int device) {
  if (!k || !v || !table || k->dim() != 4 || k->sizes() != v->sizes() || k->scalar_type() != type || v->scalar_type() != type) return false;
  if (k->size(3) != hd || hd <= 0 || hd % 8 || hd > 256 || k->size(2) <= 0 || k->size(2) % 16 || k->size(1) <= 0) return false;
  for (const Tensor* t : {k, v})
    if (t->stride(3) != 1 || t->stride(2) != hd || (t->stride(0) | t->stride(1)) % 8 || address(*t) % 16 || !on(*t, device)) return false;
  return table->scalar_type() == at::kInt && table->dim() == 2 && table->size(0) == b && (table->stride(1) == 1 || table->size(1) <= 1) &&
         on(*table, device) && table->size(1) * k->size(2) <= 0x3FFFFFFF;
}
template <typename F>
int launch(F f) {  // a full launch queue blocks: other Python threads go on meanwhile
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = f();
  Py_END_ALLOW_THREADS;
  return rc;
}

// (k, v, k_pages, v_pages, block_table, start, count, q, rope)
PyObject* paged_kv_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a{args};
  if (n != 9 || !append_fn) return other();
  const Tensor *k = a.tensor(0), *v = a.tensor(1), *kp = a.tensor(2), *vp = a.tensor(3), *table = a.tensor(4), *start = a.tensor(5);
  if (!k || !v || !k->is_cuda() || k->dim() != 4) return other();
  const int device = k->get_device();
  if (device >= kDevices || !status_words[device] || c10::cuda::current_device() != device) return other();
  const int code = type_code(k->scalar_type());
  const int64_t b = k->size(0), s = k->size(1), hkv = k->size(2), d = k->size(3);
  if (code < 0 || k->sizes() != v->sizes() || v->scalar_type() != k->scalar_type() || !on(*v, device)) return other();
  if (!pages(kp, vp, table, b, d, k->scalar_type(), device) || kp->size(1) != hkv || !ints(start, b, device)) return other();
  const bool recording = at::GradMode::is_enabled();
  const int64_t step = 16 / k->element_size();
  if (!plain(*k, recording) || !plain(*v, recording) || !plain(*kp, recording) || !plain(*vp, recording)) return other();
  if (!aligned(*k, step) || !aligned(*v, step)) return other();
  OsloPagedAppendArgs x{};
  if (a.has(6)) {
    const Tensor* count = a.tensor(6);
    if (!ints(count, b, device)) return other();
    x.count = address(*count);
  }
  const Tensor* q = nullptr;
  if (a.has(7)) {
    q = a.tensor(7);
    if (!q || q->dim() != 4 || q->size(0) != b || q->size(1) != s || q->size(2) == 0 || q->size(3) != d || q->scalar_type() != k->scalar_type() ||
        !on(*q, device) || !plain(*q, recording) || !aligned(*q, step))
      return other();
    x.q = address(*q), x.hq = q->size(2), x.q_b = q->stride(0), x.q_s = q->stride(1), x.q_h = q->stride(2);
  }
  if (a.has(8)) {
    PyObject* rope = args[8];
    if (!PyTuple_CheckExact(rope) || PyTuple_GET_SIZE(rope) != 4 || !PyLong_Check(PyTuple_GET_ITEM(rope, 2))) return other();
    PyObject* items[2] = {PyTuple_GET_ITEM(rope, 0), PyTuple_GET_ITEM(rope, 1)};
    if (!THPVariable_CheckExact(items[0]) || !THPVariable_CheckExact(items[1])) return other();
    const Tensor &cosb = THPVariable_Unpack(items[0]), &sinb = THPVariable_Unpack(items[1]);
    const long rot = PyLong_AsLong(PyTuple_GET_ITEM(rope, 2));
    const int neox = PyObject_IsTrue(PyTuple_GET_ITEM(rope, 3));
    if (PyErr_Occurred() || neox < 0) {
      PyErr_Clear();
      return other();
    }
    if (rot <= 0 || rot % 2 || rot > d || cosb.dim() != 2 || cosb.size(1) != rot / 2 || sinb.sizes() != cosb.sizes()) return other();
    for (const Tensor* t : {&cosb, &sinb})
      if (t->scalar_type() != at::kFloat || !t->is_contiguous() || !on(*t, device) || !plain(*t, recording)) return other();
    x.cosb = address(cosb), x.sinb = address(sinb), x.rot = rot, x.neox = neox, x.positions = cosb.size(0);
  }
  Tensor out;
  if (q) out = at::empty(q->sizes(), q->options().requires_grad(false)), x.q_out = address(out);
  x.k = address(*k), x.v = address(*v), x.k_pages = address(*kp), x.v_pages = address(*vp), x.table = address(*table), x.start = address(*start);
  x.status = status_words[device], x.stream = reinterpret_cast<int64_t>(c10::cuda::getCurrentCUDAStream(device).stream());
  x.k_b = k->stride(0), x.k_s = k->stride(1), x.k_h = k->stride(2), x.v_b = v->stride(0), x.v_s = v->stride(1), x.v_h = v->stride(2);
  x.k_page = kp->stride(0), x.k_head = kp->stride(1), x.v_page = vp->stride(0), x.v_head = vp->stride(1), x.table_row = table->stride(0);
  x.b = b, x.s = s, x.hkv = hkv, x.d = d, x.page_size = kp->size(2), x.max_pages = table->size(1), x.num_pages = kp->size(0), x.dtype = code;
  if (launch([&] { return append_fn(&x); })) return other();
  if (!q) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// (q, k_pages, v_pages, block_table, lengths, scale, mask)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a{args};
  if (n != 7 || !attention_fn) return other();
  const Tensor *q = a.tensor(0), *kp = a.tensor(1), *vp = a.tensor(2), *table = a.tensor(3), *lens = a.tensor(4);
  if (!q || !q->is_cuda() || q->dim() != 4) return other();
  const int device = q->get_device();
  if (device >= kDevices || !status_words[device] || c10::cuda::current_device() != device) return other();
  const int code = type_code(q->scalar_type());
  const int64_t b = q->size(0), s = q->size(1), hq = q->size(2), d = q->size(3);
  if (code < 0 || !pages(kp, vp, table, b, d, q->scalar_type(), device) || !ints(lens, b, device)) return other();
  const int64_t hkv = kp->size(1);
  const bool recording = at::GradMode::is_enabled();
  if (hq == 0 || hq % hkv || !plain(*q, recording) || !plain(*kp, recording) || !plain(*vp, recording) || !aligned(*q, 16 / q->element_size()))
    return other();
  OsloPagedAttentionArgs x{};
  x.mask_len = -1;
  x.scale = 1.0 / std::sqrt(static_cast<double>(d));
  if (a.has(5)) {
    if (!PyFloat_Check(args[5])) return other();
    x.scale = PyFloat_AS_DOUBLE(args[5]);
    if (!(std::abs(x.scale) <= 0x1p127)) return other();
  }
  if (a.has(6)) {
    const Tensor* m = a.tensor(6);
    if (!m || m->scalar_type() != at::kFloat || m->dim() != 4 || (m->size(0) != b && m->size(0) != 1) || m->size(1) != 1 ||
        (m->size(2) != s && m->size(2) != 1) || m->stride(3) != 1 || !on(*m, device) || !plain(*m, recording))
      return other();
    x.mask = address(*m), x.mask_b = m->size(0) == 1 ? 0 : m->stride(0), x.mask_s = m->size(2) == 1 ? 0 : m->stride(2), x.mask_len = m->size(3);
  }
  x.q = address(*q), x.k_pages = address(*kp), x.v_pages = address(*vp), x.table = address(*table), x.lens = address(*lens);
  x.status = status_words[device], x.stream = reinterpret_cast<int64_t>(c10::cuda::getCurrentCUDAStream(device).stream());
  x.q_b = q->stride(0), x.q_s = q->stride(1), x.q_h = q->stride(2), x.k_page = kp->stride(0), x.k_head = kp->stride(1);
  x.v_page = vp->stride(0), x.v_head = vp->stride(1), x.table_row = table->stride(0);
  x.b = b, x.s = s, x.hkv = hkv, x.group = hq / hkv, x.d = d, x.page_size = kp->size(2), x.max_pages = table->size(1);
  x.num_pages = kp->size(0), x.dtype = code;
  Tensor out = at::empty({b, s, hq * d}, q->options().requires_grad(false)), ws;
  x.out = address(out);
  const long long room = workspace_fn(&x);
  if (room < 0) return other();
  if (room > 0) ws = at::empty({room}, q->options().dtype(at::kByte).requires_grad(false)), x.workspace = address(ws);
  if (launch([&] { return attention_fn(&x); })) return other();
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// one number a row, or a number for all of them
bool penalty(const Args& a, int i, int64_t rows, int device, bool recording, long long& where, double& number) {
  if (PyFloat_Check(a.args[i])) {
    number = PyFloat_AS_DOUBLE(a.args[i]);
    return true;
  }
  const Tensor* t = a.tensor(i);
  if (!t || t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != rows || !t->is_contiguous() || !on(*t, device) || !plain(*t, recording)) return false;
  where = address(*t);
  return true;
}

// (logits, tokens, token_lengths, prompt_lengths, repetition, presence, frequency, bias, allowed)
PyObject* process_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a{args};
  if (n != 9 || !logits_fn) return other();
  const Tensor* x = a.tensor(0);
  if (!x || !x->is_cuda() || x->dim() != 2) return other();
  const int device = x->get_device();
  if (c10::cuda::current_device() != device) return other();
  const int code = type_code(x->scalar_type());
  const bool recording = at::GradMode::is_enabled();
  const int64_t rows = x->size(0), vocab = x->size(1);
  if (code < 0 || !plain(*x, recording) || x->stride(1) != 1) return other();
  OsloProcessLogitsArgs y{};
  if (!penalty(a, 4, rows, device, recording, y.rep, y.rep_s) || !penalty(a, 5, rows, device, recording, y.pres, y.pres_s) ||
      !penalty(a, 6, rows, device, recording, y.freq, y.freq_s) || (!y.rep && !(y.rep_s >= 0x1p-126 && y.rep_s <= 0x1p126)))
    return other();
  if (a.has(1)) {
    const Tensor* t = a.tensor(1);
    if (!t || t->dim() != 2 || t->size(0) != rows || !on(*t, device) || (t->stride(1) != 1 && t->size(1) > 1)) return other();
    y.tok64 = t->scalar_type() == at::kLong;
    if (!y.tok64 && t->scalar_type() != at::kInt) return other();
    if (t->size(1) > 0) y.tokens = address(*t), y.history = t->size(1), y.tok_stride = t->stride(0);
  } else if (a.has(2) || a.has(3) || y.rep || y.pres || y.freq || y.rep_s != 1.0 || y.pres_s != 0.0 || y.freq_s != 0.0) {
    return other();
  }
  if (a.has(2)) {
    const Tensor* t = a.tensor(2);
    if (!ints(t, rows, device)) return other();
    y.token_lens = address(*t);
  }
  if (a.has(3)) {
    const Tensor* t = a.tensor(3);
    if (!ints(t, rows, device)) return other();
    y.prompt_lens = address(*t);
  }
  if (a.has(7)) {
    const Tensor* t = a.tensor(7);
    if (!t || t->scalar_type() != at::kFloat || !on(*t, device) || !plain(*t, recording)) return other();
    if (t->dim() == 2 ? t->size(0) != rows || t->size(1) != vocab || t->stride(1) != 1 : t->dim() != 1 || t->size(0) != vocab || t->stride(0) != 1)
      return other();
    y.bias = address(*t), y.bias_stride = t->dim() == 2 ? t->stride(0) : 0;
  }
  if (a.has(8)) {
    const Tensor* t = a.tensor(8);
    if (!t || t->scalar_type() != at::kInt || t->dim() != 2 || (t->size(0) != rows && t->size(0) != 1) || t->size(1) != (vocab + 31) / 32 ||
        (t->stride(1) != 1 && t->size(1) > 1) || !on(*t, device))
      return other();
    y.allowed = address(*t), y.allowed_stride = t->size(0) > 1 ? t->stride(0) : 0;
  }
  Tensor out = at::empty({rows, vocab}, x->options().requires_grad(false));
  y.x = address(*x), y.y = address(out), y.x_stride = x->stride(0), y.y_stride = vocab, y.rows = rows, y.vocab = vocab, y.dtype = code;
  y.stream = reinterpret_cast<int64_t>(c10::cuda::getCurrentCUDAStream(device).stream());
  if (launch([&] { return logits_fn(&y); })) return other();
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// (append, attention, attention workspace, logits): addresses of the kernel library's entry points
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a, b, c, d;
  if (!PyArg_ParseTuple(args, "KKKK", &a, &b, &c, &d)) return nullptr;
  append_fn = reinterpret_cast<int (*)(const OsloPagedAppendArgs*)>(a);
  attention_fn = reinterpret_cast<int (*)(const OsloPagedAttentionArgs*)>(b);
  workspace_fn = reinterpret_cast<long long (*)(const OsloPagedAttentionArgs*)>(c);
  logits_fn = reinterpret_cast<int (*)(const OsloProcessLogitsArgs*)>(d);
  Py_RETURN_NONE;
}
// (device, address of its status word)
PyObject* status(PyObject*, PyObject* args) {
  int device;
  unsigned long long at;
  if (!PyArg_ParseTuple(args, "iK", &device, &at)) return nullptr;
  if (device >= 0 && device < kDevices) status_words[device] = static_cast<int64_t>(at);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"paged_kv_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_kv_append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_attention)), METH_FASTCALL, nullptr},
    {"process_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(process_logits)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {"status", status, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_oslo_b200_step", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__oslo_b200_step() { return PyModule_Create(&module); }
