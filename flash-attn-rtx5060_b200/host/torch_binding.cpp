// Native part of the Python entry points: argument checks, output allocation and the call of the C ABI for torch tensors,
// as one function of the CPython API, and a caller of flash_forward_noalloc for plain numbers; bind_operators() the same for
// flash_backward, flash_cache_append and flash_decode. Nothing is linked or kept
// here: bind() makes both for the library whose entry points it is given, the one that the package has loaded, whatever
// other copies of it the process holds. A small call is bound by
// the host: with ctypes and the checks in Python attention_forward took 9.2 us a call (2.1 of them in the library and
// the driver, 1.5 ctypes, 1.3 the output tensor) where the kernel takes 7.2 (B1 H4 N512 d64).
//
// Every function here answers NotImplemented, or passes its arguments on, where it does not know them, and the Python
// code of the package then does what it always did: errors, tensor subclasses, active torch function or dispatch modes,
// a device other than the current one, the kernels that only tests select.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/flash_forward_b200.h"

namespace {

PyObject* not_here() {
  Py_INCREF(Py_NotImplemented);
  return Py_NotImplemented;
}

bool plain_int(PyObject* o) { return PyLong_Check(o); }
// As ctypes does with an int for a C int: the low bits.
int low_int(PyObject* o) { return static_cast<int>(PyLong_AsUnsignedLongMask(o)); }
bool plain_number(PyObject* o) { return PyFloat_Check(o) || PyLong_Check(o); }

// What bind() was given; the `self` of the functions that it returns, as a capsule.
struct Library {
  decltype(&flash_forward) plain;
  decltype(&flash_forward_alibi) alibi;
  decltype(&flash_forward_lse) lse;
  decltype(&flash_forward_dropout) dropout;
  decltype(&flash_forward_noalloc) noalloc;
  PyObject* ctypes_noalloc;  // takes the calls of noalloc() with anything but plain numbers
};
const Library& library(PyObject* self) { return *static_cast<Library*>(PyCapsule_GetPointer(self, nullptr)); }

// forward(q, k, v, causal, window_left, window_right, softmax_scale, out, alibi_slopes, return_lse, dropout_p, seed):
// the result of attention_forward, an int (status code of a call that failed) or NotImplemented.
PyObject* forward(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) return not_here();
  PyObject *py_out = a[7], *py_slopes = a[8];
  for (int i = 0; i < 3; ++i)
    if (!THPVariable_CheckExact(a[i])) return not_here();
  if (py_out != Py_None && !THPVariable_CheckExact(py_out)) return not_here();
  if (py_slopes != Py_None && !THPVariable_CheckExact(py_slopes)) return not_here();
  if (!PyBool_Check(a[3]) || !PyBool_Check(a[9]) || !plain_int(a[4]) || !plain_int(a[5]) || !plain_number(a[6]) ||
      !plain_number(a[10]) || !plain_int(a[11]))
    return not_here();
  if (at::impl::torch_function_mode_enabled() || c10::impl::dispatch_mode_enabled()) return not_here();

  const at::Tensor &q = THPVariable_Unpack(a[0]), &k = THPVariable_Unpack(a[1]), &v = THPVariable_Unpack(a[2]);
  if (!q.is_cuda() || q.dim() != 4) return not_here();
  const auto device = q.get_device();
  // what the kernel may be given the address of
  auto fits = [&](const at::Tensor& t, at::ScalarType type) {
    return t.is_cuda() && t.get_device() == device && t.scalar_type() == type && t.is_contiguous();
  };
  if (!fits(q, at::kHalf) || !fits(k, at::kHalf) || !fits(v, at::kHalf)) return not_here();
  if (k.sizes() != q.sizes() || v.sizes() != q.sizes()) return not_here();
  if (py_out != Py_None && (!fits(THPVariable_Unpack(py_out), at::kHalf) || THPVariable_Unpack(py_out).numel() < q.numel()))
    return not_here();
  const bool causal = a[3] == Py_True, want_lse = a[9] == Py_True;
  const float scale = static_cast<float>(PyFloat_AsDouble(a[6]));
  const double dropout = PyFloat_AsDouble(a[10]);  // (positive, though 0 as a float, it still asks for the dropout call)
  if (PyErr_Occurred()) {  // an int beyond the range of a double
    PyErr_Clear();
    return not_here();
  }
  if (dropout > 0.0 && want_lse) return not_here();
  const auto B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  const float* slopes = nullptr;
  if (py_slopes != Py_None) {
    const at::Tensor& t = THPVariable_Unpack(py_slopes);
    if (!fits(t, at::kFloat) || t.numel() != H) return not_here();
    slopes = static_cast<const float*>(t.data_ptr());
  }
  if (device != c10::cuda::current_device()) return not_here();

  const at::Tensor out = py_out == Py_None ? at::empty_like(q) : THPVariable_Unpack(py_out);
  at::Tensor lse;
  if (want_lse) lse = at::empty({B, H, N}, q.options().dtype(at::kFloat));
  const void *pq = q.data_ptr(), *pk = k.data_ptr(), *pv = v.data_ptr();
  void* po = out.data_ptr();
  float* pl = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  void* stream = c10::cuda::getCurrentCUDAStream(device).stream();
  const int b = static_cast<int>(B), h = static_cast<int>(H), s = static_cast<int>(N), d = static_cast<int>(D);
  const int wl = low_int(a[4]), wr = low_int(a[5]);
  const unsigned long long seed = PyLong_AsUnsignedLongLongMask(a[11]);
  const Library& lib = library(self);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (dropout > 0.0)
    rc = lib.dropout(pq, pk, pv, po, b, h, s, d, scale, causal, wl, wr, slopes, static_cast<float>(dropout), seed, stream);
  else if (want_lse) rc = lib.lse(pq, pk, pv, po, pl, b, h, s, d, scale, causal, wl, wr, slopes, stream);
  else if (slopes) rc = lib.alibi(pq, pk, pv, po, b, h, s, d, scale, causal, wl, wr, slopes, stream);
  else rc = lib.plain(pq, pk, pv, po, b, h, s, d, scale, causal, wl, wr, stream);
  Py_END_ALLOW_THREADS
  if (rc != FA_OK) return PyLong_FromLong(rc);
  PyObject* py_result = py_out;
  if (py_out == Py_None) py_result = THPVariable_Wrap(out);
  else Py_INCREF(py_out);
  if (!want_lse || !py_result) return py_result;
  PyObject* py_lse = THPVariable_Wrap(lse);
  PyObject* pair = py_lse ? PyTuple_Pack(2, py_result, py_lse) : nullptr;
  Py_DECREF(py_result);
  Py_XDECREF(py_lse);
  return pair;
  END_HANDLE_TH_ERRORS
}

bool address(PyObject* o, void** p) {
  if (o == Py_None) {
    *p = nullptr;
    return true;
  }
  if (!PyLong_CheckExact(o)) return false;
  *p = reinterpret_cast<void*>(PyLong_AsUnsignedLongLongMask(o));
  return true;
}

// flash_forward_noalloc for pointers given as ints or None and numbers
PyObject* noalloc(PyObject* self, PyObject* const* a, Py_ssize_t n, PyObject* names) {
  void *q, *k, *v, *o, *stream;
  bool known = n == 15 && (names == nullptr || PyTuple_GET_SIZE(names) == 0) && address(a[0], &q) && address(a[1], &k) &&
               address(a[2], &v) && address(a[3], &o) && address(a[12], &stream) && plain_number(a[8]);
  constexpr int ints[] = {4, 5, 6, 7, 9, 10, 11, 13, 14};
  for (int i : ints) known = known && plain_int(a[i]);
  float scale = 0.f;
  if (known) {
    scale = static_cast<float>(PyFloat_AsDouble(a[8]));
    if (PyErr_Occurred()) {
      PyErr_Clear();
      known = false;
    }
  }
  const Library& lib = library(self);
  if (!known) return PyObject_Vectorcall(lib.ctypes_noalloc, a, n, names);
  const int x[] = {low_int(a[4]), low_int(a[5]), low_int(a[6]), low_int(a[7]), low_int(a[9]), low_int(a[10]), low_int(a[11]),
                   low_int(a[13]), low_int(a[14])};
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = lib.noalloc(q, k, v, o, x[0], x[1], x[2], x[3], scale, x[4], x[5], x[6], stream, x[7], x[8]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// ---- the operators beside the forward ------------------------------------------------------------------------------------
// What bind_operators() was given.
struct Operators {
  decltype(&flash_backward) backward;
  decltype(&flash_backward_workspace_bytes) backward_bytes;
  decltype(&flash_cache_append) append;
  decltype(&flash_decode) decode;
  decltype(&flash_decode_workspace_bytes) decode_bytes;
};
const Operators& operators(PyObject* self) { return *static_cast<Operators*>(PyCapsule_GetPointer(self, nullptr)); }

// A plain tensor, or None where `optional`; *t is null for None.
bool tensor(PyObject* o, bool optional, const at::Tensor** t) {
  *t = nullptr;
  if (o == Py_None) return optional;
  if (!THPVariable_CheckExact(o)) return false;
  *t = &THPVariable_Unpack(o);
  return true;
}
bool lies_on(const at::Tensor& t, int64_t device, at::ScalarType type) {
  return t.is_cuda() && t.get_device() == device && t.scalar_type() == type;
}
void* data_of(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
// at::empty() of a contiguous CUDA tensor without the dispatcher, which no mode is active to hear of (modes() is asked first):
// 0.4 us less each
at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
at::Tensor workspace_of(size_t bytes, const at::Tensor& like) {
  return new_tensor({static_cast<int64_t>(bytes)}, at::kByte, like);
}
// false (and no error) for what is not a number that the C entry points take
bool scale_of(PyObject* o, float* scale) {
  if (!plain_number(o)) return false;
  *scale = static_cast<float>(PyFloat_AsDouble(o));
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}
bool modes() { return at::impl::torch_function_mode_enabled() || c10::impl::dispatch_mode_enabled(); }

// backward(q, k, v, out, lse, dout, causal, window_left, window_right, softmax_scale, alibi_slopes, dlse, dq, dk, dv): as
// attention_backward answers, an int (status code) or NotImplemented.
PyObject* backward(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 15 || modes()) return not_here();
  const at::Tensor *q, *k, *v, *out, *lse, *dout, *slopes, *dlse, *given[3];
  float scale;
  if (!tensor(a[0], false, &q) || !tensor(a[1], false, &k) || !tensor(a[2], false, &v) || !tensor(a[3], false, &out) ||
      !tensor(a[4], false, &lse) || !tensor(a[5], false, &dout) || !PyBool_Check(a[6]) || !plain_int(a[7]) ||
      !plain_int(a[8]) || !scale_of(a[9], &scale) || !tensor(a[10], true, &slopes) || !tensor(a[11], true, &dlse))
    return not_here();
  for (int i = 0; i < 3; ++i)
    if (!tensor(a[12 + i], true, &given[i])) return not_here();
  if (!q->is_cuda() || q->dim() != 4) return not_here();
  const auto device = q->get_device();
  if (device != c10::cuda::current_device()) return not_here();
  for (const at::Tensor* t : {q, k, v, out, dout, given[0], given[1], given[2]})
    if (t && (!lies_on(*t, device, at::kHalf) || !t->is_contiguous() || t->sizes() != q->sizes())) return not_here();
  const auto B = q->size(0), H = q->size(1), N = q->size(2);
  for (const at::Tensor* t : {lse, dlse})
    if (t && (!lies_on(*t, device, at::kFloat) || !t->is_contiguous() || t->sizes() != q->sizes().slice(0, 3)))
      return not_here();
  if (slopes && (!lies_on(*slopes, device, at::kFloat) || !slopes->is_contiguous() || slopes->numel() != H)) return not_here();
  const Operators& lib = operators(self);
  at::Tensor grads[3];
  for (int i = 0; i < 3; ++i) grads[i] = given[i] ? *given[i] : new_tensor(q->sizes(), at::kHalf, *q);
  const int b = static_cast<int>(B), h = static_cast<int>(H), s = static_cast<int>(N), d = static_cast<int>(q->size(3));
  const size_t bytes = lib.backward_bytes(b, h, s);
  const at::Tensor ws = workspace_of(bytes, *q);
  void* stream = c10::cuda::getCurrentCUDAStream(device).stream();
  const int causal = a[6] == Py_True, wl = low_int(a[7]), wr = low_int(a[8]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = lib.backward(q->data_ptr(), k->data_ptr(), v->data_ptr(), out->data_ptr(), dout->data_ptr(),
                    static_cast<const float*>(lse->data_ptr()), static_cast<const float*>(data_of(dlse)), grads[0].data_ptr(),
                    grads[1].data_ptr(), grads[2].data_ptr(), b, h, s, d, scale, causal, wl, wr,
                    static_cast<const float*>(data_of(slopes)), ws.data_ptr(), bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != FA_OK) return PyLong_FromLong(rc);
  PyObject* result = PyTuple_New(3);
  for (int i = 0; i < 3 && result; ++i) {
    PyObject* x = given[i] ? Py_NewRef(a[12 + i]) : THPVariable_Wrap(grads[i]);
    if (!x) Py_CLEAR(result);
    else PyTuple_SET_ITEM(result, i, x);
  }
  return result;
  END_HANDLE_TH_ERRORS
}

// The cache of a call whose rows are [batch, heads, tokens, head_dim]; false for what the Python code has to refuse.
struct Cache {
  const at::Tensor *k, *v, *table, *lengths, *counts;
  fa_paged_cache c;
  bool read(PyObject* const* a, int64_t batch) {  // k_pages, v_pages, page_table, lengths, counts
    if (!tensor(a[0], false, &k) || !tensor(a[1], false, &v) || !tensor(a[2], false, &table) ||
        !tensor(a[3], false, &lengths) || !tensor(a[4], true, &counts))
      return false;
    if (!k->is_cuda() || k->dim() != 4 || k->stride(3) != 1) return false;
    const auto type = k->scalar_type();
    const auto device = k->get_device();
    if ((type != at::kHalf && type != at::kBFloat16) || device != c10::cuda::current_device() || !lies_on(*v, device, type) ||
        v->sizes() != k->sizes() || v->strides() != k->strides())
      return false;
    if (!lies_on(*table, device, at::kInt) || table->dim() != 2 || table->size(0) != batch || table->stride(1) != 1)
      return false;
    for (const at::Tensor* t : {lengths, counts})
      if (t && (!lies_on(*t, device, at::kInt) || t->dim() != 1 || t->size(0) != batch || !t->is_contiguous())) return false;
    c = fa_paged_cache{k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1), k->stride(2), static_cast<int>(k->size(0)),
                       static_cast<int>(k->size(2)), static_cast<int>(k->size(1)), static_cast<int>(k->size(3)),
                       type == at::kHalf ? FA_FP16 : FA_BF16, static_cast<const int*>(table->data_ptr()), table->stride(0),
                       static_cast<int>(table->size(1)), static_cast<const int*>(lengths->data_ptr()),
                       static_cast<const int*>(data_of(counts))};
    return true;
  }
  bool rows(const at::Tensor& x, int64_t heads, int64_t batch, int64_t tokens, fa_rows* r) const {
    if (!lies_on(x, k->get_device(), k->scalar_type()) || x.dim() != 4 || x.size(0) != batch || x.size(1) != heads ||
        x.size(2) != tokens || x.size(3) != k->size(3) || x.stride(3) != 1)
      return false;
    *r = fa_rows{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)};
    return true;
  }
  // an output that was given: contiguous and shaped like the rows
  bool output(const at::Tensor& x, const at::Tensor& like) const {
    return lies_on(x, k->get_device(), k->scalar_type()) && x.is_contiguous() && x.sizes() == like.sizes();
  }
};

// append(k, v, k_pages, v_pages, page_table, lengths, counts, q, rotary, interleaved, q_out): as cache_append answers
PyObject* append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor *k, *v, *q, *rotary, *given;
  if (n != 11 || modes() || !tensor(a[0], false, &k) || !tensor(a[1], false, &v) || !tensor(a[7], true, &q) ||
      !tensor(a[8], true, &rotary) || !PyBool_Check(a[9]) || !tensor(a[10], true, &given) || k->dim() != 4 || (given && !q))
    return not_here();
  const auto B = k->size(0), T = k->size(2);
  Cache cache;
  fa_rows rk, rv, rq;
  if (!cache.read(a + 2, B) || !cache.rows(*k, cache.c.kv_heads, B, T, &rk) || !cache.rows(*v, cache.c.kv_heads, B, T, &rv))
    return not_here();
  if (q && (q->dim() != 4 || !cache.rows(*q, q->size(1), B, T, &rq))) return not_here();
  if (rotary && (!lies_on(*rotary, k->get_device(), at::kFloat) || rotary->dim() != 2 || !rotary->is_contiguous()))
    return not_here();
  if (given && !cache.output(*given, *q)) return not_here();
  at::Tensor q_out;
  if (q) q_out = given ? *given : new_tensor(q->sizes(), q->scalar_type(), *q);
  void* stream = c10::cuda::getCurrentCUDAStream(k->get_device()).stream();
  const int b = static_cast<int>(B), t = static_cast<int>(T), q_heads = q ? static_cast<int>(q->size(1)) : 0;
  const int dim = rotary ? static_cast<int>(rotary->size(1)) : 0, positions = rotary ? static_cast<int>(rotary->size(0)) : 0;
  const int interleaved = a[9] == Py_True;
  const Operators& lib = operators(self);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = lib.append(&cache.c, &rk, &rv, q ? &rq : nullptr, q ? q_out.data_ptr() : nullptr, b, t, q_heads,
                  static_cast<const float*>(data_of(rotary)), dim, positions, interleaved, stream);
  Py_END_ALLOW_THREADS
  if (rc != FA_OK) return PyLong_FromLong(rc);
  if (!q) Py_RETURN_NONE;
  return given ? Py_NewRef(a[10]) : THPVariable_Wrap(q_out);
  END_HANDLE_TH_ERRORS
}

// decode(q, k_pages, v_pages, page_table, lengths, counts, softmax_scale, window_left, alibi_slopes, return_lse, out): as
// attention_decode answers
PyObject* decode(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor *q, *slopes, *given;
  float scale;
  if (n != 11 || modes() || !tensor(a[0], false, &q) || !scale_of(a[6], &scale) || !plain_int(a[7]) ||
      !tensor(a[8], true, &slopes) || !PyBool_Check(a[9]) || !tensor(a[10], true, &given) || q->dim() != 4)
    return not_here();
  const auto B = q->size(0), H = q->size(1), T = q->size(2);
  Cache cache;
  fa_rows rq;
  if (!cache.read(a + 1, B) || !cache.rows(*q, H, B, T, &rq)) return not_here();
  if (slopes && (!lies_on(*slopes, q->get_device(), at::kFloat) || !slopes->is_contiguous() || slopes->numel() != H))
    return not_here();
  if (given && !cache.output(*given, *q)) return not_here();
  const bool want_lse = a[9] == Py_True;
  const at::Tensor out = given ? *given : new_tensor(q->sizes(), q->scalar_type(), *q);
  at::Tensor lse;
  if (want_lse) lse = new_tensor({B, H, T}, at::kFloat, *q);
  const Operators& lib = operators(self);
  const int b = static_cast<int>(B), h = static_cast<int>(H), t = static_cast<int>(T), wl = low_int(a[7]);
  const size_t bytes = lib.decode_bytes(t, h, cache.c.kv_heads, cache.c.head_dim);
  const at::Tensor ws = workspace_of(bytes, *q);
  void* stream = c10::cuda::getCurrentCUDAStream(q->get_device()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = lib.decode(&cache.c, &rq, out.data_ptr(), want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, b, t, h, scale, wl,
                  static_cast<const float*>(data_of(slopes)), ws.data_ptr(), bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != FA_OK) return PyLong_FromLong(rc);
  PyObject* py_out = given ? Py_NewRef(a[10]) : THPVariable_Wrap(out);
  if (!want_lse || !py_out) return py_out;
  PyObject* py_lse = THPVariable_Wrap(lse);
  PyObject* pair = py_lse ? PyTuple_Pack(2, py_out, py_lse) : nullptr;
  Py_DECREF(py_out);
  Py_XDECREF(py_lse);
  return pair;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*fn)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef operator_def(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr};
}
PyMethodDef backward_def = operator_def<backward>("backward"), append_def = operator_def<append>("append"),
            decode_def = operator_def<decode>("decode");

// bind_operators(addresses of flash_backward, flash_backward_workspace_bytes, flash_cache_append, flash_decode,
// flash_decode_workspace_bytes as ints): (backward, append, decode)
PyObject* bind_operators(PyObject*, PyObject* args) {
  unsigned long long x[5];
  if (!PyArg_ParseTuple(args, "KKKKK", x, x + 1, x + 2, x + 3, x + 4)) return nullptr;
  Operators* ops = new Operators{
      reinterpret_cast<decltype(Operators::backward)>(x[0]), reinterpret_cast<decltype(Operators::backward_bytes)>(x[1]),
      reinterpret_cast<decltype(Operators::append)>(x[2]), reinterpret_cast<decltype(Operators::decode)>(x[3]),
      reinterpret_cast<decltype(Operators::decode_bytes)>(x[4])};
  PyObject* capsule = PyCapsule_New(ops, nullptr, [](PyObject* c) {
    delete static_cast<Operators*>(PyCapsule_GetPointer(c, nullptr));
  });
  if (!capsule) {
    delete ops;
    return nullptr;
  }
  PyObject* all = Py_BuildValue("(NNN)", PyCFunction_New(&backward_def, capsule), PyCFunction_New(&append_def, capsule),
                                PyCFunction_New(&decode_def, capsule));
  Py_DECREF(capsule);
  return all;
}

PyMethodDef forward_def = {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)), METH_FASTCALL, nullptr};
PyMethodDef noalloc_def = {"flash_forward_noalloc", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(noalloc)),
                           METH_FASTCALL | METH_KEYWORDS, nullptr};

void drop_library(PyObject* capsule) {
  Library* lib = static_cast<Library*>(PyCapsule_GetPointer(capsule, nullptr));
  Py_DECREF(lib->ctypes_noalloc);
  delete lib;
}

// bind(addresses of flash_forward, flash_forward_alibi, flash_forward_lse, flash_forward_dropout, flash_forward_noalloc as
// ints, the ctypes function of the last): (forward, noalloc)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long plain, alibi, lse, dropout, noalloc_address;
  PyObject* fn;
  if (!PyArg_ParseTuple(args, "KKKKKO", &plain, &alibi, &lse, &dropout, &noalloc_address, &fn)) return nullptr;
  Library* lib = new Library{reinterpret_cast<decltype(Library::plain)>(plain), reinterpret_cast<decltype(Library::alibi)>(alibi),
                             reinterpret_cast<decltype(Library::lse)>(lse), reinterpret_cast<decltype(Library::dropout)>(dropout),
                             reinterpret_cast<decltype(Library::noalloc)>(noalloc_address), fn};
  PyObject* capsule = PyCapsule_New(lib, nullptr, drop_library);
  if (!capsule) {
    delete lib;
    return nullptr;
  }
  Py_INCREF(fn);
  PyObject* pair = Py_BuildValue("(NN)", PyCFunction_New(&forward_def, capsule), PyCFunction_New(&noalloc_def, capsule));
  Py_DECREF(capsule);
  return pair;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"bind_operators", bind_operators, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

#define FA_STRING_OF(x) #x
#define FA_STRING(x) FA_STRING_OF(x)

PyMODINIT_FUNC PyInit__torch_binding(void) {
  PyObject* m = PyModule_Create(&module);
  // the torch whose object layouts are compiled in
  if (m && PyModule_AddStringConstant(m, "torch_version", FA_STRING(FA_TORCH_VERSION)) < 0) Py_CLEAR(m);
  return m;
}
