// Compiled front of the W8A8 operators' Python functions (int8_linear.py, block_ops.py), for the host time of small calls:
// the checks, the allocations and the call of the C ABI without the interpreter (in a loop an int8 linear of one token takes
// 6.5 us of host time a call here and 11.6 through ctypes, of 24 tokens, which are two launches, 8.0 and 16.5).  A function
// here serves the ordinary case -- plain CUDA tensors of the current device whose rows lie evenly, nothing that asks for a
// gradient -- and returns None for everything else: the Python function then goes its own way, which knows every case and
// says what is wrong with a call.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/DimVector.h>
#include <ATen/ops/empty_cuda_dispatch.h>
#include <ATen/ops/empty_strided_cuda_dispatch.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/lc_b200.h"

namespace {

int32_t* g_status[64] = {};       // a product's status word of each device, once Python has made it

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

int64_t dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return LC_F32;
    case at::kBFloat16: return LC_BF16;
    case at::kHalf: return LC_F16;
    default: return -1;
  }
}

// Plain tensors of one device, the current one; none asks for a gradient that would be recorded, none carries a tangent or
// a negation that its memory does not show.
struct Place {
  int64_t device = -1;
  bool take(const at::Tensor& t) {
    if (!t.is_cuda() || t.layout() != at::kStrided || (t.requires_grad() && c10::GradMode::is_enabled())) return false;
    if (t._fw_grad(0).defined() || t.is_neg()) return false;
    if (device < 0) device = t.get_device();
    return t.get_device() == device;
  }
  // made current inside the library; the stream to launch on
  bool enter(lc_stream_t* stream) const {
    if (device < 0 || device >= 64 || device != c10::cuda::current_device() || lc_set_device((int)device) != LC_OK) return false;
    *stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    return true;
  }
};

// t (..., cols) as rows of contiguous values that lie `pitch` elements apart; false where they do not lie so.
struct Rows {
  int64_t rows = 1, cols = 0, pitch = 0;
};
bool rows_of(const at::Tensor& t, Rows* r) {
  const int64_t d = t.dim();
  if (d < 1) return false;
  const auto size = t.sizes(), stride = t.strides();
  r->cols = size[d - 1];
  if (r->cols == 0 || (stride[d - 1] != 1 && r->cols != 1)) return false;
  r->pitch = r->cols;
  bool first = true;
  for (int64_t i = d - 2; i >= 0; --i) {
    if (size[i] == 0) return false;
    if (size[i] == 1) continue;
    if (first) r->pitch = stride[i], first = false;
    else if (stride[i] != r->pitch * r->rows) return false;
    r->rows *= size[i];
  }
  return true;
}

bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }
int64_t up16(int64_t n) { return (n + 15) & ~int64_t(15); }

// codes as the products read them: rows at multiples of 16 bytes
bool code_rows(const at::Tensor& t, Rows* r) {
  if (t.scalar_type() != at::kChar || !rows_of(t, r) || !aligned16(t)) return false;
  if (r->rows == 1) r->pitch = up16(r->cols);
  return (r->pitch & 15) == 0 && r->pitch >= r->cols;
}

bool vector_of(const at::Tensor& t, at::ScalarType type, int64_t n) {
  return t.scalar_type() == type && t.numel() == n && t.is_contiguous();
}

at::DimVector with_last(const at::Tensor& t, int64_t last) {
  at::DimVector s(t.sizes());
  s.back() = last;
  return s;
}

// New memory on t's device, from torch's allocator without the way through its dispatcher (0.1 us of host time each).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& t) {
  return at::cuda::empty(sizes, type, c10::nullopt, t.device(), c10::nullopt, c10::nullopt);
}

// Room for the codes of a tensor like t, their scales and zero points
struct Codes {
  at::Tensor codes, scales, zeros;
  int64_t pitch;
  Codes(const at::Tensor& t, bool sym) {
    const int64_t cols = t.size(-1);
    pitch = up16(cols);
    codes = fresh(with_last(t, pitch), at::kChar, t);
    scales = fresh(with_last(t, 1), at::kFloat, t);
    if (!sym) zeros = fresh(with_last(t, 1), at::kInt, t);
  }
  int8_t* at_codes() const { return codes.data_ptr<int8_t>(); }
  float* at_scales() const { return scales.data_ptr<float>(); }
  int32_t* at_zeros() const { return zeros.defined() ? zeros.data_ptr<int32_t>() : nullptr; }
  PyObject* tuple(int64_t cols) const {
    PyObject* q = THPVariable_Wrap(pitch == cols ? codes : codes.narrow(-1, 0, cols));
    PyObject* s = THPVariable_Wrap(scales);
    if (!zeros.defined()) {
      PyObject* r = PyTuple_Pack(2, q, s);
      Py_XDECREF(q), Py_XDECREF(s);
      return r;
    }
    PyObject* z = THPVariable_Wrap(zeros);
    PyObject* r = PyTuple_Pack(3, q, s, z);
    Py_XDECREF(q), Py_XDECREF(s), Py_XDECREF(z);
    return r;
  }
};

PyObject* pair_of(PyObject* a, PyObject* b) {
  PyObject* r = PyTuple_Pack(2, a, b);
  Py_XDECREF(a), Py_XDECREF(b);
  return r;
}

// Other Python threads run meanwhile: an allocation may wait for the device, a launch for room in its queue, and what the
// device waits for may need the interpreter.  Nothing of Python's is touched while one of these lives.
class Unlocked {
  PyThreadState* const state_ = PyEval_SaveThread();

 public:
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state_); }
};

// The functions below return false for what the Python function has to deal with.

// (x, sym)
bool act_quant(PyObject* const* a, Py_ssize_t n, PyObject** out) {
  if (n != 2) return false;
  const at::Tensor* x = tensor_of(a[0]);
  Place place;
  Rows r;
  lc_stream_t st;
  if (!x || !place.take(*x) || dtype_of(*x) < 0 || !rows_of(*x, &r)) return false;
  const bool sym = a[1] == Py_True;
  if ((!sym && a[1] != Py_False) || !place.enter(&st)) return false;
  c10::optional<Codes> c;
  {
    const Unlocked unlocked;
    c.emplace(*x, sym);
    if (lc_int8_act_quant(x->data_ptr(), (int)dtype_of(*x), r.rows, r.cols, r.pitch, c->at_codes(), c->pitch, c->at_scales(),
                          c->at_zeros(), st) != LC_OK)
      return false;
  }
  *out = c->tuple(r.cols);
  return true;
}

// (gate, up, activation's number, sym)
bool gated_act_quant(PyObject* const* a, Py_ssize_t n, PyObject** out) {
  if (n != 4) return false;
  const at::Tensor *g = tensor_of(a[0]), *u = tensor_of(a[1]);
  Place place;
  Rows rg, ru;
  lc_stream_t st;
  if (!g || !u || !place.take(*g) || !place.take(*u) || dtype_of(*g) < 0 || u->scalar_type() != g->scalar_type() ||
      g->sizes() != u->sizes() || !rows_of(*g, &rg) || !rows_of(*u, &ru))
    return false;
  const long act = PyLong_AsLong(a[2]);
  const bool sym = a[3] == Py_True;
  if ((!sym && a[3] != Py_False) || !place.enter(&st)) return false;
  c10::optional<Codes> c;
  {
    const Unlocked unlocked;
    c.emplace(*g, sym);
    if (lc_int8_gated_act_quant(g->data_ptr(), u->data_ptr(), (int)dtype_of(*g), rg.rows, rg.cols, rg.pitch, ru.pitch, (int)act,
                                c->at_codes(), c->pitch, c->at_scales(), c->at_zeros(), st) != LC_OK)
      return false;
  }
  *out = c->tuple(rg.cols);
  return true;
}

// the weight's side of a product
struct Weight {
  const at::Tensor *b, *scale, *sum = nullptr, *bias = nullptr;
  Rows r;
  bool take(PyObject* ob, PyObject* oscale, PyObject* obias, PyObject* osum, at::ScalarType type, Place* place) {
    b = tensor_of(ob), scale = tensor_of(oscale);
    if (!b || !scale || !place->take(*b) || !place->take(*scale) || b->dim() != 2 || !code_rows(*b, &r)) return false;
    if (!vector_of(*scale, at::kFloat, r.rows) || r.cols > (osum == Py_None ? 131071 : 65793)) return false;
    if (obias != Py_None && (!(bias = tensor_of(obias)) || !place->take(*bias) || !vector_of(*bias, type, r.rows))) return false;
    if (osum != Py_None && (!(sum = tensor_of(osum)) || !place->take(*sum) || !vector_of(*sum, at::kInt, r.rows))) return false;
    return true;
  }
  const int32_t* at_sum() const { return sum ? sum->data_ptr<int32_t>() : nullptr; }
  const void* at_bias() const { return bias ? bias->data_ptr() : nullptr; }
};

// (a, a_s, b, b_s, bias, a_z, b_sum, out_dtype)
bool int8_gemm(PyObject* const* o, Py_ssize_t n, PyObject** out) {
  if (n != 8 || !THPDtype_Check(o[7])) return false;
  const at::Tensor *a = tensor_of(o[0]), *a_s = tensor_of(o[1]), *a_z = o[5] == Py_None ? nullptr : tensor_of(o[5]);
  const at::ScalarType type = reinterpret_cast<THPDtype*>(o[7])->scalar_type;
  Place place;
  Rows r;
  Weight w;
  lc_stream_t st;
  if (!a || !a_s || (o[5] != Py_None && (!a_z || o[6] == Py_None))) return false;
  if (!place.take(*a) || !place.take(*a_s) || (a_z && !place.take(*a_z)) || !code_rows(*a, &r)) return false;
  if (!w.take(o[2], o[3], o[4], a_z ? o[6] : Py_None, type, &place) || r.cols != w.r.cols) return false;
  if (!vector_of(*a_s, at::kFloat, r.rows) || (a_z && !vector_of(*a_z, at::kInt, r.rows)) || !place.enter(&st)) return false;
  if (!g_status[place.device]) return false;
  if (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf) return false;
  at::Tensor c;
  {
    const Unlocked unlocked;
    c = fresh(with_last(*a, w.r.rows), type, *a);
    const int64_t dt = dtype_of(c);
    const lc_int8_gemm_args args = {a->data_ptr<int8_t>(), r.pitch, a_s->data_ptr<float>(), a_z ? a_z->data_ptr<int32_t>() : nullptr,
                                    w.b->data_ptr<int8_t>(), w.r.pitch, w.scale->data_ptr<float>(), w.at_sum(), w.at_bias(),
                                    r.rows, w.r.rows, r.cols, c.data_ptr(), dt, g_status[place.device]};
    if (lc_int8_gemm(&args, st) != LC_OK) return false;
  }
  *out = THPVariable_Wrap(c);
  return true;
}

// (x, w, w_scale, bias, w_sum)
bool int8_linear(PyObject* const* o, Py_ssize_t n, PyObject** out) {
  if (n != 5) return false;
  const at::Tensor* x = tensor_of(o[0]);
  Place place;
  Rows r;
  Weight w;
  lc_stream_t st;
  if (!x || !place.take(*x) || dtype_of(*x) < 0 || !rows_of(*x, &r)) return false;
  if (!w.take(o[1], o[2], o[3], o[4], x->scalar_type(), &place) || r.cols != w.r.cols || !place.enter(&st)) return false;
  if (!g_status[place.device]) return false;
  at::Tensor c;
  {
    const Unlocked unlocked;
    c = fresh(with_last(*x, w.r.rows), x->scalar_type(), *x);
    const int64_t room = lc_int8_linear_scratch(r.rows, r.cols);
    const at::Tensor scratch = room ? fresh({room}, at::kChar, *x) : at::Tensor();
    const lc_int8_linear_args args = {x->data_ptr(), dtype_of(*x), r.pitch, w.b->data_ptr<int8_t>(), w.r.pitch,
                                      w.scale->data_ptr<float>(), w.at_sum(), w.at_bias(), r.rows, w.r.rows, r.cols, w.sum == nullptr,
                                      c.data_ptr(), room ? scratch.data_ptr() : nullptr, room, g_status[place.device]};
    if (lc_int8_linear(&args, st) != LC_OK) return false;
  }
  *out = THPVariable_Wrap(c);
  return true;
}

// How many rows of gate there are, as block_ops._gate_rows has it; 0 where it does not go with x.
int64_t gate_rows_of(const at::Tensor& gate, const at::Tensor& x) {
  const int64_t lead = x.dim() - 1, g = gate.dim() - 1;
  if (g < 0 || g > lead || gate.size(-1) != x.size(-1)) return 0;
  auto size = [&](int64_t i) { return i < lead - g ? 1 : gate.size(i - (lead - g)); };
  int64_t i = 0, rows = 1;
  while (i < lead && size(i) == x.size(i)) rows *= size(i++);
  for (; i < lead; ++i)
    if (size(i) != 1) return 0;
  return rows;
}

// (x, residual, weight, post_weight, gate, scale, eps, weight_offset, quant, sym)
bool residual_norm(PyObject* const* o, Py_ssize_t n, PyObject** out) {
  if (n != 10) return false;
  const at::Tensor *x = tensor_of(o[0]), *t[5] = {x};
  Place place;
  lc_stream_t st;
  if (!x || !place.take(*x)) return false;                 // x is compared with below: it may not be left out
  for (int i = 1; i < 5; ++i) {
    t[i] = o[i] == Py_None ? nullptr : tensor_of(o[i]);
    if (o[i] != Py_None && (!t[i] || !place.take(*t[i]) || t[i]->scalar_type() != x->scalar_type())) return false;
  }
  const at::Tensor *res = t[1], *w = t[2], *pw = t[3], *gate = t[4];
  Rows rx, rr;
  if (dtype_of(*x) < 0 || !rows_of(*x, &rx)) return false;
  if (res && (res->sizes() != x->sizes() || !rows_of(*res, &rr))) return false;
  for (const at::Tensor* v : {w, pw})
    if (v && (v->dim() != 1 || !vector_of(*v, x->scalar_type(), rx.cols))) return false;
  int64_t gate_rows = 0;
  if (gate && (!gate->is_contiguous() || (gate_rows = gate_rows_of(*gate, *x)) == 0)) return false;
  for (int i = 5; i < 8; ++i)
    if (!PyFloat_CheckExact(o[i]) && !PyLong_CheckExact(o[i])) return false;
  const double scale = PyFloat_AsDouble(o[5]), eps = PyFloat_AsDouble(o[6]), offset = PyFloat_AsDouble(o[7]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  const bool quant = o[8] == Py_True, sym = o[9] == Py_True, kept = !res && !pw && !gate && scale == 1.0;
  if ((!quant && o[8] != Py_False) || (!sym && o[9] != Py_False) || (!w && (quant || kept)) || !place.enter(&st)) return false;
  at::Tensor h, y;
  c10::optional<Codes> c;
  {
    const Unlocked unlocked;
    if (!kept) h = fresh(x->sizes(), x->scalar_type(), *x);
    if (w && !quant) y = fresh(x->sizes(), x->scalar_type(), *x);
    if (quant) c.emplace(*x, sym);
    const lc_residual_norm_args args = {x->data_ptr(), res ? res->data_ptr() : nullptr, pw ? pw->data_ptr() : nullptr,
                                        gate ? gate->data_ptr() : nullptr, gate_rows, w ? w->data_ptr() : nullptr, dtype_of(*x),
                                        rx.rows, rx.cols, rx.pitch, rr.pitch, scale, eps, offset, kept ? nullptr : h.data_ptr(),
                                        y.defined() ? y.data_ptr() : nullptr, c ? c->at_codes() : nullptr, c ? c->pitch : 0,
                                        c ? c->at_scales() : nullptr, c ? c->at_zeros() : nullptr};
    if (lc_residual_norm(&args, st) != LC_OK) return false;
  }
  PyObject* first = kept ? (Py_INCREF(o[0]), o[0]) : THPVariable_Wrap(h);
  PyObject* second = quant ? c->tuple(rx.cols) : y.defined() ? THPVariable_Wrap(y) : (Py_INCREF(Py_None), Py_None);
  *out = pair_of(first, second);
  return true;
}

// (q, k, positions, inv_freq, interleaved, attention_scale)
bool rotary_embed(PyObject* const* o, Py_ssize_t n, PyObject** out) {
  if (n != 6) return false;
  const at::Tensor *q = tensor_of(o[0]), *k = o[1] == Py_None ? nullptr : tensor_of(o[1]), *pos = tensor_of(o[2]),
                   *freq = tensor_of(o[3]);
  Place place;
  lc_stream_t st;
  if (!q || !pos || !freq || (o[1] != Py_None && !k) || !place.take(*q) || !place.take(*pos) || !place.take(*freq)) return false;
  if (dtype_of(*q) < 0 || q->dim() != 4 || q->numel() == 0) return false;
  const int64_t B = q->size(0), H = q->size(1), T = q->size(2), D = q->size(3), G = k && k->dim() == 4 ? k->size(1) : 0;
  if (k && (!place.take(*k) || k->dim() != 4 || k->scalar_type() != q->scalar_type() || k->size(0) != B || k->size(2) != T ||
            k->size(3) != D || G == 0))
    return false;
  const bool own_rows = pos->dim() == 2 && pos->size(0) == B && B > 1;
  if (pos->scalar_type() != at::kLong || !pos->is_contiguous() || pos->dim() < 1 || pos->dim() > 2 || pos->size(-1) != T ||
      (pos->dim() == 2 && pos->size(0) != 1 && pos->size(0) != B))
    return false;
  const int64_t half = freq->numel();
  if (freq->scalar_type() != at::kFloat || freq->dim() != 1 || !freq->is_contiguous() || half < 1 || 2 * half > D) return false;
  if (q->stride(3) != 1 || (k && k->stride(3) != 1) || D > 1024 || H + G > 1023) return false;
  const bool inter = o[4] == Py_True;
  if ((!inter && o[4] != Py_False) || !PyFloat_CheckExact(o[5]) || !place.enter(&st)) return false;
  auto like = [&](const at::Tensor& t) {
    const int64_t heads = t.size(1);
    return at::cuda::empty_strided(t.sizes(), {T * heads * D, D, heads * D, 1}, t.scalar_type(), c10::nullopt, t.device(), c10::nullopt);
  };
  at::Tensor qo, ko;
  const double scale = PyFloat_AS_DOUBLE(o[5]);
  {
    const Unlocked unlocked;
    qo = like(*q);
    if (k) ko = like(*k);
    const lc_rotary_embed_args args = {q->data_ptr(), qo.data_ptr(), H, q->stride(0), q->stride(2), q->stride(1),
                                       k ? k->data_ptr() : nullptr, k ? ko.data_ptr() : nullptr, G, k ? k->stride(0) : 0,
                                       k ? k->stride(2) : 0, k ? k->stride(1) : 0, pos->data_ptr<int64_t>(), own_rows ? T : 0,
                                       freq->data_ptr<float>(), dtype_of(*q), B, T, D, 2 * half, inter, scale};
    if (lc_rotary_embed(&args, st) != LC_OK) return false;
  }
  *out = pair_of(THPVariable_Wrap(qo), k ? THPVariable_Wrap(ko) : (Py_INCREF(Py_None), Py_None));
  return true;
}

// No C++ exception (an allocation that fails, say) passes into the interpreter: the Python function runs into it again and
// raises it in its own manner.
template <bool (*F)(PyObject* const*, Py_ssize_t, PyObject**)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  PyObject* out = nullptr;
  try {
    if (F(args, n, &out)) return out;
  } catch (...) {
  }
  if (PyErr_Occurred()) PyErr_Clear();
  Py_RETURN_NONE;
}

// (device, address): the status word of a device's products
PyObject* set_status(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) return PyErr_Format(PyExc_TypeError, "set_status takes a device and an address");
  const long device = PyLong_AsLong(args[0]);
  void* p = PyLong_AsVoidPtr(args[1]);
  if (PyErr_Occurred()) return nullptr;
  if (device >= 0 && device < 64) g_status[device] = static_cast<int32_t*>(p);
  Py_RETURN_NONE;
}

#define LC_ENTRY(name) {#name, (PyCFunction)(void*)entry<name>, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {LC_ENTRY(act_quant),
                           LC_ENTRY(gated_act_quant),
                           LC_ENTRY(int8_gemm),
                           LC_ENTRY(int8_linear),
                           LC_ENTRY(residual_norm),
                           LC_ENTRY(rotary_embed),
                           {"set_status", (PyCFunction)(void*)set_status, METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_calls", "Compiled front of the W8A8 operators", -1, g_methods};

}  // namespace

// built_for: the torch and the interpreter whose binary interfaces are compiled in, to be compared before anything is called
PyMODINIT_FUNC PyInit__calls() {
  PyObject* m = PyModule_Create(&g_module);
  if (m && PyModule_AddStringConstant(m, "built_for", LC_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
