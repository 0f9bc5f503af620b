// Host path of the voxel-sequence operators (ops/sequence.py): arguments checked, outputs and workspace taken from torch's
// allocator, the C-ABI function called on the current stream of the features' device.  The same steps in Python take 13 to
// 18 us, several times what the kernels of a small call do; here they take 3 to 5 with the launch.
//
// Every function takes its arguments by position, None for one that is left out; ops/sequence.py documents them.
#include "host.h"

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>

namespace {

decltype(&d3d_layer_norm) f_layer_norm;
decltype(&d3d_layer_norm_int8) f_layer_norm_int8;
decltype(&d3d_layer_norm_backward) f_layer_norm_backward;
decltype(&d3d_layer_norm_backward_workspace) f_layer_norm_backward_workspace;
decltype(&d3d_quantize_rows) f_quantize_rows;
decltype(&d3d_int8_linear) f_int8_linear;
decltype(&d3d_int8_linear_workspace) f_int8_linear_workspace;
decltype(&d3d_gated_recurrence) f_gated_recurrence;
decltype(&d3d_gated_recurrence_backward) f_gated_recurrence_backward;
decltype(&d3d_gated_recurrence_step) f_gated_recurrence_step;
decltype(&d3d_gated_recurrence_state_rows) f_gated_recurrence_state_rows;
decltype(&d3d_gated_recurrence_workspace) f_gated_recurrence_workspace;

// A Python exception is set.
struct Refused {};

[[noreturn]] void refuse(PyObject* type, const char* format, const char* a = "", const char* b = "") {
  PyErr_Format(type, format, a, b);
  throw Refused();
}

// A matrix argument: rows side by side in memory, `ld` elements apart.
struct Rows {
  at::Tensor t;
  int64_t rows = 0, channels = 0, ld = 0;
  const void* p() const { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
};

Rows matrix(PyObject* o, const char* what, int64_t single_ld_unit) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s: a tensor is needed", what);
  Rows r;
  r.t = THPVariable_Unpack(o);
  if (r.t.dim() != 2 || !r.t.is_cuda())
    refuse(PyExc_ValueError, "%s: a CUDA tensor [rows, channels] is needed; this library has no CPU path", what);
  r.rows = r.t.size(0), r.channels = r.t.size(1);
  if (r.channels == 0) refuse(PyExc_ValueError, "%s: no channels", what);
  if (r.channels > INT32_MAX) refuse(PyExc_ValueError, "%s: too many channels", what);
  // nothing lies behind a single row
  r.ld = r.rows > 1 ? r.t.stride(0) : (r.channels + single_ld_unit - 1) / single_ld_unit * single_ld_unit;
  if ((r.channels > 1 && r.t.stride(1) != 1) || r.ld < r.channels) r.t = r.t.contiguous(), r.ld = r.channels;
  return r;
}

// Features: float, half or bfloat16; where `like` is given of its shape, type and device.
Rows features(PyObject* o, const char* what, const Rows* like = nullptr) {
  Rows r = matrix(o, what, 1);
  const at::ScalarType s = r.t.scalar_type();
  if (s != at::kFloat && s != at::kHalf && s != at::kBFloat16)
    refuse(PyExc_TypeError, "%s: unsupported tensor dtype %s", what, c10::toString(s));
  if (like && (r.rows != like->rows || r.channels != like->channels || s != like->t.scalar_type() || r.t.device() != like->t.device()))
    refuse(PyExc_ValueError, "%s: shape, dtype and device of the features are needed", what);
  return r;
}
Rows maybe_features(PyObject* o, const char* what, const Rows& like) { return o == Py_None ? Rows() : features(o, what, &like); }

// A dense tensor of this shape and type on the device; its address.
void* dense_tensor(PyObject* o, const char* what, std::initializer_list<int64_t> shape, at::ScalarType type, c10::Device device) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s: a tensor is needed", what);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.sizes() != at::IntArrayRef(shape) || t.scalar_type() != type || t.device() != device || !t.is_contiguous())
    refuse(PyExc_ValueError, "%s: a dense %s tensor of the right shape, on the device of the features, is needed", what,
           c10::toString(type));
  return t.numel() ? t.data_ptr() : nullptr;
}
float* floats(PyObject* o, const char* what, std::initializer_list<int64_t> shape, c10::Device device) {
  return static_cast<float*>(dense_tensor(o, what, shape, at::kFloat, device));
}
float* maybe_floats(PyObject* o, const char* what, std::initializer_list<int64_t> shape, c10::Device device) {
  return o == Py_None ? nullptr : floats(o, what, shape, device);
}
const int32_t* count_of(PyObject* o, c10::Device device) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s: a tensor is needed", "num_rows");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != at::kInt || t.numel() != 1 || t.device() != device)
    refuse(PyExc_ValueError, "num_rows: an int32 tensor of one element on the device of the features is needed");
  return static_cast<const int32_t*>(t.data_ptr());
}

at::Tensor made(std::initializer_list<int64_t> shape, at::ScalarType type, c10::Device device) {
  return at::empty(at::IntArrayRef(shape), at::TensorOptions().dtype(type).device(device));
}
// `out` where given, else a new tensor.
at::Tensor output(PyObject* o, std::initializer_list<int64_t> shape, at::ScalarType type, c10::Device device) {
  if (o == Py_None) return made(shape, type, device);
  dense_tensor(o, "out", shape, type, device);
  return THPVariable_Unpack(o);
}
// `out`, where it was given, has other contents now: autograd refuses to go back through what it has kept of the old ones.
void wrote(PyObject* o, const at::Tensor& out) {
  if (o != Py_None && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}
void* at_of(const at::Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
float* floats_of(const at::Tensor& t) { return static_cast<float*>(at_of(t)); }

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) throw Refused();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused();
  return v != 0;
}

// Calls `fn` without the interpreter's lock, on the device and its current stream; raises for any status but 0.
template <class F> void launch(const char* name, c10::Device device, F fn) {
  c10::cuda::CUDAGuard guard(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = fn(stream);
  Py_END_ALLOW_THREADS;
  if (status == D3D_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "si", name, status);
  Py_XDECREF(r);
  if (r) PyErr_Format(PyExc_RuntimeError, "%s failed", name);
  throw Refused();
}

PyObject* tuple_of(std::initializer_list<at::Tensor> list) {
  Py_ssize_t n = 0;
  for (const at::Tensor& t : list) n += t.defined();
  PyObject* r = PyTuple_New(n);
  if (!r) throw Refused();
  n = 0;
  for (const at::Tensor& t : list)
    if (t.defined()) PyTuple_SET_ITEM(r, n++, THPVariable_Wrap(t));
  return r;
}

void want(Py_ssize_t given, Py_ssize_t n) {
  if (given != n) refuse(PyExc_TypeError, "wrong number of arguments");
}

using Args = PyObject* const*;

// feats, weight, bias, eps, residual, num_rows, with_stats, out
PyObject* layer_norm(Args a, Py_ssize_t n) {
  want(n, 8);
  const Rows x = features(a[0], "feats"), r = maybe_features(a[4], "residual", x);
  const c10::Device device = x.t.device();
  const at::ScalarType type = x.t.scalar_type();
  const float* weight = maybe_floats(a[1], "weight", {x.channels}, device);
  const float* bias = maybe_floats(a[2], "bias", {x.channels}, device);
  const int32_t* count = count_of(a[5], device);
  at::Tensor out = output(a[7], {x.rows, x.channels}, type, device), total, mean, rstd;
  if (r.t.defined()) total = made({x.rows, x.channels}, type, device);
  if (truth(a[6])) mean = made({x.rows}, at::kFloat, device), rstd = made({x.rows}, at::kFloat, device);
  const float eps = (float)number(a[3]);
  launch("d3d_layer_norm", device, [&](void* stream) {
    return f_layer_norm(dtype_of(x.t), x.p(), x.ld, r.p(), r.ld, weight, bias, eps, x.rows, (int)x.channels, count, at_of(total),
                        at_of(out), floats_of(mean), floats_of(rstd), stream);
  });
  wrote(a[7], out);
  if (!total.defined() && !mean.defined()) return THPVariable_Wrap(out);
  return tuple_of({out, total, mean, rstd});
}

// grad_out, feats, weight, mean, rstd, num_rows, grad_total
PyObject* layer_norm_backward(Args a, Py_ssize_t n) {
  want(n, 7);
  const Rows x = features(a[1], "feats"), g = features(a[0], "grad_out", &x), t = maybe_features(a[6], "grad_total", x);
  const c10::Device device = x.t.device();
  const float* weight = maybe_floats(a[2], "weight", {x.channels}, device);
  const float *mean = floats(a[3], "mean", {x.rows}, device), *rstd = floats(a[4], "rstd", {x.rows}, device);
  const int32_t* count = count_of(a[5], device);
  at::Tensor dx = made({x.rows, x.channels}, x.t.scalar_type(), device);
  at::Tensor dw = made({x.channels}, at::kFloat, device), db = made({x.channels}, at::kFloat, device);
  const size_t bytes = f_layer_norm_backward_workspace(x.rows, (int)x.channels);
  at::Tensor ws = made({(int64_t)bytes}, at::kByte, device);
  launch("d3d_layer_norm_backward", device, [&](void* stream) {
    return f_layer_norm_backward(dtype_of(x.t), g.p(), g.ld, x.p(), x.ld, t.p(), t.ld, weight, mean, rstd, x.rows, (int)x.channels,
                                 count, at_of(dx), floats_of(dw), floats_of(db), at_of(ws), bytes, stream);
  });
  return tuple_of({dx, dw, db});
}

// 8-bit rows a multiple of 16 bytes apart.
at::Tensor int8_rows(int64_t rows, int64_t channels, int64_t* pitch, c10::Device device) {
  *pitch = (channels + 15) / 16 * 16;
  at::Tensor q = made({rows, *pitch}, at::kChar, device);
  return *pitch == channels ? q : q.narrow(1, 0, channels);
}

// feats, weight, bias, eps, residual, num_rows
PyObject* layer_norm_int8(Args a, Py_ssize_t n) {
  want(n, 6);
  const Rows x = features(a[0], "feats"), r = maybe_features(a[4], "residual", x);
  const c10::Device device = x.t.device();
  const float* weight = maybe_floats(a[1], "weight", {x.channels}, device);
  const float* bias = maybe_floats(a[2], "bias", {x.channels}, device);
  const int32_t* count = count_of(a[5], device);
  int64_t pitch;
  at::Tensor q = int8_rows(x.rows, x.channels, &pitch, device), scales = made({x.rows}, at::kFloat, device), total;
  if (r.t.defined()) total = made({x.rows, x.channels}, x.t.scalar_type(), device);
  const float eps = (float)number(a[3]);
  launch("d3d_layer_norm_int8", device, [&](void* stream) {
    return f_layer_norm_int8(dtype_of(x.t), x.p(), x.ld, r.p(), r.ld, weight, bias, eps, x.rows, (int)x.channels, count, at_of(total),
                             static_cast<int8_t*>(at_of(q)), pitch, floats_of(scales), stream);
  });
  return tuple_of({q, scales, total});
}

// feats, num_rows
PyObject* quantize_rows(Args a, Py_ssize_t n) {
  want(n, 2);
  const Rows x = features(a[0], "feats");
  const c10::Device device = x.t.device();
  const int32_t* count = count_of(a[1], device);
  int64_t pitch;
  at::Tensor q = int8_rows(x.rows, x.channels, &pitch, device), scales = made({x.rows}, at::kFloat, device);
  launch("d3d_quantize_rows", device, [&](void* stream) {
    return f_quantize_rows(dtype_of(x.t), x.p(), x.ld, x.rows, (int)x.channels, count, static_cast<int8_t*>(at_of(q)), pitch,
                           floats_of(scales), stream);
  });
  return tuple_of({q, scales});
}

Rows bytes_of(PyObject* o, const char* what) {
  Rows r = matrix(o, what, 16);
  if (r.t.scalar_type() != at::kChar) refuse(PyExc_TypeError, "%s: an int8 tensor is needed", what);
  return r;
}

// feats, scales, weight, weight_scales, bias, dtype, num_rows, out
PyObject* int8_linear(Args a, Py_ssize_t n) {
  want(n, 8);
  const Rows x = bytes_of(a[0], "feats"), w = bytes_of(a[2], "weight");
  const c10::Device device = x.t.device();
  if (w.channels != x.channels || w.t.device() != device || w.rows == 0 || w.rows > INT32_MAX)
    refuse(PyExc_ValueError, "weight: [outputs, inputs] on the device of the features is needed");
  if (!THPDtype_Check(a[5])) refuse(PyExc_TypeError, "dtype: a torch.dtype is needed");
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  if (type != at::kFloat && type != at::kHalf && type != at::kBFloat16)
    refuse(PyExc_TypeError, "%s: unsupported tensor dtype %s", "dtype", c10::toString(type));
  const float *scales = floats(a[1], "scales", {x.rows}, device), *w_scales = floats(a[3], "weight_scales", {w.rows}, device);
  const float* bias = maybe_floats(a[4], "bias", {w.rows}, device);
  const int32_t* count = count_of(a[6], device);
  at::Tensor out = output(a[7], {x.rows, w.rows}, type, device), ws;
  const int8_t *px = static_cast<const int8_t*>(x.p()), *pw = static_cast<const int8_t*>(w.p());
  const size_t bytes = f_int8_linear_workspace(px, x.ld, x.rows, pw, w.ld, (int)x.channels, (int)w.rows);
  if (bytes) ws = made({(int64_t)bytes}, at::kByte, device);
  launch("d3d_int8_linear", device, [&](void* stream) {
    return f_int8_linear(dtype_of(out), px, x.ld, scales, x.rows, count, pw, w.ld, w_scales, bias, (int)x.channels, (int)w.rows,
                         at_of(out), at_of(ws), bytes, stream);
  });
  wrote(a[7], out);
  return THPVariable_Wrap(out);
}

struct Sequences {
  at::Tensor t;
  int count;
};
Sequences sequences(PyObject* o, c10::Device device) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s: a tensor is needed", "seq_offsets");
  at::Tensor t = THPVariable_Unpack(o);
  if (t.dim() != 1 || t.size(0) < 1 || t.size(0) > INT32_MAX || t.scalar_type() != at::kInt || t.device() != device)
    refuse(PyExc_ValueError, "seq_offsets: an int32 tensor [sequences + 1] on the device of the features is needed");
  if (!t.is_contiguous()) t = t.contiguous();
  return {t, (int)t.size(0) - 1};
}

// feats, gates, seq_offsets, initial, reverse, with_states, out
PyObject* gated_recurrence(Args a, Py_ssize_t n) {
  want(n, 7);
  const Rows x = features(a[0], "feats"), g = features(a[1], "gates", &x);
  const c10::Device device = x.t.device();
  const Sequences s = sequences(a[2], device);
  const float* initial = maybe_floats(a[3], "initial", {s.count, x.channels}, device);
  const int reverse = truth(a[4]);
  at::Tensor out = output(a[6], {x.rows, x.channels}, x.t.scalar_type(), device);
  at::Tensor final_state = made({s.count, x.channels}, at::kFloat, device), states;
  if (truth(a[5])) states = made({f_gated_recurrence_state_rows(x.rows), x.channels}, at::kFloat, device);
  const size_t bytes = f_gated_recurrence_workspace(x.rows, (int)x.channels);
  at::Tensor ws;
  if (bytes) ws = made({(int64_t)bytes}, at::kByte, device);
  launch("d3d_gated_recurrence", device, [&](void* stream) {
    return f_gated_recurrence(dtype_of(x.t), x.p(), x.ld, g.p(), g.ld, static_cast<const int32_t*>(s.t.data_ptr()), s.count, x.rows,
                              (int)x.channels, reverse, initial, at_of(out), floats_of(final_state), floats_of(states), at_of(ws),
                              bytes, stream);
  });
  wrote(a[6], out);
  return tuple_of({out, final_state, states});
}

// grad_out, feats, gates, seq_offsets, states, initial, grad_final, reverse
PyObject* gated_recurrence_backward(Args a, Py_ssize_t n) {
  want(n, 8);
  const Rows x = features(a[1], "feats"), g = features(a[2], "gates", &x), d = features(a[0], "grad_out", &x);
  const c10::Device device = x.t.device();
  const at::ScalarType type = x.t.scalar_type();
  const Sequences s = sequences(a[3], device);
  const float* states = floats(a[4], "states", {f_gated_recurrence_state_rows(x.rows), x.channels}, device);
  const float* initial = maybe_floats(a[5], "initial", {s.count, x.channels}, device);
  const float* grad_final = maybe_floats(a[6], "grad_final", {s.count, x.channels}, device);
  const int reverse = truth(a[7]);
  at::Tensor dx = made({x.rows, x.channels}, type, device), dg = made({x.rows, x.channels}, type, device);
  at::Tensor di = made({s.count, x.channels}, at::kFloat, device);
  const size_t bytes = f_gated_recurrence_workspace(x.rows, (int)x.channels);
  at::Tensor ws;
  if (bytes) ws = made({(int64_t)bytes}, at::kByte, device);
  launch("d3d_gated_recurrence_backward", device, [&](void* stream) {
    return f_gated_recurrence_backward(dtype_of(x.t), d.p(), d.ld, x.p(), x.ld, g.p(), g.ld,
                                       static_cast<const int32_t*>(s.t.data_ptr()), s.count, x.rows, (int)x.channels, reverse, states,
                                       initial, grad_final, at_of(dx), at_of(dg), floats_of(di), at_of(ws), bytes, stream);
  });
  return tuple_of({dx, dg, di});
}

// feats, gates, state, state_out
PyObject* gated_recurrence_step(Args a, Py_ssize_t n) {
  want(n, 4);
  const Rows x = features(a[0], "feats"), g = features(a[1], "gates", &x);
  const c10::Device device = x.t.device();
  const float* state = floats(a[2], "state", {x.rows, x.channels}, device);
  at::Tensor next = output(a[3], {x.rows, x.channels}, at::kFloat, device);
  at::Tensor out = made({x.rows, x.channels}, x.t.scalar_type(), device);
  launch("d3d_gated_recurrence_step", device, [&](void* stream) {
    return f_gated_recurrence_step(dtype_of(x.t), x.p(), x.ld, g.p(), g.ld, state, floats_of(next), at_of(out), x.rows,
                                   (int)x.channels, stream);
  });
  wrote(a[3], next);
  return tuple_of({out, next});
}

template <PyObject* (*kFn)(Args, Py_ssize_t)> PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    return kFn(args, n);
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind_sequence(addresses): the library's entry points, in the order of `targets`.
PyObject* bind(PyObject*, PyObject* list) {
  void** targets[] = {
      reinterpret_cast<void**>(&f_layer_norm), reinterpret_cast<void**>(&f_layer_norm_int8),
      reinterpret_cast<void**>(&f_layer_norm_backward), reinterpret_cast<void**>(&f_layer_norm_backward_workspace),
      reinterpret_cast<void**>(&f_quantize_rows), reinterpret_cast<void**>(&f_int8_linear),
      reinterpret_cast<void**>(&f_int8_linear_workspace), reinterpret_cast<void**>(&f_gated_recurrence),
      reinterpret_cast<void**>(&f_gated_recurrence_backward), reinterpret_cast<void**>(&f_gated_recurrence_step),
      reinterpret_cast<void**>(&f_gated_recurrence_state_rows), reinterpret_cast<void**>(&f_gated_recurrence_workspace)};
  constexpr Py_ssize_t kTargets = sizeof(targets) / sizeof(targets[0]);
  if (!PyTuple_Check(list) || PyTuple_GET_SIZE(list) != kTargets) {
    PyErr_SetString(PyExc_TypeError, "bind_sequence takes a tuple of addresses");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < kTargets; ++i) {
    void* p = PyLong_AsVoidPtr(PyTuple_GET_ITEM(list, i));
    if (!p) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address is null");
      return nullptr;
    }
    *targets[i] = p;
  }
  Py_RETURN_NONE;
}

template <PyObject* (*kFn)(Args, Py_ssize_t)> PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<kFn>)), METH_FASTCALL, nullptr};
}

}  // namespace

PyMethodDef sequence_methods[] = {
    method<layer_norm>("layer_norm"), method<layer_norm_backward>("layer_norm_backward"), method<layer_norm_int8>("layer_norm_int8"),
    method<quantize_rows>("quantize_rows"), method<int8_linear>("int8_linear"), method<gated_recurrence>("gated_recurrence"),
    method<gated_recurrence_backward>("gated_recurrence_backward"), method<gated_recurrence_step>("gated_recurrence_step"),
    {"bind_sequence", bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
