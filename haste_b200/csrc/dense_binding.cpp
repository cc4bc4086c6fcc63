// The Python side of layer norm, AdamW, gradient norm and the decoding of moments: tensors are looked at, outputs and workspaces are allocated and the
// library is called without a line of Python in between.  A call over a hundred tensors spends its time asking each of them for address, type, size and
// contiguity: 0.28 us a tensor from Python, a tenth of that here (norm of 99 gradients 41 us a call from Python, 25 so, which is the kernels' time; AdamW over 150 small
// tensors with 8-bit moments 130 and 19; layer norm of one row 9.1 and 4.6).
//
// The library itself (libhaste_ffi.so) knows neither torch nor Python; the addresses of its functions are handed to bind().
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/haste_ffi.h"

namespace {

struct Library {
  decltype(&haste_last_error_string) last_error;
  decltype(&haste_layer_norm_forward) layer_norm_forward;
  decltype(&haste_layer_norm_backward_scratch) layer_norm_backward_scratch;
  decltype(&haste_layer_norm_backward) layer_norm_backward;
  decltype(&haste_adamw_step) adamw_step;
  decltype(&haste_grad_norm) grad_norm;
  decltype(&haste_dequantize_moment) dequantize_moment;
} lib;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
[[noreturn]] void refuse(const std::string& why) { throw Refused(why); }

std::string text(at::IntArrayRef sizes) {
  std::string s = "(";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + (sizes.size() == 1 ? ",)" : ")");
}
std::string text(at::ScalarType t) { return std::string("torch.") + (t == at::kHalf ? "float16" : t == at::kDouble ? "float64" : c10::toString(t)); }

// Element type as the library counts them, -1 for any other
int code_of(at::ScalarType t) { return t == at::kBFloat16 ? HASTE_BF16 : t == at::kFloat ? HASTE_F32 : -1; }
int type_of(const at::Tensor& t, const char* name) {
  const int code = code_of(t.scalar_type());
  if (code < 0) refuse(std::string(name) + " must be torch.bfloat16 or torch.float32, got " + text(t.scalar_type()));
  return code;
}
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
// On no device that this library runs on: -1
int gpu_of(const at::Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }
// (half a microsecond less than through the dispatcher; every output is written in full)
at::Tensor empty_on(int dev, at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)), std::nullopt);
}
// A tensor that was written by address: a graph that holds its old values is to be refused (inference tensors are in none)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void* address(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// f(stream) with device `dev` current, and without the interpreter's lock (a launch may have to wait for room in the stream)
template <class F>
void run(int dev, const char* what, F&& f) {
  const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)));
  const auto stream = static_cast<haste_stream_t>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream());
  int rc;
  std::string why;
  Py_BEGIN_ALLOW_THREADS
  rc = f(stream);
  if (rc != 0) why = lib.last_error();
  Py_END_ALLOW_THREADS
  if (rc != 0) refuse(std::string(what) + ": haste status " + std::to_string(rc) + ": " + why);
}

// t [..., D] as rows of unit column stride, and their stride; copied only where no such view exists
std::pair<at::Tensor, int64_t> rows_of(const at::Tensor& t, int64_t D) {
  if (t.is_contiguous()) return {t, D};
  at::Tensor r = t.reshape({-1, D});
  if (D > 1 && r.stride(1) != 1) r = r.contiguous();
  return {r, r.size(0) > 1 ? r.stride(0) : D};
}

struct Rows {
  int dev, type;
  int64_t D;
};
Rows check_x(PyObject* o) {
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) refuse("x must be a CUDA tensor (this library has no CPU path)");
  const at::Tensor& x = THPVariable_Unpack(o);
  if (x.dim() < 1 || x.size(-1) < 1) refuse("x must be [..., D] with D >= 1, got " + text(x.sizes()));
  return {gpu_of(x), type_of(x, "x"), x.size(-1)};
}
int check_norm_parameter(const at::Tensor& t, const char* name, const Rows& x) {
  if (gpu_of(t) != x.dev) refuse(std::string(name) + " must be a CUDA tensor on cuda:" + std::to_string(x.dev) + ", as x is, got " + t.device().str());
  if (t.dim() != 1 || t.size(0) != x.D || !t.is_contiguous()) refuse(std::string(name) + " must be a contiguous [" + std::to_string(x.D) + "], got " + text(t.sizes()));
  return type_of(t, name);
}

// (x, weight, bias, eps, stats) -> (y, mean, rstd), or y
PyObject* layer_norm_forward(PyObject* const* a) {
  const Rows r = check_x(a[0]);
  const at::Tensor& x = THPVariable_Unpack(a[0]);
  const double eps = PyFloat_AsDouble(a[3]);
  const int stats = PyObject_IsTrue(a[4]);
  if (PyErr_Occurred()) throw python_error();
  int w_type = -1;
  const void *w = nullptr, *b = nullptr;
  if (a[1] != Py_None) {
    const at::Tensor& t = tensor(a[1], "weight");
    w_type = check_norm_parameter(t, "weight", r);
    w = t.data_ptr();
  }
  if (a[2] != Py_None) {
    const at::Tensor& t = tensor(a[2], "bias");
    const int type = check_norm_parameter(t, "bias", r);
    if (w_type >= 0 && type != w_type) refuse("weight and bias must have one type, got " + text(THPVariable_Unpack(a[1]).scalar_type()) + " and " + text(t.scalar_type()));
    w_type = type;
    b = t.data_ptr();
  }
  const auto [src, ldx] = rows_of(x, r.D);
  const int64_t rows = x.numel() / r.D, ld = ldx;
  at::Tensor y = empty_on(r.dev, x.sizes(), x.scalar_type()), mean, rstd;
  if (stats) {
    mean = empty_on(r.dev, x.sizes().slice(0, x.dim() - 1), at::kFloat);
    rstd = empty_on(r.dev, x.sizes().slice(0, x.dim() - 1), at::kFloat);
  }
  const void* xp = src.data_ptr();
  void* yp = y.data_ptr();
  float *mp = static_cast<float*>(address(mean)), *rp = static_cast<float*>(address(rstd));
  run(r.dev, "layer_norm_forward", [&](haste_stream_t st) {
    return lib.layer_norm_forward(xp, w, b, yp, mp, rp, rows, r.D, ld, static_cast<float>(eps), r.type, w_type < 0 ? 0 : w_type, st);
  });
  if (!stats) return THPVariable_Wrap(y);
  PyObject* out = PyTuple_New(3);
  if (out == nullptr) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(y));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(mean));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(rstd));
  return out;
}

// (dy, x, weight, mean, rstd, want_weight, want_bias, param_dtype) -> (dx, dweight, dbias)
PyObject* layer_norm_backward(PyObject* const* a) {
  const Rows r = check_x(a[1]);
  const at::Tensor& x = THPVariable_Unpack(a[1]);
  const int64_t rows = x.numel() / r.D;
  if (!THPVariable_Check(a[0]) || gpu_of(THPVariable_Unpack(a[0])) != r.dev || !THPVariable_Unpack(a[0]).sizes().equals(x.sizes()))
    refuse("dy must be a CUDA tensor of x's shape " + text(x.sizes()) + " on " + x.device().str());
  const at::Tensor& dy = THPVariable_Unpack(a[0]);
  const int dy_type = type_of(dy, "dy");
  const at::Tensor &mean = tensor(a[3], "mean"), &rstd = tensor(a[4], "rstd");
  for (const at::Tensor* t : {&mean, &rstd})
    if (gpu_of(*t) != r.dev || t->scalar_type() != at::kFloat || t->numel() != rows || !t->is_contiguous())
      refuse(std::string(t == &mean ? "mean" : "rstd") + " must be contiguous and hold " + std::to_string(rows) + " fp32 values on " + x.device().str());
  const int want_w = PyObject_IsTrue(a[5]), want_b = PyObject_IsTrue(a[6]);
  if (PyErr_Occurred()) throw python_error();
  at::ScalarType type = x.scalar_type();
  const void* w = nullptr;
  if (a[2] != Py_None) {
    const at::Tensor& t = tensor(a[2], "weight");
    check_norm_parameter(t, "weight", r);
    type = t.scalar_type();
    w = t.data_ptr();
  }
  if (a[7] != Py_None) {
    const bool fine = THPDtype_Check(a[7]) && (w == nullptr ? code_of(reinterpret_cast<THPDtype*>(a[7])->scalar_type) >= 0 : reinterpret_cast<THPDtype*>(a[7])->scalar_type == type);
    if (!fine) refuse("param_dtype must be the weight's type, torch.bfloat16 or torch.float32");
    type = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
  }
  const auto [src, ldx] = rows_of(x, r.D);
  const auto [grad, lddy] = rows_of(dy, r.D);
  const int64_t ld = ldx, ldg = lddy;
  at::Tensor dx = empty_on(r.dev, x.sizes(), x.scalar_type()), dw, db, scratch;
  if (want_w) dw = empty_on(r.dev, {r.D}, type);
  if (want_b) db = empty_on(r.dev, {r.D}, type);
  int64_t bytes = 0;
  if (want_w || want_b) {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    bytes = lib.layer_norm_backward_scratch(rows, r.D);
    scratch = empty_on(r.dev, {bytes}, at::kByte);
  }
  const void *gp = grad.data_ptr(), *xp = src.data_ptr();
  const float *mp = static_cast<const float*>(mean.data_ptr()), *rp = static_cast<const float*>(rstd.data_ptr());
  void *dxp = dx.data_ptr(), *dwp = address(dw), *dbp = address(db), *sp = address(scratch);
  run(r.dev, "layer_norm_backward", [&](haste_stream_t st) {
    return lib.layer_norm_backward(gp, xp, w, mp, rp, dxp, dwp, dbp, sp, bytes, rows, r.D, ldg, ld, r.type, dy_type, code_of(type), st);
  });
  PyObject* out = PyTuple_New(3);
  if (out == nullptr) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(dx));
  for (int i = 1; i < 3; ++i) {
    const at::Tensor& t = i == 1 ? dw : db;
    if (t.defined()) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(t));
    else { Py_INCREF(Py_None); PyTuple_SET_ITEM(out, i, Py_None); }
  }
  return out;
}

// A list or tuple of tensors, or anything that can be walked over, as it is now: other threads may change a list while a launch has let go of the lock
struct Sequence {
  PyObject* items;
  explicit Sequence(PyObject* o) : items(PySequence_Tuple(o)) {
    if (items == nullptr) throw python_error();
  }
  ~Sequence() { Py_DECREF(items); }
  Sequence(const Sequence&) = delete;
  Sequence& operator=(const Sequence&) = delete;
  int64_t size() const { return PyTuple_GET_SIZE(items); }
  PyObject* operator[](int64_t i) const { return PyTuple_GET_ITEM(items, i); }
};

struct TensorList {
  int dev = -1;
  std::vector<const void*> p;      // NULL where the list has None
  std::vector<int32_t> types;
  std::vector<int64_t> sizes;
  int64_t present = 0;
  TensorList(const Sequence& list, const char* what) {
    const int64_t n = list.size();
    p.reserve(n); types.reserve(n); sizes.reserve(n);
    for (int64_t i = 0; i < n; ++i) {
      if (list[i] == Py_None) { p.push_back(nullptr); types.push_back(0); sizes.push_back(0); continue; }
      const at::Tensor& t = tensor(list[i], what);
      const int d = gpu_of(t);
      if (d < 0 || (present > 0 && d != dev)) refuse(std::string(what) + " must be CUDA tensors on one device (this library has no CPU path)");
      if (!t.is_contiguous()) refuse(std::string(what) + " must be contiguous");
      dev = d;
      types.push_back(type_of(t, what));
      sizes.push_back(t.numel());
      p.push_back(t.data_ptr());
      ++present;
    }
  }
};

at::Tensor norm_of(const TensorList& g, double scale) {
  at::Tensor norm = empty_on(g.dev, {}, at::kFloat), scratch = empty_on(g.dev, {HASTE_GRAD_NORM_PARTIALS}, at::kFloat);
  float *np = static_cast<float*>(norm.data_ptr()), *sp = static_cast<float*>(scratch.data_ptr());
  const TensorList* all = &g;
  std::vector<const void*> p;
  std::vector<int32_t> types;
  std::vector<int64_t> sizes;
  if (g.present != static_cast<int64_t>(g.p.size()))
    for (size_t i = 0; i < g.p.size(); ++i)
      if (g.sizes[i] > 0) { p.push_back(g.p[i]); types.push_back(g.types[i]); sizes.push_back(g.sizes[i]); }
  const bool some = g.present != static_cast<int64_t>(g.p.size());
  const void* const* ps = some ? p.data() : all->p.data();
  const int32_t* ts = some ? types.data() : all->types.data();
  const int64_t* ss = some ? sizes.data() : all->sizes.data();
  const int64_t n = static_cast<int64_t>(some ? p.size() : all->p.size());
  run(g.dev, "grad_norm", [&](haste_stream_t st) { return lib.grad_norm(ps, ts, ss, n, static_cast<float>(scale), sp, np, st); });
  return norm;
}

// (grads, grad_scale) -> norm
PyObject* grad_norm(PyObject* const* a) {
  const double scale = PyFloat_AsDouble(a[1]);
  if (PyErr_Occurred()) throw python_error();
  const Sequence list(a[0]);
  const TensorList g(list, "gradients");
  if (g.present == 0) refuse("grad_norm needs at least one tensor");
  return THPVariable_Wrap(norm_of(g, scale));
}

constexpr int64_t MOMENT_BLOCK = 256;

// (params, grads, exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale, bits, step, lr, beta1, beta2, eps, weight_decay, grad_scale, norm, max_norm, seed,
// stream_index, flags) -> norm or None
PyObject* adamw_step(PyObject* const* a) {
  const Sequence params(a[0]), grads(a[1]);
  if (params.size() != grads.size()) refuse(std::to_string(params.size()) + " parameters and " + std::to_string(grads.size()) + " gradients");
  const int64_t bits = PyLong_AsLongLong(a[6]), step = PyLong_AsLongLong(a[7]);
  double number[6];                     // lr, beta1, beta2, eps, weight_decay, grad_scale
  for (int i = 0; i < 6; ++i) number[i] = PyFloat_AsDouble(a[8 + i]);
  const double max_norm = a[15] == Py_None ? 0.0 : PyFloat_AsDouble(a[15]);
  const uint64_t seed = PyLong_AsUnsignedLongLongMask(a[16]);
  const uint32_t stream_index = static_cast<uint32_t>(PyLong_AsUnsignedLongMask(a[17])), flags = static_cast<uint32_t>(PyLong_AsUnsignedLongMask(a[18]));
  if (PyErr_Occurred()) throw python_error();
  const TensorList g(grads, "gradients");
  if (g.present == 0) Py_RETURN_NONE;       // nothing to do
  const TensorList p(params, "parameters");
  if (p.present != params.size()) refuse("parameters must be tensors");
  if (p.dev != g.dev) refuse("parameters and gradients must be on one device");
  int g_type = -1;
  for (int64_t i = 0; i < params.size(); ++i) {
    bool fine = p.types[i] == p.types[0];
    if (grads[i] != Py_None) {
      if (g_type < 0) g_type = g.types[i];
      fine = fine && g.types[i] == g_type && THPVariable_Unpack(params[i]).sizes().equals(THPVariable_Unpack(grads[i]).sizes());
    }
    if (!fine) refuse("all parameters must have one type, all gradients one type, and every gradient its parameter's shape");
  }
  const at::Tensor &m = tensor(a[2], "exp_avg"), &v = tensor(a[4], "exp_avg_sq");
  const int64_t moments = m.numel();
  for (const at::Tensor* t : {&m, &v})
    if (gpu_of(*t) != p.dev || t->scalar_type() != (bits == 32 ? at::kFloat : at::kByte) || t->numel() != moments || !t->is_contiguous())
      refuse(std::string("both moments must be contiguous ") + (bits == 32 ? "fp32" : "uint8") + " tensors of one size on the parameters' device");
  float *ms = nullptr, *vs = nullptr;
  if (bits == 8)
    for (int i : {3, 5}) {
      const at::Tensor& t = tensor(a[i], "scales");
      if (gpu_of(t) != p.dev || t.scalar_type() != at::kFloat || t.numel() * MOMENT_BLOCK < moments || !t.is_contiguous())
        refuse("scales must be contiguous, fp32, one value per 256 elements of the moments, on the parameters' device");
      (i == 3 ? ms : vs) = static_cast<float*>(t.data_ptr());
    }
  at::Tensor norm;
  if (a[15] != Py_None) {
    if (a[14] == Py_None) {
      norm = norm_of(g, number[5]);
    } else {
      norm = tensor(a[14], "norm");
      if (gpu_of(norm) != p.dev || norm.scalar_type() != at::kFloat || norm.numel() != 1) refuse("norm must be one fp32 value on the parameters' device");
    }
  }
  void *mp = m.data_ptr(), *vp = v.data_ptr();
  const float* np = static_cast<const float*>(address(norm));
  run(p.dev, "adamw_step", [&](haste_stream_t st) {
    return lib.adamw_step(const_cast<void* const*>(p.p.data()), g.p.data(), p.sizes.data(), params.size(), mp, ms, vp, vs, moments, static_cast<int32_t>(bits), p.types[0], g_type,
                          number[0], number[1], number[2], number[3], number[4], step, static_cast<float>(number[5]), static_cast<float>(max_norm), np, seed, stream_index, flags, st);
  });
  for (int64_t i = 0; i < params.size(); ++i)
    if (grads[i] != Py_None) written(THPVariable_Unpack(params[i]));
  written(m);
  written(v);
  if (bits == 8)
    for (int i : {3, 5}) written(THPVariable_Unpack(a[i]));
  if (!norm.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(norm);
}

// (codes, scales, signed, dtype) -> values
PyObject* dequantize_moment(PyObject* const* a) {
  const at::Tensor &codes = tensor(a[0], "codes"), &scales = tensor(a[1], "scales");
  const int dev = gpu_of(codes), is_signed = PyObject_IsTrue(a[2]);
  if (PyErr_Occurred()) throw python_error();
  if (dev < 0) refuse("codes must be a CUDA tensor (this library has no CPU path)");
  if (codes.scalar_type() != at::kByte || !codes.is_contiguous()) refuse("codes must be contiguous uint8");
  if (gpu_of(scales) != dev || scales.scalar_type() != at::kFloat || !scales.is_contiguous() || scales.numel() * MOMENT_BLOCK != codes.numel())
    refuse("scales must be contiguous fp32 and hold one value per 256 codes, on their device");
  const at::ScalarType type = THPDtype_Check(a[3]) ? reinterpret_cast<THPDtype*>(a[3])->scalar_type : at::kByte;
  if (code_of(type) < 0) refuse("dtype must be torch.bfloat16 or torch.float32");
  at::Tensor out = empty_on(dev, codes.sizes(), type);
  const auto* cp = static_cast<const uint8_t*>(codes.data_ptr());
  const auto* sp = static_cast<const float*>(scales.data_ptr());
  void* op = out.data_ptr();
  const int64_t n = codes.numel();
  run(dev, "dequantize_moment", [&](haste_stream_t st) { return lib.dequantize_moment(cp, sp, op, n, is_signed, code_of(type), st); });
  return THPVariable_Wrap(out);
}

// (three tensors or None) -> whether one has a tangent of forward-mode differentiation
PyObject* has_tangent(PyObject* const* a) {
  for (int i = 0; i < 3; ++i)
    if (THPVariable_Check(a[i]) && THPVariable_Unpack(a[i])._fw_grad(/*level=*/0).defined()) Py_RETURN_TRUE;
  Py_RETURN_FALSE;
}

// Addresses of the library's functions, in the order of Library's members
PyObject* bind(PyObject* const* a) {
  void* at[7];
  for (int i = 0; i < 7; ++i) at[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) throw python_error();
  lib = {reinterpret_cast<decltype(lib.last_error)>(at[0]),
         reinterpret_cast<decltype(lib.layer_norm_forward)>(at[1]),
         reinterpret_cast<decltype(lib.layer_norm_backward_scratch)>(at[2]),
         reinterpret_cast<decltype(lib.layer_norm_backward)>(at[3]),
         reinterpret_cast<decltype(lib.adamw_step)>(at[4]),
         reinterpret_cast<decltype(lib.grad_norm)>(at[5]),
         reinterpret_cast<decltype(lib.dequantize_moment)>(at[6])};
  Py_RETURN_NONE;
}

// A function of N positional arguments; what it refuses becomes a RuntimeError
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define ENTRY(f, n) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(bind, 7), ENTRY(layer_norm_forward, 5), ENTRY(layer_norm_backward, 8), ENTRY(grad_norm, 2), ENTRY(adamw_step, 19),
                         ENTRY(dequantize_moment, 4), ENTRY(has_tangent, 3), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_dense", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dense() { return PyModule_Create(&module); }
