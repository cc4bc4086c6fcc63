// The Python side of the dense operators (layer norm, AdamW, gradient norm and the decoding of moments, token embedding, the gated feed-forward block, Muon): tensors are looked at, outputs and workspaces are allocated and the
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

#include <algorithm>
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
  decltype(&haste_embedding_forward) embedding_forward;
  decltype(&haste_embedding_backward_scratch) embedding_backward_scratch;
  decltype(&haste_embedding_backward) embedding_backward;
  decltype(&haste_gated_forward_scratch) gated_forward_scratch;
  decltype(&haste_gated_forward) gated_forward;
  decltype(&haste_gated_backward_scratch) gated_backward_scratch;
  decltype(&haste_gated_backward) gated_backward;
  decltype(&haste_muon_scratch) muon_scratch;
  decltype(&haste_muon_step) muon_step;
  decltype(&haste_orthogonalize) orthogonalize;
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

// rows_of, but with rows that do not overlap
std::pair<at::Tensor, int64_t> own_rows_of(const at::Tensor& t, int64_t D) {
  auto r = rows_of(t, D);
  if (r.second < D) return {r.first.contiguous(), D};
  return r;
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

// ---------------------------------------------------------------- token embedding
// ids as the library takes them: contiguous, on `dev`
struct Ids {
  at::Tensor t;
  int bytes;
};
Ids check_ids(PyObject* o, int dev) {
  if (!THPVariable_Check(o)) refuse("ids must be a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (gpu_of(t) < 0) refuse("ids must be a CUDA tensor (this library has no CPU path)");
  if (dev >= 0 && gpu_of(t) != dev) refuse("ids must be on cuda:" + std::to_string(dev) + ", as the other tensors are, got " + t.device().str());
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt) refuse("ids must be torch.int64 or torch.int32, got " + text(t.scalar_type()));
  return {t.is_contiguous() ? t : t.contiguous(), t.scalar_type() == at::kLong ? 8 : 4};
}

// (ids, table, scale) -> y
PyObject* embedding_forward(PyObject* const* a) {
  const at::Tensor& table = tensor(a[1], "table");
  const int dev = gpu_of(table);
  if (dev < 0) refuse("table must be a CUDA tensor (this library has no CPU path)");
  if (table.dim() != 2 || table.size(0) < 1 || table.size(1) < 1) refuse("table must be [V, D], got " + text(table.sizes()));
  const int type = type_of(table, "table");
  const Ids ids = check_ids(a[0], dev);
  const double scale = PyFloat_AsDouble(a[2]);
  if (PyErr_Occurred()) throw python_error();
  const int64_t V = table.size(0), D = table.size(1), tokens = ids.t.numel();
  const auto [src, stride] = own_rows_of(table, D);
  std::vector<int64_t> sizes(ids.t.sizes().begin(), ids.t.sizes().end());
  sizes.push_back(D);
  at::Tensor y = empty_on(dev, sizes, table.scalar_type());
  const void *ip = ids.t.data_ptr(), *tp = src.data_ptr();
  void* yp = y.data_ptr();
  const int64_t ld = stride;
  run(dev, "embedding_forward", [&](haste_stream_t st) { return lib.embedding_forward(ip, ids.bytes, tp, yp, tokens, D, V, ld, static_cast<float>(scale), type, st); });
  return THPVariable_Wrap(y);
}

// (dy, ids, rows, scale, padding, dtype) -> dtable
PyObject* embedding_backward(PyObject* const* a) {
  const at::Tensor& dy = tensor(a[0], "dy");
  const int dev = gpu_of(dy);
  if (dev < 0) refuse("dy must be a CUDA tensor (this library has no CPU path)");
  const int dy_type = type_of(dy, "dy");
  const Ids ids = check_ids(a[1], dev);
  const int64_t V = PyLong_AsLongLong(a[2]), padding = PyLong_AsLongLong(a[4]);
  const double scale = PyFloat_AsDouble(a[3]);
  if (PyErr_Occurred()) throw python_error();
  if (V < 1) refuse("a table of " + std::to_string(V) + " rows");
  if (dy.dim() != ids.t.dim() + 1 || !dy.sizes().slice(0, ids.t.dim()).equals(ids.t.sizes()) || dy.size(-1) < 1)
    refuse("dy must be [..., D] for ids of shape " + text(ids.t.sizes()) + ", got " + text(dy.sizes()));
  at::ScalarType type = dy.scalar_type();
  if (a[5] != Py_None) {
    if (!THPDtype_Check(a[5]) || code_of(reinterpret_cast<THPDtype*>(a[5])->scalar_type) < 0) refuse("dtype must be torch.bfloat16 or torch.float32");
    type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  }
  const int64_t D = dy.size(-1), tokens = ids.t.numel();
  const auto [grad, stride] = rows_of(dy, D);
  at::Tensor out = empty_on(dev, {V, D}, type), scratch;
  int64_t bytes = 0;
  {
    const c10::cuda::OptionalCUDAGuard guard(dy.device());
    bytes = lib.embedding_backward_scratch(tokens, D, V);
  }
  scratch = empty_on(dev, {bytes}, at::kByte);
  const void *gp = grad.data_ptr(), *ip = ids.t.data_ptr();
  void *op = out.data_ptr(), *sp = scratch.data_ptr();
  const int64_t ld = stride;
  run(dev, "embedding_backward", [&](haste_stream_t st) {
    return lib.embedding_backward(ip, ids.bytes, gp, op, sp, bytes, tokens, D, V, ld, static_cast<float>(scale), padding, dy_type, code_of(type), st);
  });
  return THPVariable_Wrap(out);
}

// ---------------------------------------------------------------- gated feed-forward block
struct GatedSizes {
  int dev;
  int64_t T, D, F, O;
};
void check_bf16(const at::Tensor& t, const char* name, int dev) {
  if (gpu_of(t) != dev) refuse(std::string(name) + " must be a CUDA tensor on cuda:" + std::to_string(dev) + ", as x is, got " + t.device().str());
  if (t.scalar_type() != at::kBFloat16) refuse(std::string(name) + " must be torch.bfloat16, got " + text(t.scalar_type()));
}
// x and the weights at a[0 .. 3]
GatedSizes check_gated(PyObject* const* a) {
  if (!THPVariable_Check(a[0]) || !THPVariable_Unpack(a[0]).is_cuda()) refuse("x must be a CUDA tensor (this library has no CPU path)");
  const at::Tensor& x = THPVariable_Unpack(a[0]);
  GatedSizes s;
  s.dev = gpu_of(x);
  check_bf16(x, "x", s.dev);
  if (x.dim() < 1 || x.size(-1) < 1) refuse("x must be [..., D] with D >= 1, got " + text(x.sizes()));
  s.D = x.size(-1);
  s.T = x.numel() / s.D;
  const at::Tensor &wg = tensor(a[1], "w_gate"), &wu = tensor(a[2], "w_up"), &wd = tensor(a[3], "w_down");
  for (const auto& [t, name] : {std::pair<const at::Tensor*, const char*>{&wg, "w_gate"}, {&wu, "w_up"}, {&wd, "w_down"}}) {
    check_bf16(*t, name, s.dev);
    if (t->dim() != 2 || !t->is_contiguous() || t->numel() == 0) refuse(std::string(name) + " must be a contiguous matrix, got " + text(t->sizes()));
  }
  s.F = wg.size(0);
  s.O = wd.size(0);
  if (wg.size(1) != s.D || !wu.sizes().equals(wg.sizes()) || wd.size(1) != s.F)
    refuse("w_gate and w_up must be [F, " + std::to_string(s.D) + "], w_down [O, F], got " + text(wg.sizes()) + ", " + text(wu.sizes()) + " and " + text(wd.sizes()));
  return s;
}
bool on16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
// rows x F, a row's stride a multiple of 8
at::Tensor padded(int dev, int64_t rows, int64_t F) {
  const int64_t ld = (F + 7) / 8 * 8;
  at::Tensor t = empty_on(dev, {rows, ld}, at::kBFloat16);
  return ld == F ? t : t.narrow(1, 0, F);
}
std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> s(sizes.begin(), sizes.end());
  s.back() = last;
  return s;
}
int activation_of(PyObject* o) {
  const long act = PyLong_AsLong(o);
  if (PyErr_Occurred()) throw python_error();
  return static_cast<int>(act);
}

// (x, w_gate, w_up, w_down, activation, keep) -> y, or (y, gate, up)
PyObject* gated_forward(PyObject* const* a) {
  const GatedSizes s = check_gated(a);
  const int act = activation_of(a[4]), keep = PyObject_IsTrue(a[5]);
  if (PyErr_Occurred()) throw python_error();
  const at::Tensor &x = THPVariable_Unpack(a[0]), &wg = THPVariable_Unpack(a[1]), &wu = THPVariable_Unpack(a[2]), &wd = THPVariable_Unpack(a[3]);
  const auto [src, stride] = own_rows_of(x, s.D);
  const int64_t ldx = stride;
  at::Tensor y = empty_on(s.dev, with_last(x.sizes(), s.O), at::kBFloat16), gate, up, scratch;
  if (keep) {
    gate = padded(s.dev, s.T, s.F);
    up = padded(s.dev, s.T, s.F);
  }
  const bool aligned = (s.D | s.F | s.O | ldx) % 8 == 0 && on16(src) && on16(wg) && on16(wu) && on16(wd);
  int64_t bytes = 0;
  {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    bytes = lib.gated_forward_scratch(s.T, s.D, s.F, s.O, aligned);
  }
  scratch = empty_on(s.dev, {bytes}, at::kByte);
  const void *xp = src.data_ptr(), *gp = wg.data_ptr(), *up_ = wu.data_ptr(), *dp = wd.data_ptr();
  void *yp = y.data_ptr(), *kg = address(gate), *ku = address(up), *sp = scratch.data_ptr();
  const int64_t ldh = (s.F + 7) / 8 * 8;
  run(s.dev, "gated_forward", [&](haste_stream_t st) { return lib.gated_forward(xp, gp, up_, dp, kg, ku, yp, sp, bytes, s.T, s.D, s.F, s.O, ldx, ldh, act, st); });
  if (!keep) return THPVariable_Wrap(y);
  const std::vector<int64_t> shape = with_last(x.sizes(), s.F);
  PyObject* out = PyTuple_New(3);
  if (out == nullptr) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(y));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(gate.view(shape)));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(up.view(shape)));
  return out;
}

// (x, w_gate, w_up, w_down, dy, gate, up, activation, want_x, want_gate, want_up, want_down) -> (dx, dw_gate, dw_up, dw_down)
PyObject* gated_backward(PyObject* const* a) {
  const GatedSizes s = check_gated(a);
  const at::Tensor &x = THPVariable_Unpack(a[0]), &wg = THPVariable_Unpack(a[1]), &wu = THPVariable_Unpack(a[2]), &wd = THPVariable_Unpack(a[3]);
  const at::Tensor &dy = tensor(a[4], "dy"), &gate = tensor(a[5], "gate"), &up = tensor(a[6], "up");
  const std::vector<int64_t> shape_y = with_last(x.sizes(), s.O), shape_h = with_last(x.sizes(), s.F);
  for (const auto& [t, name, shape] : {std::tuple<const at::Tensor*, const char*, const std::vector<int64_t>*>{&dy, "dy", &shape_y}, {&gate, "gate", &shape_h}, {&up, "up", &shape_h}}) {
    check_bf16(*t, name, s.dev);
    if (!t->sizes().equals(*shape)) refuse(std::string(name) + " must be " + text(*shape) + ", got " + text(t->sizes()));
  }
  const int act = activation_of(a[7]);
  int want[4];
  for (int i = 0; i < 4; ++i) want[i] = PyObject_IsTrue(a[8 + i]);
  if (PyErr_Occurred()) throw python_error();
  const auto [xs, sx] = own_rows_of(x, s.D);
  const auto [ys, sy] = own_rows_of(dy, s.O);
  const auto [gs, sg] = own_rows_of(gate, s.F);
  const auto [us, su] = own_rows_of(up, s.F);
  const int64_t ldx = sx, lddy = sy, ldg = sg, ldu = su;
  at::Tensor out[4], scratch;
  if (want[0]) out[0] = empty_on(s.dev, x.sizes(), at::kBFloat16);
  if (want[1]) out[1] = empty_on(s.dev, {s.F, s.D}, at::kBFloat16);
  if (want[2]) out[2] = empty_on(s.dev, {s.F, s.D}, at::kBFloat16);
  if (want[3]) out[3] = empty_on(s.dev, {s.O, s.F}, at::kBFloat16);
  bool aligned = (s.D | s.F | s.O | ldx | lddy | ldg) % 8 == 0 && ldg == ldu;
  for (const at::Tensor* t : {&xs, &ys, &gs, &us, &wg, &wu, &wd}) aligned = aligned && on16(*t);
  int64_t bytes = 0;
  {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    bytes = lib.gated_backward_scratch(s.T, s.D, s.F, s.O, aligned);
  }
  scratch = empty_on(s.dev, {bytes}, at::kByte);
  const void *yp = ys.data_ptr(), *xp = xs.data_ptr(), *w0 = wg.data_ptr(), *w1 = wu.data_ptr(), *w2 = wd.data_ptr(), *gp = gs.data_ptr(), *up_ = us.data_ptr();
  void *o0 = address(out[0]), *o1 = address(out[1]), *o2 = address(out[2]), *o3 = address(out[3]), *sp = scratch.data_ptr();
  run(s.dev, "gated_backward", [&](haste_stream_t st) {
    return lib.gated_backward(yp, xp, w0, w1, w2, gp, up_, o0, o1, o2, o3, sp, bytes, s.T, s.D, s.F, s.O, lddy, ldx, ldg, ldu, act, st);
  });
  PyObject* result = PyTuple_New(4);
  if (result == nullptr) throw python_error();
  for (int i = 0; i < 4; ++i) {
    if (out[i].defined()) PyTuple_SET_ITEM(result, i, THPVariable_Wrap(out[i]));
    else { Py_INCREF(Py_None); PyTuple_SET_ITEM(result, i, Py_None); }
  }
  return result;
}

// ---------------------------------------------------------------- Muon
// Rows and columns of a list of matrices; None counts as an empty one
void sizes_of(const Sequence& list, const TensorList& t, const char* what, std::vector<int64_t>& rows, std::vector<int64_t>& cols) {
  for (int64_t i = 0; i < list.size(); ++i) {
    if (t.p[i] == nullptr && list[i] == Py_None) { rows.push_back(0); cols.push_back(0); continue; }
    const at::Tensor& x = THPVariable_Unpack(list[i]);
    if (x.dim() != 2) refuse(std::string(what) + " must be matrices, got " + text(x.sizes()));
    rows.push_back(x.size(0));
    cols.push_back(x.size(1));
  }
}
at::Tensor muon_workspace(int dev, const std::vector<int64_t>& rows, const std::vector<int64_t>& cols, int64_t& bytes) {
  bytes = lib.muon_scratch(rows.data(), cols.data(), static_cast<int64_t>(rows.size()));
  return empty_on(dev, {bytes}, at::kByte);
}

// The number of Newton-Schulz steps: what does not fit the library's 32 bits is no other number of steps
int32_t steps_of(PyObject* o) {
  const long steps = PyLong_AsLong(o);
  if (PyErr_Occurred()) throw python_error();
  if (steps != static_cast<int32_t>(steps)) refuse("steps=" + std::to_string(steps) + " is out of range");
  return static_cast<int32_t>(steps);
}

// (params, grads, momentum, step, lr, mu, nesterov, weight_decay, adjust, steps, a, b, c, eps, seed, stream_index, flags)
PyObject* muon_step(PyObject* const* a) {
  const Sequence params(a[0]), grads(a[1]);
  if (params.size() != grads.size()) refuse(std::to_string(params.size()) + " parameters and " + std::to_string(grads.size()) + " gradients");
  const int64_t step = PyLong_AsLongLong(a[3]);
  const double lr = PyFloat_AsDouble(a[4]), mu = PyFloat_AsDouble(a[5]), weight_decay = PyFloat_AsDouble(a[7]);
  const int nesterov = PyObject_IsTrue(a[6]);
  const long adjust = PyLong_AsLong(a[8]);
  double number[4];                     // a, b, c, eps
  for (int i = 0; i < 4; ++i) number[i] = PyFloat_AsDouble(a[10 + i]);
  const uint64_t seed = PyLong_AsUnsignedLongLongMask(a[14]);
  const uint32_t stream_index = static_cast<uint32_t>(PyLong_AsUnsignedLongMask(a[15])), flags = static_cast<uint32_t>(PyLong_AsUnsignedLongMask(a[16]));
  if (PyErr_Occurred()) throw python_error();
  const int32_t steps = steps_of(a[9]);
  const TensorList g(grads, "gradients");
  if (g.present == 0) Py_RETURN_NONE;       // nothing to do
  const TensorList p(params, "parameters");
  if (p.present != params.size()) refuse("parameters must be tensors");
  if (p.dev != g.dev) refuse("parameters and gradients must be on one device");
  std::vector<int64_t> rows, cols;
  sizes_of(params, p, "parameters", rows, cols);
  int g_type = -1;
  for (int64_t i = 0; i < params.size(); ++i) {
    bool fine = p.types[i] == p.types[0];
    if (grads[i] != Py_None) {
      if (g_type < 0) g_type = g.types[i];
      fine = fine && g.types[i] == g_type && THPVariable_Unpack(params[i]).sizes().equals(THPVariable_Unpack(grads[i]).sizes());
    }
    if (!fine) refuse("all parameters must have one type, all gradients one type, and every gradient its parameter's shape");
  }
  std::vector<const void*> once;
  for (int64_t i = 0; i < params.size(); ++i)
    if (p.p[i] != nullptr && p.sizes[i] > 0 && grads[i] != Py_None) once.push_back(p.p[i]);
  std::sort(once.begin(), once.end());
  if (std::adjacent_find(once.begin(), once.end()) != once.end()) refuse("a parameter stands in the list twice");
  const at::Tensor& m = tensor(a[2], "momentum_buffer");
  if (gpu_of(m) != p.dev || m.scalar_type() != at::kFloat || !m.is_contiguous()) refuse("momentum_buffer must be a contiguous fp32 tensor on the parameters' device");
  int64_t bytes = 0;
  const at::Tensor scratch = muon_workspace(p.dev, rows, cols, bytes);
  float* mp = static_cast<float*>(m.data_ptr());
  void* sp = scratch.data_ptr();
  const int64_t moments = m.numel();
  run(p.dev, "muon_step", [&](haste_stream_t st) {
    return lib.muon_step(const_cast<void* const*>(p.p.data()), g.p.data(), rows.data(), cols.data(), params.size(), mp, moments, p.types[0], g_type, lr, mu, nesterov, weight_decay,
                         static_cast<int32_t>(adjust), steps, number[0], number[1], number[2], number[3], step, seed, stream_index, flags, sp, bytes, st);
  });
  for (int64_t i = 0; i < params.size(); ++i)
    if (grads[i] != Py_None) written(THPVariable_Unpack(params[i]));
  written(m);
  Py_RETURN_NONE;
}

// (matrices, steps, a, b, c, eps) -> list of bf16 matrices
PyObject* orthogonalize(PyObject* const* a) {
  const Sequence list(a[0]);
  const int32_t steps = steps_of(a[1]);
  double number[4];
  for (int i = 0; i < 4; ++i) number[i] = PyFloat_AsDouble(a[2 + i]);
  if (PyErr_Occurred()) throw python_error();
  const TensorList in(list, "matrices");
  if (in.present != list.size()) refuse("matrices must be tensors");
  std::vector<int64_t> rows, cols;
  sizes_of(list, in, "matrices", rows, cols);
  for (int64_t i = 1; i < list.size(); ++i)
    if (in.types[i] != in.types[0]) refuse("all matrices must have one type");
  std::vector<at::Tensor> out;
  std::vector<void*> to;
  for (int64_t i = 0; i < list.size(); ++i) {
    out.push_back(empty_on(in.dev, {rows[i], cols[i]}, at::kBFloat16));
    to.push_back(out.back().data_ptr());
  }
  if (!out.empty()) {
    int64_t bytes = 0;
    const at::Tensor scratch = muon_workspace(in.dev, rows, cols, bytes);
    void* sp = scratch.data_ptr();
    run(in.dev, "orthogonalize", [&](haste_stream_t st) {
      return lib.orthogonalize(in.p.data(), to.data(), rows.data(), cols.data(), list.size(), in.types[0], steps, number[0], number[1], number[2], number[3], sp, bytes, st);
    });
  }
  PyObject* result = PyList_New(list.size());
  if (result == nullptr) throw python_error();
  for (int64_t i = 0; i < list.size(); ++i) PyList_SET_ITEM(result, i, THPVariable_Wrap(out[i]));
  return result;
}

// (three tensors or None) -> whether one has a tangent of forward-mode differentiation
PyObject* has_tangent(PyObject* const* a) {
  for (int i = 0; i < 3; ++i)
    if (THPVariable_Check(a[i]) && THPVariable_Unpack(a[i])._fw_grad(/*level=*/0).defined()) Py_RETURN_TRUE;
  Py_RETURN_FALSE;
}

// Addresses of the library's functions, in the order of Library's members
constexpr int LIBRARY = 17;
PyObject* bind(PyObject* const* a) {
  void* at[LIBRARY];
  for (int i = 0; i < LIBRARY; ++i) at[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) throw python_error();
  lib = {reinterpret_cast<decltype(lib.last_error)>(at[0]),
         reinterpret_cast<decltype(lib.layer_norm_forward)>(at[1]),
         reinterpret_cast<decltype(lib.layer_norm_backward_scratch)>(at[2]),
         reinterpret_cast<decltype(lib.layer_norm_backward)>(at[3]),
         reinterpret_cast<decltype(lib.adamw_step)>(at[4]),
         reinterpret_cast<decltype(lib.grad_norm)>(at[5]),
         reinterpret_cast<decltype(lib.dequantize_moment)>(at[6]),
         reinterpret_cast<decltype(lib.embedding_forward)>(at[7]),
         reinterpret_cast<decltype(lib.embedding_backward_scratch)>(at[8]),
         reinterpret_cast<decltype(lib.embedding_backward)>(at[9]),
         reinterpret_cast<decltype(lib.gated_forward_scratch)>(at[10]),
         reinterpret_cast<decltype(lib.gated_forward)>(at[11]),
         reinterpret_cast<decltype(lib.gated_backward_scratch)>(at[12]),
         reinterpret_cast<decltype(lib.gated_backward)>(at[13]),
         reinterpret_cast<decltype(lib.muon_scratch)>(at[14]),
         reinterpret_cast<decltype(lib.muon_step)>(at[15]),
         reinterpret_cast<decltype(lib.orthogonalize)>(at[16])};
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
PyMethodDef methods[] = {ENTRY(bind, LIBRARY), ENTRY(layer_norm_forward, 5), ENTRY(layer_norm_backward, 8), ENTRY(grad_norm, 2), ENTRY(adamw_step, 19),
                         ENTRY(dequantize_moment, 4), ENTRY(has_tangent, 3), ENTRY(embedding_forward, 3),
                         ENTRY(embedding_backward, 6), ENTRY(gated_forward, 6), ENTRY(gated_backward, 12), ENTRY(muon_step, 17), ENTRY(orthogonalize, 6), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_dense", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dense() { return PyModule_Create(&module); }
