// Python module _dense: the host side of a call of a dense operator
// (lib/nn/dense.py): checks of the arguments, outputs, and the call of the
// library's C ABI.
//
// These calls are a few microseconds of GPU work where the batch is small, and
// an AdamW step looks at six properties of hundreds of tensors: from Python,
// through ctypes, that is 4 us an operator call and 3 us a tensor. The module
// is the same code against torch's tensors directly. The library's functions
// are handed over by bind(), so there is one copy of it in the process.
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <algorithm>
#include <cstring>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "../../include/scemb.h"

namespace {

using at::Tensor;

struct Library {
  decltype(&scemb_last_error) last_error;
  decltype(&scemb_layer_norm) layer_norm;
  decltype(&scemb_layer_norm_grad_workspace_size) layer_norm_grad_workspace;
  decltype(&scemb_layer_norm_grad) layer_norm_grad;
  decltype(&scemb_sort_by_expert_workspace_size) sort_by_expert_workspace;
  decltype(&scemb_sort_by_expert) sort_by_expert;
  decltype(&scemb_tokens_to_experts) tokens_to_experts;
  decltype(&scemb_tokens_from_experts) tokens_from_experts;
  decltype(&scemb_tokens_from_experts_grad) tokens_from_experts_grad;
  decltype(&scemb_expert_matmul_workspace_size) expert_matmul_workspace;
  decltype(&scemb_expert_matmul) expert_matmul;
  decltype(&scemb_expert_matmul_weights_grad_workspace_size)
      expert_matmul_weights_grad_workspace;
  decltype(&scemb_expert_matmul_weights_grad) expert_matmul_weights_grad;
  decltype(&scemb_quantize_weights) quantize_weights;
  decltype(&scemb_matmul_8bit_workspace_size) matmul_8bit_workspace;
  decltype(&scemb_matmul_8bit) matmul_8bit;
  decltype(&scemb_gradient_norm_workspace_size) gradient_norm_workspace;
  decltype(&scemb_gradient_norm) gradient_norm;
  decltype(&scemb_clip_gradients) clip_gradients;
  decltype(&scemb_adamw_update) adamw_update;
  decltype(&scemb_adamw_moments) adamw_moments;
};
Library lib = {};
PyObject* raw_stream = nullptr;  // the handle of a device's current stream

// A Python exception that is already set.
struct Raised {};

[[noreturn]] void Refuse(const std::string& message) {
  throw std::invalid_argument(message);
}

void Check(int rc) {
  if (rc == SCEMB_OK) return;
  const std::string message = lib.last_error();
  if (rc == SCEMB_ERR_INVALID_ARGUMENT) Refuse(message);
  throw std::runtime_error("libscemb error " + std::to_string(rc) + ": " +
                           message);
}

// Runs a call and turns its C++ exceptions into Python's.
template <typename F>
PyObject* Guarded(F f) {
  try {
    if (lib.last_error == nullptr) {
      throw std::runtime_error("_dense.bind() was not called");
    }
    return f();
  } catch (const Raised&) {
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (...) {
    // torch's own, running out of memory among them, stay what callers catch.
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

// ---------------------------------------------------------------------------
// Arguments.
// ---------------------------------------------------------------------------

int CurrentDevice() {
  return c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getDevice().index();
}

int64_t Int(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
double Float(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}
void* Address(PyObject* o) {
  return o == Py_None ? nullptr : reinterpret_cast<void*>(Int(o));
}

void* Stream(int device) {
  PyObject* index = PyLong_FromLong(device);
  if (index == nullptr) throw Raised();
  PyObject* o = PyObject_CallOneArg(raw_stream, index);
  Py_DECREF(index);
  if (o == nullptr) throw Raised();
  void* stream = PyLong_AsVoidPtr(o);
  Py_DECREF(o);
  if (stream == nullptr && PyErr_Occurred()) throw Raised();
  return stream;
}

constexpr uint32_t Bit(at::ScalarType t) {
  return 1u << static_cast<uint32_t>(t);
}
constexpr uint32_t kF32 = Bit(at::kFloat);
constexpr uint32_t kBf16 = Bit(at::kBFloat16);
constexpr uint32_t kF16 = Bit(at::kHalf);
constexpr uint32_t kI32 = Bit(at::kInt);
constexpr uint32_t kI64 = Bit(at::kLong);
constexpr uint32_t kRowTypes = kF32 | kBf16 | kF16;

template <typename T>
std::string Text(const T& v) {
  std::ostringstream s;
  s << v;
  return s.str();
}

std::string TypeNames(uint32_t types) {
  std::string s;
  for (int i = 0; i < 32; ++i) {
    if (types >> i & 1u) {
      s += (s.empty() ? "" : ", ") + Text(static_cast<at::ScalarType>(i));
    }
  }
  return s;
}

// Whether the tensor's memory holds its values: views that are negated when
// they are read, and zeros that were never written, have others.
bool HoldsValues(const Tensor& t) { return !t.is_neg() && !t._is_zerotensor(); }

// Whether the tensor carries a tangent of forward-mode differentiation.
bool HasTangent(const Tensor& t) {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
         t._fw_grad(/*level=*/0).defined();
}

// The kernels know no tangents: a result without one would be taken for a
// constant.
void CheckTangent(const Tensor& t, const std::string& name) {
  if (HasTangent(t)) {
    Refuse(name + " carries a tangent: the dense operators have no "
                  "forward-mode derivatives");
  }
}

// The tensor of an argument, on GPU `device` and of one of `types`.
const Tensor& AnyTensorOf(PyObject* o, const std::string& name, int device,
                          uint32_t types) {
  if (!THPVariable_Check(o)) {
    Refuse(name + " must be a torch tensor, got " + Py_TYPE(o)->tp_name);
  }
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != device) {
    Refuse(name + " must be on the current GPU, it is on " + Text(t.device()));
  }
  if (!(types & Bit(t.scalar_type()))) {
    Refuse(name + " must be one of " + TypeNames(types) + ", got " +
           Text(t.scalar_type()));
  }
  if (t.layout() != at::kStrided) Refuse(name + " must be a dense tensor");
  CheckTangent(t, name);
  return t;
}

// The same with its values in memory, for arguments that are read.
Tensor TensorOf(PyObject* o, const std::string& name, int device,
                uint32_t types) {
  const Tensor& t = AnyTensorOf(o, name, device, types);
  return HoldsValues(t) ? t : t.clone();
}

// The same for arguments that are written.
const Tensor& PlaceOf(PyObject* o, const std::string& name, int device,
                      uint32_t types) {
  const Tensor& t = AnyTensorOf(o, name, device, types);
  if (!HoldsValues(t) || !t.is_contiguous()) {
    Refuse(name + " must be contiguous and hold its values");
  }
  return t;
}

int32_t Code(at::ScalarType t) {
  return t == at::kFloat      ? SCEMB_F32
         : t == at::kBFloat16 ? SCEMB_BF16
                              : SCEMB_F16;
}

Tensor New(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  return at::empty(shape, like.options().dtype(type));
}

// A matrix of rows of `dim` neighbouring values, `stride` values apart (a copy
// where the tensor's strides allow no such view).
struct Rows {
  Tensor t;
  int64_t n;
  int64_t stride;
};
Rows RowsOf(const Tensor& x, int64_t dim) {
  Tensor t = x;
  if (t.dim() != 2) t = t.reshape({dim == 0 ? 0 : t.numel() / dim, dim});
  if (t.stride(1) != 1 && dim != 1) t = t.contiguous();
  return {t, t.size(0), t.stride(0)};
}

Tensor OptionalTensor(PyObject* o, const char* name, int device,
                      uint32_t types) {
  return o == Py_None ? Tensor() : TensorOf(o, name, device, types);
}

void* Data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* FloatData(const Tensor& t) { return static_cast<float*>(Data(t)); }

PyObject* Wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

PyObject* Tuple(std::initializer_list<Tensor> tensors) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (out == nullptr) throw Raised();
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) {
    PyObject* o = Wrap(t);
    if (o == nullptr) {
      Py_DECREF(out);
      throw Raised();
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

// A workspace of at least `bytes`, from the caller's function of a size. It is
// held until the work on it is enqueued.
Tensor Workspace(PyObject* get, size_t bytes) {
  PyObject* size = PyLong_FromSize_t(bytes);
  if (size == nullptr) throw Raised();
  PyObject* o = PyObject_CallOneArg(get, size);
  Py_DECREF(size);
  if (o == nullptr) throw Raised();
  const Tensor t = THPVariable_Check(o) ? THPVariable_Unpack(o) : Tensor();
  Py_DECREF(o);
  return t;
}

// ---------------------------------------------------------------------------
// Layer norm.
// ---------------------------------------------------------------------------

struct Affine {
  Tensor weight;
  Tensor bias;
};

Affine AffineOf(const Tensor& x, PyObject* weight, PyObject* bias, int dev) {
  if (x.dim() < 1 || x.size(-1) < 1) {
    Refuse("x must have a last dimension of at least 1, got shape " +
           Text(x.sizes()));
  }
  const uint32_t types = kF32 | Bit(x.scalar_type());
  Affine a{OptionalTensor(weight, "weight", dev, types),
           OptionalTensor(bias, "bias", dev, types)};
  const int64_t dim = x.size(-1);
  for (const auto& [p, name] : {std::make_pair(&a.weight, "weight"),
                                std::make_pair(&a.bias, "bias")}) {
    if (!p->defined()) continue;
    if (p->dim() != 1 || p->size(0) != dim) {
      Refuse(std::string(name) + " must have shape [" + std::to_string(dim) +
             "], got " + Text(p->sizes()));
    }
    *p = p->contiguous();
  }
  if (a.weight.defined() && a.bias.defined() &&
      a.weight.scalar_type() != a.bias.scalar_type()) {
    Refuse("weight and bias must be of one type, got " +
           Text(a.weight.scalar_type()) + " and " +
           Text(a.bias.scalar_type()));
  }
  return a;
}

// layer_norm(x, weight, bias, epsilon, stats) -> y or (y, mean, rstd)
PyObject* LayerNorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 5) Refuse("layer_norm takes 5 arguments");
    const int dev = CurrentDevice();
    const Tensor x = TensorOf(a[0], "x", dev, kRowTypes);
    const Affine p = AffineOf(x, a[1], a[2], dev);
    const double epsilon = Float(a[3]);
    if (!(epsilon >= 0)) {
      Refuse("epsilon must not be negative, got " + Text(epsilon));
    }
    const bool stats = a[4] == Py_True;
    const int64_t dim = x.size(-1);
    const Rows r = RowsOf(x, dim);
    const Tensor y = New(x.sizes(), x.scalar_type(), x);
    Tensor mean, rstd;
    if (stats) {
      const auto shape = x.sizes().slice(0, x.dim() - 1);
      mean = New(shape, at::kFloat, x);
      rstd = New(shape, at::kFloat, x);
    }
    const Tensor& w = p.weight.defined() ? p.weight : p.bias;
    Check(lib.layer_norm(
        r.t.data_ptr(), Code(x.scalar_type()), r.n, dim, r.stride,
        Data(p.weight), Data(p.bias),
        w.defined() ? Code(w.scalar_type()) : SCEMB_F32,
        static_cast<float>(epsilon), y.data_ptr(), FloatData(mean),
        FloatData(rstd), Stream(dev)));
    return stats ? Tuple({y, mean, rstd}) : Wrap(y);
  });
}

// layer_norm_grad(y_grad, x, mean, rstd, weight, want_weight, want_bias,
//                 bias_f32, workspace) -> (dx, dweight, dbias)
// bias_f32: the bias's type where there is no weight to say it (float32 or
// x's).
PyObject* LayerNormGrad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 9) Refuse("layer_norm_grad takes 9 arguments");
    const int dev = CurrentDevice();
    const Tensor x = TensorOf(a[1], "x", dev, kRowTypes);
    const Affine p = AffineOf(x, a[4], Py_None, dev);
    const Tensor dy = TensorOf(a[0], "y_grad", dev, Bit(x.scalar_type()));
    if (dy.sizes() != x.sizes()) {
      Refuse("y_grad must have x's shape " + Text(x.sizes()) + ", got " +
             Text(dy.sizes()));
    }
    const int64_t dim = x.size(-1);
    Tensor stats[2];
    for (int i = 0; i < 2; ++i) {
      const char* name = i == 0 ? "mean" : "rstd";
      const Tensor s = TensorOf(a[2 + i], name, dev, kF32);
      if (s.numel() * dim != x.numel()) {
        Refuse(std::string(name) + " must have a value for each row of x, got "
               "shape " + Text(s.sizes()));
      }
      stats[i] = s.contiguous();
    }
    const auto type = p.weight.defined() ? p.weight.scalar_type()
                      : a[7] == Py_True  ? at::kFloat
                                         : x.scalar_type();
    const Rows r = RowsOf(x, dim);
    const Rows g = RowsOf(dy, dim);
    const Tensor dx = New(x.sizes(), x.scalar_type(), x);
    Tensor dw, db;
    if (a[5] == Py_True && p.weight.defined()) dw = New({dim}, type, x);
    if (a[6] == Py_True) db = New({dim}, type, x);
    const int32_t code = Code(x.scalar_type());
    Tensor ws;
    size_t bytes = 0;
    if (dw.defined() || db.defined()) {
      bytes = lib.layer_norm_grad_workspace(code, r.n, dim);
      if (bytes == 0) Check(SCEMB_ERR_INVALID_ARGUMENT);
      ws = Workspace(a[8], bytes);
    }
    Check(lib.layer_norm_grad(
        g.t.data_ptr(), g.stride, r.t.data_ptr(), r.stride, code, r.n, dim,
        FloatData(stats[0]), FloatData(stats[1]), Data(p.weight), Code(type),
        dx.data_ptr(), Data(dw), Data(db), Data(ws), bytes, Stream(dev)));
    return Tuple({dx, dw, db});
  });
}

// ---------------------------------------------------------------------------
// Tokens and experts.
// ---------------------------------------------------------------------------

// sort_by_expert(ids, num_experts, workspace)
//   -> (positions, sources, offsets)
PyObject* SortByExpert(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 3) Refuse("sort_by_expert takes 3 arguments");
    const int dev = CurrentDevice();
    const Tensor ids = TensorOf(a[0], "expert_ids", dev, kI32 | kI64);
    if (ids.dim() != 1 && ids.dim() != 2) {
      Refuse("expert_ids must have shape [tokens, choices] or [tokens], got " +
             Text(ids.sizes()));
    }
    const int64_t experts = Int(a[1]);
    if (experts < 1 || experts > SCEMB_MAX_EXPERTS) {
      Refuse("num_experts must be within [1, " +
             std::to_string(SCEMB_MAX_EXPERTS) + "], got " + Text(experts));
    }
    const int64_t count = ids.numel();
    if (count > 0x7fffffff) {
      Refuse("at most 2^31 - 1 choices can be ordered, got " + Text(count));
    }
    const Tensor in = ids.contiguous();
    const Tensor positions = New(ids.sizes(), at::kInt, ids);
    const Tensor sources = New({count}, at::kInt, ids);
    const Tensor offsets = New({experts + 1}, at::kInt, ids);
    const int32_t e = static_cast<int32_t>(experts);
    const size_t bytes = lib.sort_by_expert_workspace(count, e);
    const Tensor ws = bytes > 0 ? Workspace(a[2], bytes) : Tensor();
    Check(lib.sort_by_expert(
        in.data_ptr(), static_cast<int32_t>(in.element_size()), count, e,
        static_cast<int32_t*>(positions.data_ptr()),
        static_cast<int32_t*>(sources.data_ptr()),
        static_cast<int32_t*>(offsets.data_ptr()), Data(ws), bytes,
        Stream(dev)));
    return Tuple({positions, sources, offsets});
  });
}

struct OrderOf {
  Tensor positions;
  Tensor offsets;
  scemb_expert_order_t order;

  OrderOf(PyObject* p, PyObject* o, int dev)
      : positions(TensorOf(p, "order.positions", dev, kI32)),
        offsets(TensorOf(o, "order.offsets", dev, kI32)) {
    if ((positions.dim() != 1 && positions.dim() != 2) ||
        (positions.dim() == 2 && positions.size(1) < 1)) {
      Refuse("order.positions must have shape [tokens, choices] or [tokens], "
             "got " + Text(positions.sizes()));
    }
    if (offsets.dim() != 1 || offsets.size(0) < 2 ||
        offsets.size(0) > SCEMB_MAX_EXPERTS + 1) {
      Refuse("order.offsets must have shape [num_experts + 1], got " +
             Text(offsets.sizes()));
    }
    positions = positions.contiguous();
    offsets = offsets.contiguous();
    const int64_t choices = positions.dim() == 1 ? 1 : positions.size(1);
    if (choices > 0x7fffffff) Refuse("order.positions has too many choices");
    order = {static_cast<const int32_t*>(positions.data_ptr()),
             static_cast<const int32_t*>(offsets.data_ptr()),
             positions.size(0), static_cast<int32_t>(choices),
             static_cast<int32_t>(offsets.size(0) - 1)};
  }
};

Tensor RowsArg(PyObject* o, const char* name, int64_t n, int dev,
                      uint32_t types) {
  const Tensor x = TensorOf(o, name, dev, types);
  if (x.dim() != 2 || x.size(0) != n || x.size(1) < 1) {
    Refuse(std::string(name) + " must have shape [" + std::to_string(n) +
           ", dim], got " + Text(x.sizes()));
  }
  return x;
}

Tensor WeightsArg(PyObject* o, const OrderOf& order, const Tensor& rows,
                  int dev) {
  const Tensor w =
      OptionalTensor(o, "weights", dev, kF32 | Bit(rows.scalar_type()));
  if (w.defined() && w.sizes() != order.positions.sizes()) {
    Refuse("weights must have the shape of the ids, " +
           Text(order.positions.sizes()) + ", got " + Text(w.sizes()));
  }
  return w.defined() ? w.contiguous() : w;
}

int32_t WeightsCode(const Tensor& w) {
  return w.defined() ? Code(w.scalar_type()) : SCEMB_F32;
}

// tokens_to_experts(x, positions, offsets) -> rows
PyObject* TokensToExperts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 3) Refuse("tokens_to_experts takes 3 arguments");
    const int dev = CurrentDevice();
    const OrderOf o(a[1], a[2], dev);
    const Tensor x = RowsArg(a[0], "x", o.positions.size(0), dev, kRowTypes);
    const int64_t dim = x.size(1);
    const Rows r = RowsOf(x, dim);
    const Tensor rows = New({o.positions.numel(), dim}, x.scalar_type(), x);
    Check(lib.tokens_to_experts(r.t.data_ptr(), Code(x.scalar_type()),
                                r.stride, dim, &o.order, rows.data_ptr(),
                                Stream(dev)));
    return Wrap(rows);
  });
}

// tokens_from_experts(rows, weights, positions, offsets, name) -> y
PyObject* TokensFromExperts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 5) Refuse("tokens_from_experts takes 5 arguments");
    const int dev = CurrentDevice();
    const OrderOf o(a[2], a[3], dev);
    const char* name = PyUnicode_AsUTF8(a[4]);
    if (name == nullptr) throw Raised();
    const Tensor rows =
        RowsArg(a[0], name, o.positions.numel(), dev, kRowTypes);
    const Tensor w = WeightsArg(a[1], o, rows, dev);
    const int64_t dim = rows.size(1);
    const Rows r = RowsOf(rows, dim);
    const Tensor y =
        New({o.positions.size(0), dim}, rows.scalar_type(), rows);
    Check(lib.tokens_from_experts(r.t.data_ptr(), Code(rows.scalar_type()),
                                  r.stride, dim, Data(w), WeightsCode(w),
                                  &o.order, y.data_ptr(), Stream(dev)));
    return Wrap(y);
  });
}

// tokens_from_experts_grad(y_grad, rows, weights, positions, offsets)
//   -> (drows, dweights)
PyObject* TokensFromExpertsGrad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 5) Refuse("tokens_from_experts_grad takes 5 arguments");
    const int dev = CurrentDevice();
    const OrderOf o(a[3], a[4], dev);
    const Tensor rows =
        RowsArg(a[1], "rows", o.positions.numel(), dev, kRowTypes);
    const Tensor w = WeightsArg(a[2], o, rows, dev);
    const int64_t dim = rows.size(1);
    const Tensor dy = TensorOf(a[0], "y_grad", dev, Bit(rows.scalar_type()));
    if (dy.dim() != 2 || dy.size(0) != o.positions.size(0) ||
        dy.size(1) != dim) {
      Refuse("y_grad must have shape [" + std::to_string(o.positions.size(0)) +
             ", " + std::to_string(dim) + "], got " + Text(dy.sizes()));
    }
    const Rows r = RowsOf(rows, dim);
    const Rows g = RowsOf(dy, dim);
    const Tensor drows = New(rows.sizes(), rows.scalar_type(), rows);
    Tensor dweights;
    if (w.defined()) dweights = New(w.sizes(), w.scalar_type(), w);
    Check(lib.tokens_from_experts_grad(
        g.t.data_ptr(), g.stride, r.t.data_ptr(), Code(rows.scalar_type()),
        r.stride, dim, Data(w), WeightsCode(w), &o.order, drows.data_ptr(),
        Data(dweights), Stream(dev)));
    return Tuple({drows, dweights});
  });
}

// ---------------------------------------------------------------------------
// The experts' products.
// ---------------------------------------------------------------------------

Tensor OffsetsArg(PyObject* o, int dev) {
  const Tensor t = TensorOf(o, "order.offsets", dev, kI32);
  if (t.dim() != 1 || t.size(0) < 2 || t.size(0) > SCEMB_MAX_EXPERTS + 1) {
    Refuse("order.offsets must have shape [num_experts + 1], got " +
           Text(t.sizes()));
  }
  return t.contiguous();
}

// The strides of weights [experts, inner, outer] that are contiguous along inner
// or outer; others are copied first.
struct WeightStrides {
  int64_t expert;
  int64_t inner;
  int64_t outer;

  explicit WeightStrides(Tensor* t) {
    const int64_t i = t->size(1), o = t->size(2);
    if ((i > 1 && o > 1 && t->stride(1) != 1 && t->stride(2) != 1) ||
        (i == 1 && t->stride(2) != 1) || (o == 1 && t->stride(1) != 1)) {
      *t = t->contiguous();
    }
    expert = t->stride(0);
    // The stride of a dimension of one value says nothing.
    outer = o == 1 ? (i == 1 ? 1 : i) : t->stride(2);
    inner = i == 1 ? (o == 1 ? 1 : o) : t->stride(1);
  }
};

// The experts' weights, [experts, inner, outer].
struct ExpertWeights {
  Tensor t;
  int64_t experts;
  int64_t inner;
  int64_t outer;
  std::optional<WeightStrides> stride;

  ExpertWeights(PyObject* o, const Tensor& offsets, const Tensor& rows,
                int dev)
      : t(TensorOf(o, "weights", dev, Bit(rows.scalar_type()))) {
    experts = offsets.size(0) - 1;
    if (t.dim() != 3 || t.size(0) != experts || t.size(1) < 1 ||
        t.size(2) < 1) {
      Refuse("weights must have shape [" + std::to_string(experts) +
             ", inner, outer], got " + Text(t.sizes()));
    }
    inner = t.size(1);
    outer = t.size(2);
    stride.emplace(&t);
  }
  // Stored by output: the gradient is laid out the same.
  bool ByOuter() const { return stride->outer != 1; }
};

Tensor MatrixArg(PyObject* o, const char* name, const Tensor& like,
                 int64_t rows, int64_t columns, int dev) {
  const Tensor x = TensorOf(o, name, dev, Bit(like.scalar_type()));
  if (x.dim() != 2 || x.size(0) != rows || x.size(1) != columns) {
    Refuse(std::string(name) + " must have shape [" + std::to_string(rows) +
           ", " + std::to_string(columns) + "], got " + Text(x.sizes()));
  }
  return x;
}

Tensor ExpertRows(PyObject* o, int dev) {
  const Tensor x = TensorOf(o, "rows", dev, kRowTypes);
  if (x.dim() != 2 || x.size(1) < 1) {
    Refuse("rows must have shape [choices, inner], got " + Text(x.sizes()));
  }
  return x;
}

void CheckInner(const ExpertWeights& w, const Tensor& rows) {
  if (w.inner != rows.size(1)) {
    Refuse("weights must have shape [experts, " + Text(rows.size(1)) +
           ", outer] for these rows, got " + Text(w.t.sizes()));
  }
}

// rows * weights, or with `turned` rows * the weights' transpose.
Tensor Product(const Rows& r, const ExpertWeights& w, bool turned,
               const Tensor& offsets, PyObject* workspace, int dev) {
  const int64_t inner = turned ? w.outer : w.inner;
  const int64_t outer = turned ? w.inner : w.outer;
  const int32_t code = Code(r.t.scalar_type());
  const int32_t experts = static_cast<int32_t>(w.experts);
  const Tensor y = New({r.n, outer}, r.t.scalar_type(), r.t);
  const size_t bytes =
      lib.expert_matmul_workspace(code, r.n, inner, outer, experts);
  const Tensor ws = bytes > 0 ? Workspace(workspace, bytes) : Tensor();
  Check(lib.expert_matmul(
      r.t.data_ptr(), code, r.stride, r.n, inner, outer, w.t.data_ptr(),
      w.stride->expert, turned ? w.stride->outer : w.stride->inner,
      turned ? w.stride->inner : w.stride->outer,
      static_cast<const int32_t*>(offsets.data_ptr()), experts, y.data_ptr(),
      Data(ws), bytes, Stream(dev)));
  return y;
}

// expert_matmul(rows, weights, offsets, workspace) -> y
PyObject* ExpertMatmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 4) Refuse("expert_matmul takes 4 arguments");
    const int dev = CurrentDevice();
    const Tensor x = ExpertRows(a[0], dev);
    const Tensor offsets = OffsetsArg(a[2], dev);
    const ExpertWeights w(a[1], offsets, x, dev);
    CheckInner(w, x);
    return Wrap(Product(RowsOf(x, w.inner), w, false, offsets, a[3], dev));
  });
}

// expert_matmul_grad(y_grad, rows, weights, offsets, want_rows, want_weights,
//                    workspace) -> (drows, dweights)
PyObject* ExpertMatmulGrad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 7) Refuse("expert_matmul_grad takes 7 arguments");
    const int dev = CurrentDevice();
    const Tensor x = ExpertRows(a[1], dev);
    const Tensor offsets = OffsetsArg(a[3], dev);
    const ExpertWeights w(a[2], offsets, x, dev);
    CheckInner(w, x);
    const Tensor dy = MatrixArg(a[0], "y_grad", x, x.size(0), w.outer, dev);
    const Rows g = RowsOf(dy, w.outer);
    const auto* first = static_cast<const int32_t*>(offsets.data_ptr());
    const int32_t code = Code(x.scalar_type());
    const int32_t experts = static_cast<int32_t>(w.experts);
    Tensor drows, dw;
    if (a[4] == Py_True) drows = Product(g, w, true, offsets, a[6], dev);
    if (a[5] == Py_True) {
      const Rows r = RowsOf(x, w.inner);
      // The transposed gradient is that of the operands changed about.
      const bool turned = w.ByOuter();
      const Rows& left = turned ? g : r;
      const Rows& right = turned ? r : g;
      const int64_t inner = turned ? w.outer : w.inner;
      const int64_t outer = turned ? w.inner : w.outer;
      dw = New({w.experts, inner, outer}, x.scalar_type(), x);
      const size_t bytes = lib.expert_matmul_weights_grad_workspace(
          code, r.n, inner, outer, experts);
      const Tensor ws = bytes > 0 ? Workspace(a[6], bytes) : Tensor();
      Check(lib.expert_matmul_weights_grad(
          left.t.data_ptr(), left.stride, right.t.data_ptr(), right.stride,
          code, r.n, inner, outer, first, experts, dw.data_ptr(), Data(ws),
          bytes, Stream(dev)));
      if (turned) dw = dw.transpose(1, 2);
    }
    return Tuple({drows, dw});
  });
}

// quantize_weights(weights) -> (codes, exponents)
PyObject* QuantizeWeights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 1) Refuse("quantize_weights takes 1 argument");
    const int dev = CurrentDevice();
    Tensor w = TensorOf(a[0], "weights", dev, kRowTypes);
    if ((w.dim() != 2 && w.dim() != 3) || w.numel() == 0 ||
        (w.dim() == 3 && w.size(0) > SCEMB_MAX_EXPERTS)) {
      Refuse("weights must have shape [inner, outer] or [experts, inner, "
             "outer], none 0 and at most " +
             std::to_string(SCEMB_MAX_EXPERTS) + " experts, got " +
             Text(w.sizes()));
    }
    const bool single = w.dim() == 2;
    if (single) w = w.unsqueeze(0);
    const int64_t experts = w.size(0), inner = w.size(1), outer = w.size(2);
    const WeightStrides stride(&w);
    const auto blocks = [](int64_t v) {
      return (v + SCEMB_BLOCK_8BIT - 1) / SCEMB_BLOCK_8BIT;
    };
    Tensor codes = New({experts, outer, blocks(inner) * SCEMB_BLOCK_8BIT},
                       at::kFloat8_e4m3fn, w);
    Tensor exponents =
        New({experts, blocks(outer), blocks(inner)}, at::kInt, w);
    Check(lib.quantize_weights(
        w.data_ptr(), Code(w.scalar_type()), stride.expert, stride.inner,
        stride.outer, inner, outer, static_cast<int32_t>(experts),
        static_cast<uint8_t*>(codes.data_ptr()),
        static_cast<int32_t*>(exponents.data_ptr()), Stream(dev)));
    if (single) {
      codes = codes.squeeze(0);
      exponents = exponents.squeeze(0);
    }
    return Tuple({codes, exponents});
  });
}

// matmul_8bit(rows, codes, exponents, inner, offsets or None, workspace) -> y
PyObject* Matmul8bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 6) Refuse("matmul_8bit takes 6 arguments");
    const int dev = CurrentDevice();
    const Tensor x = ExpertRows(a[0], dev);
    const int64_t inner = Int(a[3]);
    if (x.size(1) != inner) {
      Refuse("rows must have shape [rows, " + std::to_string(inner) +
             "] for these weights, got " + Text(x.sizes()));
    }
    const bool grouped = a[4] != Py_None;
    Tensor codes =
        TensorOf(a[1], "weights.codes", dev, Bit(at::kFloat8_e4m3fn));
    Tensor exponents = TensorOf(a[2], "weights.exponents", dev, kI32);
    const Tensor offsets = grouped ? OffsetsArg(a[4], dev) : Tensor();
    const int64_t experts = grouped ? offsets.size(0) - 1 : 1;
    const int64_t blocks = (inner + SCEMB_BLOCK_8BIT - 1) / SCEMB_BLOCK_8BIT;
    const int64_t d = grouped ? 3 : 2;
    const bool fits =
        codes.dim() == d && exponents.dim() == d &&
        (!grouped || (codes.size(0) == experts &&
                      exponents.size(0) == experts)) &&
        codes.size(-1) == blocks * SCEMB_BLOCK_8BIT && codes.size(-2) > 0 &&
        exponents.size(-1) == blocks &&
        exponents.size(-2) ==
            (codes.size(-2) + SCEMB_BLOCK_8BIT - 1) / SCEMB_BLOCK_8BIT;
    if (!fits) {
      Refuse(std::string(grouped ? "weights must be of as many experts as the "
                                   "order's, "
                                 : "weights of several experts need an order, "
                                   "and others have none, ") +
             "got codes of shape " + Text(codes.sizes()) +
             " and exponents of shape " + Text(exponents.sizes()));
    }
    codes = codes.contiguous();
    exponents = exponents.contiguous();
    if (reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 != 0) {
      codes = codes.clone();
    }
    const int64_t outer = codes.size(-2);
    const Rows r = RowsOf(x, inner);
    const Tensor y = New({r.n, outer}, x.scalar_type(), x);
    const size_t bytes = lib.matmul_8bit_workspace(r.n, inner);
    if (bytes == 0) Check(SCEMB_ERR_INVALID_ARGUMENT);
    const Tensor ws = Workspace(a[5], bytes);
    Check(lib.matmul_8bit(
        r.t.data_ptr(), Code(x.scalar_type()), r.stride, r.n, inner, outer,
        static_cast<const uint8_t*>(codes.data_ptr()),
        static_cast<const int32_t*>(exponents.data_ptr()),
        static_cast<const int32_t*>(Data(offsets)),
        static_cast<int32_t>(experts), y.data_ptr(), Data(ws), bytes,
        Stream(dev)));
    return Wrap(y);
  });
}

// ---------------------------------------------------------------------------
// AdamW.
// ---------------------------------------------------------------------------

// A list or tuple of tensors (or None).
struct Sequence {
  PyObject* fast;
  Py_ssize_t n;
  Sequence(PyObject* o, const char* what)
      : fast(PySequence_Fast(o, what)),
        n(fast != nullptr ? PySequence_Fast_GET_SIZE(fast) : 0) {
    if (fast == nullptr) throw Raised();
  }
  ~Sequence() { Py_XDECREF(fast); }
  Sequence(const Sequence&) = delete;
  PyObject* operator[](Py_ssize_t i) const {
    return PySequence_Fast_GET_ITEM(fast, i);
  }
};

std::string At(const char* name, Py_ssize_t i) {
  return std::string(name) + "[" + std::to_string(i) + "]";
}

// Whether an element is a contiguous tensor that fits. If not, TensorOf and
// PlaceOf say why, or make one, with a name that is only made for them.
bool Fits(PyObject* o, int dev, uint32_t types) {
  if (!THPVariable_Check(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == dev &&
         (types & Bit(t.scalar_type())) && t.layout() == at::kStrided &&
         HoldsValues(t) && t.is_contiguous() && !HasTangent(t);
}

const Tensor& ElementOf(PyObject* o, const char* name, Py_ssize_t i, int dev,
                        uint32_t types) {
  return Fits(o, dev, types) ? THPVariable_Unpack(o)
                             : PlaceOf(o, At(name, i), dev, types);
}

const Tensor& ParamOf(PyObject* o, Py_ssize_t i, int dev) {
  return ElementOf(o, "params", i, dev, kF32 | kBf16);
}

// adamw_sizes(params) -> list of their numbers of values
PyObject* AdamwSizes(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 1) Refuse("adamw_sizes takes 1 argument");
    const int dev = CurrentDevice();
    const Sequence params(a[0], "params must be a sequence of tensors");
    PyObject* out = PyList_New(params.n);
    if (out == nullptr) throw Raised();
    try {
      for (Py_ssize_t i = 0; i < params.n; ++i) {
        PyList_SET_ITEM(out, i, PyLong_FromLongLong(
                                    ParamOf(params[i], i, dev).numel()));
      }
    } catch (...) {
      Py_DECREF(out);
      throw;
    }
    return out;
  });
}

scemb_adamw_state_t StateOf(PyObject* m, PyObject* v, PyObject* m_scale,
                            PyObject* v_scale, PyObject* scratch, int dev) {
  const bool bits8 = m_scale != Py_None;
  const auto one = [&](PyObject* o, const char* name,
                       at::ScalarType type) -> const Tensor& {
    return PlaceOf(o, name, dev, Bit(type));
  };
  const Tensor& tm = one(m, "state.m", bits8 ? at::kChar : at::kFloat);
  const Tensor& tv = one(v, "state.v", bits8 ? at::kByte : at::kFloat);
  scemb_adamw_state_t s = {};
  s.m = tm.data_ptr();
  s.v = tv.data_ptr();
  s.size = tm.numel();
  s.bits = bits8 ? 8 : 32;
  bool sizes = tv.numel() == s.size;
  if (bits8) {
    const Tensor& ms = one(m_scale, "state.m_scale", at::kFloat);
    const Tensor& vs = one(v_scale, "state.v_scale", at::kFloat);
    s.m_scale = FloatData(ms);
    s.v_scale = FloatData(vs);
    sizes = sizes && ms.numel() * SCEMB_ADAMW_BLOCK == s.size &&
            vs.numel() == ms.numel();
  }
  if (scratch != Py_None) {
    const Tensor& t = one(scratch, "state.scratch", at::kFloat);
    sizes = sizes && t.numel() >= 4;
    s.scratch = FloatData(t);
  }
  if (!sizes) Refuse("the state's tensors are not of matching sizes");
  return s;
}

// Bytes [first, second) of memory.
using Spans = std::vector<std::pair<uintptr_t, uintptr_t>>;

void AddSpan(Spans* spans, const void* p, int64_t bytes) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  spans->emplace_back(at, at + static_cast<uintptr_t>(bytes));
}

// Two tensors that share memory would be written by two work-groups at once.
void CheckApart(Spans* spans, const char* what) {
  std::sort(spans->begin(), spans->end());
  for (size_t i = 1; i < spans->size(); ++i) {
    if ((*spans)[i].first < (*spans)[i - 1].second) {
      Refuse(std::string("two ") + what + " share memory");
    }
  }
}

void CheckApart(const std::vector<scemb_adamw_tensor_t>& tensors) {
  Spans spans;
  spans.reserve(2 * tensors.size());
  for (const auto& t : tensors) {
    if (t.numel == 0) continue;
    AddSpan(&spans, t.param, t.numel * (t.param_type == SCEMB_F32 ? 4 : 2));
    if (t.copy != nullptr) AddSpan(&spans, t.copy, t.numel * 2);
  }
  CheckApart(&spans, "params or copies");
}

// Autograd is told of a write: a backward pass that needs the old values raises.
void Written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// adamw_scalar(x, is_int) -> x, a tensor of one value on a GPU, as a tensor on
// the current GPU whose memory holds it as float32 or int64 (x itself if it
// does).
PyObject* AdamwScalar(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 2 || !THPVariable_Check(a[0])) {
      Refuse("adamw_scalar takes a tensor and its kind");
    }
    const Tensor& x = THPVariable_Unpack(a[0]);
    if (x.numel() != 1) {
      Refuse("a hyperparameter on the GPU must be one value, got shape " +
             Text(x.sizes()));
    }
    CheckTangent(x, "a hyperparameter");
    const auto type = a[1] == Py_True ? at::kLong : at::kFloat;
    const int dev = CurrentDevice();
    if (x.scalar_type() == type && x.get_device() == dev && HoldsValues(x)) {
      return Py_NewRef(a[0]);
    }
    const Tensor t = x.to(at::TensorOptions(type).device(at::kCUDA, dev));
    return Wrap(HoldsValues(t) ? t : t.clone());
  });
}

// adamw_update(params, grads, copies, layout, m, v, m_scale, v_scale, scratch,
//              learning_rate, beta_1, beta_2, epsilon, weight_decay,
//              grad_scale, step, learning_rate_ptr, step_ptr, grad_scale_ptr)
// layout: bytes of scemb_adamw_tensor_t, of which numel and decay are set.
PyObject* AdamwUpdate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 19) Refuse("adamw_update takes 19 arguments");
    const int dev = CurrentDevice();
    const Sequence params(a[0], "params must be a sequence of tensors");
    const Sequence grads(a[1], "grads must be a sequence of tensors");
    char* bytes = nullptr;
    Py_ssize_t size = 0;
    if (PyBytes_AsStringAndSize(a[3], &bytes, &size) != 0) throw Raised();
    const Py_ssize_t count =
        size / static_cast<Py_ssize_t>(sizeof(scemb_adamw_tensor_t));
    if (params.n != count || grads.n != count) {
      Refuse(std::to_string(params.n) + " params and " +
             std::to_string(grads.n) + " grads for a state of " +
             std::to_string(count));
    }
    std::vector<scemb_adamw_tensor_t> tensors(count);
    if (count > 0) std::memcpy(tensors.data(), bytes, size);
    std::vector<Tensor> keep;
    for (Py_ssize_t i = 0; i < count; ++i) {
      scemb_adamw_tensor_t& t = tensors[i];
      const Tensor& p = ParamOf(params[i], i, dev);
      if (p.numel() != t.numel) {
        Refuse("the state was made for weights of other sizes: " +
               At("params", i) + " has " + Text(p.numel()) +
               " values instead of " + Text(t.numel));
      }
      t.param = p.data_ptr();
      t.param_type = Code(p.scalar_type());
      if (grads[i] != Py_None) {
        constexpr uint32_t kTypes = kF32 | kBf16;
        const bool fits = Fits(grads[i], dev, kTypes);
        if (!fits) {
          keep.push_back(
              TensorOf(grads[i], At("grads", i), dev, kTypes).contiguous());
        }
        const Tensor& g = fits ? THPVariable_Unpack(grads[i]) : keep.back();
        if (g.sizes() != p.sizes()) {
          Refuse(At("grads", i) + " must have the shape " + Text(p.sizes()) +
                 " of its weight, got " + Text(g.sizes()));
        }
        t.grad_type = Code(g.scalar_type());
        t.grad = g.data_ptr();
      }
    }
    std::optional<Sequence> copies;
    if (a[2] != Py_None) {
      copies.emplace(a[2], "copies must be a sequence of tensors");
      if (copies->n != count) {
        Refuse(std::to_string(copies->n) + " copies for " +
               std::to_string(count) + " params");
      }
      for (Py_ssize_t i = 0; i < count; ++i) {
        if ((*copies)[i] == Py_None) continue;
        const Tensor& c = ElementOf((*copies)[i], "copies", i, dev, kBf16);
        const Tensor& p = THPVariable_Unpack(params[i]);
        if (c.sizes() != p.sizes()) {
          Refuse(At("copies", i) + " must have the shape " + Text(p.sizes()) +
                 " of its weight, got " + Text(c.sizes()));
        }
        // A bfloat16 weight's own tensor is its copy already.
        if (p.scalar_type() == at::kFloat ||
            c.data_ptr() != tensors[i].param) {
          tensors[i].copy = c.data_ptr();
        }
      }
    }
    CheckApart(tensors);
    const scemb_adamw_state_t state =
        StateOf(a[4], a[5], a[6], a[7], a[8], dev);
    scemb_adamw_options_t o = {};
    o.learning_rate = Float(a[9]);
    o.beta_1 = Float(a[10]);
    o.beta_2 = Float(a[11]);
    o.epsilon = Float(a[12]);
    o.weight_decay = Float(a[13]);
    o.grad_scale = Float(a[14]);
    o.step = Int(a[15]);
    o.learning_rate_ptr = static_cast<const float*>(Address(a[16]));
    o.step_ptr = static_cast<const int64_t*>(Address(a[17]));
    o.grad_scale_ptr = static_cast<const float*>(Address(a[18]));
    Check(lib.adamw_update(tensors.data(), static_cast<int32_t>(count), &state,
                           &o, Stream(dev)));
    for (Py_ssize_t i = 0; i < count; ++i) {
      if (tensors[i].grad == nullptr) continue;
      Written(THPVariable_Unpack(params[i]));
      if (tensors[i].copy != nullptr) {
        Written(THPVariable_Unpack((*copies)[i]));
      }
    }
    Py_RETURN_NONE;
  });
}

// adamw_moments(m, v, m_scale, v_scale) -> (m, v)
PyObject* AdamwMoments(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 4) Refuse("adamw_moments takes 4 arguments");
    const int dev = CurrentDevice();
    const scemb_adamw_state_t state =
        StateOf(a[0], a[1], a[2], a[3], Py_None, dev);
    const Tensor& like = THPVariable_Unpack(a[0]);
    const Tensor m = New({state.size}, at::kFloat, like);
    const Tensor v = New({state.size}, at::kFloat, like);
    Check(lib.adamw_moments(&state, FloatData(m), FloatData(v),
                            Stream(dev)));
    return Tuple({m, v});
  });
}

// ---------------------------------------------------------------------------
// The gradients' norm.
// ---------------------------------------------------------------------------

// Gradients as the library takes them; those that are None are left out. A
// tensor without gaps is taken as it lies in memory, whatever its strides. With
// `write` it has to be such a tensor, else a copy is.
struct Gradients {
  std::vector<scemb_gradient_t> list;
  std::vector<Tensor> keep;

  Gradients(const Sequence& grads, int dev, bool write) {
    list.reserve(grads.n);
    const bool recorded = at::GradMode::is_enabled();
    for (Py_ssize_t i = 0; i < grads.n; ++i) {
      if (grads[i] == Py_None) continue;
      const bool fits = Fits(grads[i], dev, kRowTypes);
      if (!fits) {
        const Tensor& t = AnyTensorOf(grads[i], At("grads", i), dev, kRowTypes);
        const bool whole = t.is_non_overlapping_and_dense();
        if (write && !(whole && HoldsValues(t))) {
          Refuse(At("grads", i) + " must have no gaps in memory and hold its "
                                  "values");
        }
        // A negated view has the same squares.
        keep.push_back(t._is_zerotensor() ? t.clone()
                       : whole            ? t
                                          : t.contiguous());
      }
      // Autograd would take what comes out for constants.
      if (recorded && THPVariable_Unpack(grads[i]).requires_grad()) {
        Refuse(At("grads", i) + " takes part in a graph that the norm does not "
                                "follow: call under torch.no_grad(), or "
                                "detach it");
      }
      const Tensor& t = fits ? THPVariable_Unpack(grads[i]) : keep.back();
      list.push_back({t.numel() > 0 ? t.data_ptr() : nullptr, t.numel(),
                      Code(t.scalar_type()), 0});
    }
  }
  int32_t size() const { return static_cast<int32_t>(list.size()); }
};

double LimitOf(PyObject* max_norm) {
  const double limit = Float(max_norm);
  if (!(limit >= 0)) {
    Refuse("max_norm must not be negative, got " + Text(limit));
  }
  return limit;
}

Tensor NormWorkspace(const Gradients& g, PyObject* get, size_t* bytes) {
  *bytes = lib.gradient_norm_workspace(g.list.data(), g.size());
  if (*bytes == 0) Check(SCEMB_ERR_INVALID_ARGUMENT);
  return Workspace(get, *bytes);
}

Tensor Single(int dev) {
  return at::empty({}, at::TensorOptions(at::kFloat).device(at::kCUDA, dev));
}

// gradient_norm(grads, max_norm, workspace) -> (norm, factor)
PyObject* GradientNorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 3) Refuse("gradient_norm takes 3 arguments");
    const int dev = CurrentDevice();
    const Sequence grads(a[0], "grads must be a sequence of tensors");
    const Gradients g(grads, dev, false);
    const bool limited = a[1] != Py_None;
    const double limit = limited ? LimitOf(a[1]) : 0.0;
    const Tensor norm = Single(dev);
    const Tensor factor = limited ? Single(dev) : Tensor();
    size_t bytes = 0;
    const Tensor ws = NormWorkspace(g, a[2], &bytes);
    Check(lib.gradient_norm(g.list.data(), g.size(), limit, FloatData(norm),
                            FloatData(factor), Data(ws), bytes, Stream(dev)));
    return Tuple({norm, factor});
  });
}

// clip_gradients(grads, max_norm, workspace) -> norm
PyObject* ClipGradients(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject* {
    if (n != 3) Refuse("clip_gradients takes 3 arguments");
    const int dev = CurrentDevice();
    const Sequence grads(a[0], "grads must be a sequence of tensors");
    const Gradients g(grads, dev, true);
    Spans spans;
    spans.reserve(g.list.size());
    for (const auto& t : g.list) {
      if (t.numel > 0) {
        AddSpan(&spans, t.data, t.numel * (t.type == SCEMB_F32 ? 4 : 2));
      }
    }
    CheckApart(&spans, "grads");
    if (a[1] == Py_None) Refuse("max_norm must be a number");
    const double limit = LimitOf(a[1]);
    const Tensor norm = Single(dev);
    size_t bytes = 0;
    const Tensor ws = NormWorkspace(g, a[2], &bytes);
    Check(lib.clip_gradients(g.list.data(), g.size(), limit, FloatData(norm),
                             Data(ws), bytes, Stream(dev)));
    for (Py_ssize_t i = 0; i < grads.n; ++i) {
      if (grads[i] != Py_None) Written(THPVariable_Unpack(grads[i]));
    }
    return Wrap(norm);
  });
}

// ---------------------------------------------------------------------------
// The module.
// ---------------------------------------------------------------------------

// bind(addresses, raw_stream): the library's functions, in the order of
// Library, and a function from a device's index to its current stream's handle.
PyObject* Bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 2 || !PyCallable_Check(a[1])) {
      PyErr_SetString(PyExc_ValueError, "bind takes addresses and a function");
      return nullptr;
    }
    const Sequence s(a[0], "bind takes a sequence of addresses");
    constexpr Py_ssize_t kCount = sizeof(Library) / sizeof(void*);
    void* p[kCount];
    if (s.n != kCount) {
      PyErr_SetString(PyExc_ValueError, "bind: wrong number of functions");
      return nullptr;
    }
    for (Py_ssize_t i = 0; i < kCount; ++i) p[i] = Address(s[i]);
    static_assert(sizeof(p) == sizeof(Library), "pointers only");
    Py_INCREF(a[1]);
    Py_XSETREF(raw_stream, a[1]);
    std::memcpy(&lib, p, sizeof(lib));
    Py_RETURN_NONE;
  } catch (const Raised&) {
    return nullptr;
  }
}

// wants_grad(tensors...): whether autograd records and one of them (tensors
// or None) takes part.
PyObject* WantsGrad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (at::GradMode::is_enabled()) {
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (THPVariable_Check(a[i]) && THPVariable_Unpack(a[i]).requires_grad()) {
        Py_RETURN_TRUE;
      }
    }
  }
  Py_RETURN_FALSE;
}

#define SCEMB_METHOD(name, f) \
  {name, reinterpret_cast<PyCFunction>(f), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {
    SCEMB_METHOD("bind", Bind),
    SCEMB_METHOD("wants_grad", WantsGrad),
    SCEMB_METHOD("layer_norm", LayerNorm),
    SCEMB_METHOD("layer_norm_grad", LayerNormGrad),
    SCEMB_METHOD("sort_by_expert", SortByExpert),
    SCEMB_METHOD("tokens_to_experts", TokensToExperts),
    SCEMB_METHOD("tokens_from_experts", TokensFromExperts),
    SCEMB_METHOD("tokens_from_experts_grad", TokensFromExpertsGrad),
    SCEMB_METHOD("expert_matmul", ExpertMatmul),
    SCEMB_METHOD("expert_matmul_grad", ExpertMatmulGrad),
    SCEMB_METHOD("quantize_weights", QuantizeWeights),
    SCEMB_METHOD("matmul_8bit", Matmul8bit),
    SCEMB_METHOD("gradient_norm", GradientNorm),
    SCEMB_METHOD("clip_gradients", ClipGradients),
    SCEMB_METHOD("adamw_sizes", AdamwSizes),
    SCEMB_METHOD("adamw_scalar", AdamwScalar),
    SCEMB_METHOD("adamw_update", AdamwUpdate),
    SCEMB_METHOD("adamw_moments", AdamwMoments),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT,
                       "_dense",
                       "Calls of the dense operators.",
                       -1,
                       kMethods,
                       nullptr,
                       nullptr,
                       nullptr,
                       nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dense() { return PyModule_Create(&kModule); }
