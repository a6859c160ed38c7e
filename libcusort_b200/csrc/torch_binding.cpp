// torch_binding.cpp -- the PyTorch side of the routing and placement
// operators: argument checks, output allocation and the call of the C ABI, in
// one native call.  These operators take a few microseconds on the GPU in a
// decode step, so what the host spends on a call is what the call costs: from
// Python through ctypes it was 16 us for cusort_route, from here it is 5.
//
// Plain CPython functions of positional arguments; libcusort_b200/routing.py,
// experts.py and paging.py give them their names, defaults and documentation.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/TensorImpl.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <string>
#include <vector>

#include "../../include/cusort_b200.h"

namespace {

constexpr int kMaxExperts = 1024, kMaxChosen = 32, kMaxGroups = 32, kMaxRequests = 16384;
constexpr int64_t kMaxWidth = 1 << 20;

// A Python exception on its way to the entry point.
struct Refused {
  PyObject* type;  // null: already set
  std::string what;
};

// Messages are joined from strings: writing a number to an ostringstream crashed in a process with torch loaded.
std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(at::Device d) { return d.str(); }
std::string text(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + ")";
}

template <typename... A>
[[noreturn]] void refuse(PyObject* type, const A&... parts) {
  throw Refused{type, (std::string() + ... + text(parts))};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, name, " must be a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  // memory that does not hold the values: the kernels would read it as it is
  if (t.is_conj() || t.is_neg() || t._is_zerotensor())
    refuse(PyExc_ValueError, name, " must not be a lazy view (call resolve_conj() or resolve_neg(), or clone it, first)");
  return t;
}

const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

int64_t whole(PyObject* o) {
  PyObject* index = PyNumber_Index(o);
  if (index == nullptr) throw Refused{nullptr, {}};
  const int64_t v = PyLong_AsLongLong(index);
  Py_DECREF(index);
  if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, {}};
  return v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, {}};
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused{nullptr, {}};
  return v != 0;
}

at::IntArrayRef shape_of(const at::Tensor& t) { return t.sizes(); }

const char* name_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "float32";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    case at::kInt: return "int32";
    case at::kLong: return "int64";
    default: return c10::toString(t);
  }
}

cusort_float_type float_type(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return CUSORT_FLOAT_F32;
    case at::kHalf: return CUSORT_FLOAT_F16;
    case at::kBFloat16: return CUSORT_FLOAT_BF16;
    default: refuse(PyExc_TypeError, name, " must be float32, float16 or bfloat16 (got ", name_of(t.scalar_type()), ")");
  }
}

// A matrix whose rows may lie any distance apart, each contiguous in itself.
void check_rows(const at::Tensor& t, const char* name) {
  if (t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1 && t.numel() > 0))
    refuse(PyExc_ValueError, name, " must be a 2-D tensor whose rows are contiguous (got shape ", shape_of(t),
           ", strides ", t.strides(), ")");
}

void check(const at::Tensor& t, const char* name, at::ScalarType type, at::Device device, at::IntArrayRef shape) {
  if (t.scalar_type() != type || t.device() != device || t.sizes() != shape || !t.is_contiguous())
    refuse(PyExc_ValueError, name, " must be a contiguous ", name_of(type), " tensor of shape ", shape, " on ", device,
           " (got ", name_of(t.scalar_type()), ", ", shape_of(t), ", ", t.device(), ")");
}

// As another tensor's rows: its type and device, and this shape.
void check_like(const at::Tensor& t, const char* name, const at::Tensor& like, int64_t rows, int64_t columns) {
  check_rows(t, name);
  if (t.scalar_type() != like.scalar_type() || t.device() != like.device() || t.size(0) != rows || t.size(1) != columns)
    refuse(PyExc_ValueError, name, " must be ", name_of(like.scalar_type()), " of shape (", rows, ", ", columns,
           ") on ", like.device(), " (got ", name_of(t.scalar_type()), ", ", shape_of(t), ", ", t.device(), ")");
}

void check_cuda(const at::Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse(PyExc_ValueError, name, " must be a CUDA tensor (this path has no CPU implementation)");
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, at::Device device) {
  return at::Tensor(at::detail::empty_cuda(shape, type, device, std::nullopt));
}

// The outputs of one call: each an allocation of its own, or all of them parts
// of one (five allocations took as long as the launch).
class Outputs {
 public:
  Outputs(at::Device device, bool separate) : device_(device), separate_(separate) {}

  // Asks for an output; its number.
  int add(at::IntArrayRef shape, at::ScalarType type) {
    Output& o = outputs_[count_];
    o.type = type;
    o.shape.assign(shape.begin(), shape.end());
    int64_t bytes = (int64_t)c10::elementSize(type);
    for (const int64_t n : shape) bytes *= n;
    o.offset = bytes_;
    bytes_ += (bytes + 15) & ~int64_t(15);
    return count_++;
  }

  void allocate() {
    if (separate_) {
      for (int i = 0; i < count_; ++i) outputs_[i].tensor = empty(outputs_[i].shape, outputs_[i].type, device_);
      return;
    }
    const at::Tensor all = empty({bytes_}, at::kByte, device_);
    for (int i = 0; i < count_; ++i) {
      Output& o = outputs_[i];
      o.tensor = at::detail::make_tensor<c10::TensorImpl>(
          c10::Storage(all.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(o.type));
      o.tensor.unsafeGetTensorImpl()->set_storage_offset(o.offset / (int64_t)c10::elementSize(o.type));
      o.tensor.unsafeGetTensorImpl()->set_sizes_contiguous(o.shape);
    }
  }

  template <typename T>
  T* ptr(int i) const {
    return static_cast<T*>(outputs_[i].tensor.data_ptr());
  }

  // The outputs as a tuple; extra None: one more element.
  PyObject* tuple(bool extra_none = false) {
    PyObject* t = PyTuple_New(count_ + extra_none);
    if (t == nullptr) throw Refused{nullptr, {}};
    for (int i = 0; i < count_; ++i) PyTuple_SET_ITEM(t, i, THPVariable_Wrap(std::move(outputs_[i].tensor)));
    if (extra_none) {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(t, count_, Py_None);
    }
    return t;
  }

 private:
  struct Output {
    at::ScalarType type;
    c10::SmallVector<int64_t, 4> shape;
    int64_t offset;
    at::Tensor tensor;
  };
  at::Device device_;
  bool separate_;
  int count_ = 0;
  int64_t bytes_ = 0;
  Output outputs_[8];
};

template <typename T>
T* ptr(const at::Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <typename T>
T* ptr(const at::Tensor* t) {
  return t == nullptr ? nullptr : static_cast<T*>(t->data_ptr());
}

// Sets the Python exception module.name(*args); takes args over.
void set_error(const char* module, const char* name, PyObject* args) {
  PyObject* m = args ? PyImport_ImportModule(module) : nullptr;
  PyObject* type = m ? PyObject_GetAttrString(m, name) : nullptr;
  PyObject* error = type ? PyObject_CallObject(type, args) : nullptr;
  if (error) PyErr_SetObject(type, error);
  Py_XDECREF(error);
  Py_XDECREF(type);
  Py_XDECREF(m);
  Py_XDECREF(args);
}

// Calls f with the device current and its current stream.
template <typename F>
void launch(const char* what, at::Device device, F&& f) {
  const c10::cuda::OptionalCUDAGuard guard(device);
  const cudaError_t e = f(c10::cuda::getCurrentCUDAStream(device.index()).stream());
  if (e == cudaSuccess) return;
  set_error("libcusort_b200._capi", "CusortError", Py_BuildValue("(is)", (int)e, what));  // as the rest of the package
  throw Refused{nullptr, {}};
}

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

template <typename... T>
PyObject* tuple(T... objects) {
  PyObject* t = PyTuple_New(sizeof...(T));
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(t, i++, objects), ...);
  return t;
}

void check_route(const at::Tensor& logits, int64_t k, const at::Tensor* bias) {
  check_rows(logits, "logits");
  const int64_t experts = logits.size(1);
  if (experts < 1 || experts > kMaxExperts)
    refuse(PyExc_ValueError, "1 to ", kMaxExperts, " experts are supported (got ", experts, ")");
  const int64_t most = std::min<int64_t>(kMaxChosen, experts);
  if (k < 1 || k > most) refuse(PyExc_ValueError, "k must be between 1 and ", most, " (got ", k, ")");
  if (bias != nullptr) check(*bias, "bias", at::kFloat, logits.device(), {experts});
}

// logits, k, bias, score, groups, groups_kept, group_score, renormalize, scale
PyObject* route(PyObject* const* p) {
  const at::Tensor& logits = tensor(p[0], "logits");
  const int64_t k = whole(p[1]);
  const at::Tensor* bias = maybe(p[2], "bias");
  const cusort_float_type type = float_type(logits, "logits");
  check_route(logits, k, bias);
  const int64_t tokens = logits.size(0), experts = logits.size(1), groups = whole(p[4]);
  const int64_t kept = p[5] == Py_None ? groups : whole(p[5]);
  if (groups < 1 || groups > kMaxGroups || experts % groups != 0)
    refuse(PyExc_ValueError, "groups must divide the ", experts, " experts and be at most ", kMaxGroups, " (got ",
           groups, ")");
  if (kept < 1 || kept > groups || k > kept * (experts / groups))
    refuse(PyExc_ValueError, "groups_kept must be between 1 and groups=", groups, " and leave at least k=", k,
           " experts (got ", kept, ")");
  const auto score = (cusort_score)whole(p[3]);
  const auto group_score = (cusort_group_score)whole(p[6]);
  const bool renormalize = truth(p[7]);
  const float scale = (float)real(p[8]);
  check_cuda(logits, "logits");
  at::Tensor weights = empty({tokens, k}, at::kFloat, logits.device());
  at::Tensor chosen = empty({tokens, k}, at::kInt, logits.device());
  launch("cusort_route", logits.device(), [&](cudaStream_t s) {
    return cusort_route(type, logits.data_ptr(), logits.stride(0), ptr<float>(bias), ptr<float>(weights),
                        ptr<int32_t>(chosen), tokens, (int)experts, (int)k, (int)groups, (int)kept, score,
                        group_score, renormalize, scale, s);
  });
  return tuple(wrap(std::move(weights)), wrap(std::move(chosen)));
}

// grad_weights, logits, experts, bias, score, renormalize, scale
PyObject* route_backward(PyObject* const* p) {
  const at::Tensor &grad = tensor(p[0], "grad_weights"), &logits = tensor(p[1], "logits"),
                   &experts = tensor(p[2], "experts");
  const at::Tensor* bias = maybe(p[3], "bias");
  if (experts.dim() != 2) refuse(PyExc_ValueError, "experts must be [tokens, k] (got shape ", shape_of(experts), ")");
  const int64_t k = experts.size(1);
  const cusort_float_type type = float_type(logits, "logits");
  check_route(logits, k, bias);
  const int64_t tokens = logits.size(0), num = logits.size(1);
  check(experts, "experts", at::kInt, logits.device(), {tokens, k});
  check(grad, "grad_weights", at::kFloat, logits.device(), {tokens, k});
  const auto score = (cusort_score)whole(p[4]);
  const bool renormalize = truth(p[5]);
  const float scale = (float)real(p[6]);
  check_cuda(logits, "logits");
  at::Tensor out = empty({tokens, num}, logits.scalar_type(), logits.device());
  launch("cusort_route_backward", logits.device(), [&](cudaStream_t s) {
    return cusort_route_backward(type, ptr<float>(grad), logits.data_ptr(), logits.stride(0), ptr<float>(bias),
                                 ptr<int32_t>(experts), out.data_ptr(), tokens, (int)num, (int)k, score, renormalize,
                                 scale, s);
  });
  return wrap(std::move(out));
}

// experts, num_experts, align, separate
PyObject* plan_dispatch(PyObject* const* p) {
  const at::Tensor& experts = tensor(p[0], "experts");
  const int64_t num = whole(p[1]), align = whole(p[2]);
  const bool wide = experts.scalar_type() == at::kLong;
  if ((!wide && experts.scalar_type() != at::kInt) || !experts.is_contiguous())
    refuse(PyExc_ValueError, "experts must be a contiguous int32 or int64 tensor (got ",
           name_of(experts.scalar_type()), ", strides ", experts.strides(), ")");
  if (num < 1 || num > kMaxExperts)
    refuse(PyExc_ValueError, "1 to ", kMaxExperts, " experts are supported (got ", num, ")");
  if (align < 1 || align > 1 << 20) refuse(PyExc_ValueError, "align must be between 1 and 2^20 (got ", align, ")");
  const int64_t pairs = experts.numel(), capacity = pairs + std::min(num, pairs) * (align - 1);
  if (capacity > INT32_MAX)
    refuse(PyExc_ValueError, pairs, " pairs over ", num, " segments aligned to ", align,
           " rows need more than 2^31 rows");
  check_cuda(experts, "experts");
  const at::Device device = experts.device();
  size_t bytes = 0;
  launch("cusort_plan_dispatch", device, [&](cudaStream_t s) {
    return cusort_plan_dispatch(nullptr, &bytes, wide ? 8 : 4, nullptr, pairs, (int)num, (int)align, capacity, nullptr,
                                nullptr, nullptr, nullptr, s);
  });
  Outputs out(device, truth(p[3]));
  const int counts = out.add({num}, at::kInt), offsets = out.add({num + 1}, at::kInt);
  const int sources = out.add({capacity}, at::kInt), positions = out.add(experts.sizes(), at::kInt);
  out.allocate();
  // one byte is asked for where nothing is needed: any address does
  const at::Tensor temp = bytes > 1 ? empty({(int64_t)bytes}, at::kByte, device) : at::Tensor();
  launch("cusort_plan_dispatch", device, [&](cudaStream_t s) {
    return cusort_plan_dispatch(bytes > 1 ? temp.data_ptr() : out.ptr<void>(counts), &bytes, wide ? 8 : 4,
                                experts.data_ptr(), pairs, (int)num, (int)align, capacity, out.ptr<int32_t>(counts),
                                out.ptr<int32_t>(offsets), out.ptr<int32_t>(sources), out.ptr<int32_t>(positions), s);
  });
  return out.tuple();
}

// A plan's positions [tokens, k], and its sources where they are given.
void check_plan(const at::Tensor& positions, const at::Tensor* sources, at::Device device) {
  if (positions.dim() != 2)
    refuse(PyExc_ValueError, "positions must be [tokens, k] (got shape ", shape_of(positions), ")");
  const int64_t k = positions.size(1);
  if (k < 1 || k > kMaxChosen) refuse(PyExc_ValueError, "k must be between 1 and ", kMaxChosen, " (got ", k, ")");
  check(positions, "positions", at::kInt, device, positions.sizes());
  if (sources != nullptr) check(*sources, "sources", at::kInt, device, {sources->numel()});
}

// x, sources, positions
PyObject* dispatch(PyObject* const* p) {
  const at::Tensor &x = tensor(p[0], "x"), &sources = tensor(p[1], "sources"), &positions = tensor(p[2], "positions");
  check_rows(x, "x");
  check_plan(positions, &sources, x.device());
  const int64_t tokens = positions.size(0), k = positions.size(1), capacity = sources.numel(), hidden = x.size(1);
  if (x.size(0) != tokens) refuse(PyExc_ValueError, "x has ", x.size(0), " rows, positions ", tokens);
  check_cuda(x, "x");
  at::Tensor rows = empty({capacity, hidden}, x.scalar_type(), x.device());
  const int64_t size = x.element_size();
  launch("cusort_dispatch_rows", x.device(), [&](cudaStream_t s) {
    return cusort_dispatch_rows(x.data_ptr(), x.stride(0) * size, hidden * size, ptr<int32_t>(sources),
                                ptr<int32_t>(positions), rows.data_ptr(), tokens, (int)k, capacity, s);
  });
  return wrap(std::move(rows));
}

// rows, weights, positions, residual, the rows' name
PyObject* combine(PyObject* const* p) {
  const char* name = PyUnicode_AsUTF8(p[4]);
  const at::Tensor &rows = tensor(p[0], name), &positions = tensor(p[2], "positions");
  const at::Tensor *weights = maybe(p[1], "weights"), *residual = maybe(p[3], "residual");
  const cusort_float_type type = float_type(rows, name);
  if (rows.dim() != 2 || !rows.is_contiguous())
    refuse(PyExc_ValueError, name, " must be a contiguous 2-D tensor (got shape ", shape_of(rows), ")");
  check_plan(positions, nullptr, rows.device());
  const int64_t tokens = positions.size(0), k = positions.size(1), capacity = rows.size(0), hidden = rows.size(1);
  if (weights != nullptr) check(*weights, "weights", at::kFloat, rows.device(), positions.sizes());
  if (residual != nullptr) check_like(*residual, "residual", rows, tokens, hidden);
  check_cuda(rows, name);
  at::Tensor out = empty({tokens, hidden}, rows.scalar_type(), rows.device());
  launch("cusort_combine_rows", rows.device(), [&](cudaStream_t s) {
    return cusort_combine_rows(type, rows.data_ptr(), ptr<float>(weights), ptr<int32_t>(positions),
                               ptr<void>(residual), residual == nullptr ? 0 : residual->stride(0), out.data_ptr(),
                               tokens, (int)k, capacity, hidden, s);
  });
  return wrap(std::move(out));
}

// grad_out, rows, weights, sources, positions
PyObject* combine_backward(PyObject* const* p) {
  const at::Tensor &grad = tensor(p[0], "grad_out"), &rows = tensor(p[1], "rows"), &weights = tensor(p[2], "weights"),
                   &sources = tensor(p[3], "sources"), &positions = tensor(p[4], "positions");
  const cusort_float_type type = float_type(rows, "rows");
  if (rows.dim() != 2 || !rows.is_contiguous())
    refuse(PyExc_ValueError, "rows must be a contiguous 2-D tensor (got shape ", shape_of(rows), ")");
  const int64_t capacity = rows.size(0), hidden = rows.size(1);
  check_plan(positions, &sources, rows.device());
  const int64_t tokens = positions.size(0), k = positions.size(1);
  if (sources.numel() != capacity) refuse(PyExc_ValueError, "rows has ", capacity, " rows, sources ", sources.numel());
  check(weights, "weights", at::kFloat, rows.device(), positions.sizes());
  check_like(grad, "grad_out", rows, tokens, hidden);
  check_cuda(rows, "rows");
  at::Tensor grad_rows = empty({capacity, hidden}, rows.scalar_type(), rows.device());
  at::Tensor grad_weights = empty({tokens, k}, at::kFloat, rows.device());
  launch("cusort_combine_rows_backward", rows.device(), [&](cudaStream_t s) {
    return cusort_combine_rows_backward(type, grad.data_ptr(), grad.stride(0), rows.data_ptr(), ptr<float>(weights),
                                        ptr<int32_t>(sources), ptr<int32_t>(positions), grad_rows.data_ptr(),
                                        ptr<float>(grad_weights), tokens, (int)k, capacity, hidden, s);
  });
  return tuple(wrap(std::move(grad_rows)), wrap(std::move(grad_weights)));
}

// A plan's segments over the rows of t.
void check_segments(const at::Tensor& counts, const at::Tensor& offsets, const at::Tensor& t) {
  if (counts.dim() != 1 || counts.numel() < 1 || counts.numel() > kMaxExperts)
    refuse(PyExc_ValueError, "counts must be [experts], 1 to ", kMaxExperts, " of them (got shape ", shape_of(counts),
           ")");
  check(counts, "counts", at::kInt, t.device(), {counts.numel()});
  check(offsets, "offsets", at::kInt, t.device(), {counts.numel() + 1});
  if (t.size(0) > INT32_MAX - 1024)
    refuse(PyExc_ValueError, "fewer than 2^31 - 1024 rows are supported (got ", t.size(0), ")");
}

void check_width(const char* name, int64_t width) {
  if (width < 1 || width > kMaxWidth)
    refuse(PyExc_ValueError, "rows of 1 to ", kMaxWidth, " elements are supported (got ", name, " of ", width, ")");
}

// Whether the last dimension but one is the contiguous one of the experts' matrices.
bool in_contiguous(const at::Tensor& weights) {
  const bool out = weights.stride(2) == 1 || weights.size(2) == 1, in = weights.stride(1) == 1 || weights.size(1) == 1;
  if (!out && !in && weights.numel() > 0)
    refuse(PyExc_ValueError, "weights must be contiguous along one of their last two dimensions (got strides ",
           weights.strides(), ")");
  return !out;
}

// The workspace of a call: f(its address, its size) is the call itself.
template <typename F>
void launch_with_temp(const char* what, at::Device device, F&& f) {
  size_t bytes = 0;
  if (f(nullptr, &bytes, nullptr) != cudaSuccess) {
    launch(what, device, [&](cudaStream_t s) { return f(nullptr, &bytes, s); });  // says so
  }
  // one byte is asked for where nothing is needed: any address does
  const at::Tensor temp = bytes > 1 ? empty({(int64_t)bytes}, at::kByte, device) : at::Tensor();
  launch(what, device, [&](cudaStream_t s) { return f(bytes > 1 ? temp.data_ptr() : (void*)&bytes, &bytes, s); });
}

// rows, weights, counts, offsets, whether the weights are taken the other way round, the rows' name
PyObject* expert_products(PyObject* const* p) {
  const char* name = PyUnicode_AsUTF8(p[5]);
  const at::Tensor &rows = tensor(p[0], name), &weights = tensor(p[1], "weights"), &counts = tensor(p[2], "counts"),
                   &offsets = tensor(p[3], "offsets");
  const bool back = truth(p[4]);
  const cusort_float_type type = float_type(rows, name);
  check_rows(rows, name);
  check_segments(counts, offsets, rows);
  const int64_t experts = counts.numel(), capacity = rows.size(0);
  if (weights.dim() != 3 || weights.size(0) != experts || weights.size(back ? 2 : 1) != rows.size(1) ||
      weights.scalar_type() != rows.scalar_type() || weights.device() != rows.device())
    refuse(PyExc_ValueError, "weights must be ", name_of(rows.scalar_type()), " of shape (", experts, ", ",
           back ? "in, " + text(rows.size(1)) : text(rows.size(1)) + ", out", ") on ", rows.device(), " (got ",
           name_of(weights.scalar_type()), ", ", shape_of(weights), ", ", weights.device(), ")");
  const int64_t in = rows.size(1), out = weights.size(back ? 1 : 2);
  check_width(name, in);
  check_width("the result", out);
  in_contiguous(weights);
  check_cuda(rows, name);
  at::Tensor result = empty({capacity, out}, rows.scalar_type(), rows.device());
  launch_with_temp("cusort_expert_products", rows.device(), [&](void* temp, size_t* bytes, cudaStream_t s) {
    return cusort_expert_products(temp, bytes, type, rows.data_ptr(), rows.stride(0), weights.data_ptr(),
                                  weights.stride(0), weights.stride(back ? 2 : 1), weights.stride(back ? 1 : 2),
                                  ptr<int32_t>(counts), ptr<int32_t>(offsets), result.data_ptr(), capacity, in, out,
                                  (int)experts, s);
  });
  return wrap(std::move(result));
}

// grad_out, rows, counts, offsets, whether the gradient lies with its second dimension contiguous
PyObject* expert_products_grad_weights(PyObject* const* p) {
  const at::Tensor &grad = tensor(p[0], "grad_out"), &rows = tensor(p[1], "rows"), &counts = tensor(p[2], "counts"),
                   &offsets = tensor(p[3], "offsets");
  const bool in_last = truth(p[4]);
  const cusort_float_type type = float_type(rows, "rows");
  check_rows(rows, "rows");
  check_segments(counts, offsets, rows);
  const int64_t experts = counts.numel(), capacity = rows.size(0), in = rows.size(1);
  if (grad.dim() != 2) refuse(PyExc_ValueError, "grad_out must be [capacity, out] (got shape ", shape_of(grad), ")");
  const int64_t out = grad.size(1);
  check_like(grad, "grad_out", rows, capacity, out);
  check_width("rows", in);
  check_width("grad_out", out);
  check_cuda(rows, "rows");
  at::Tensor result = empty({experts, in_last ? out : in, in_last ? in : out}, rows.scalar_type(), rows.device());
  launch_with_temp("cusort_expert_products_grad_weights", rows.device(),
                   [&](void* temp, size_t* bytes, cudaStream_t s) {
                     return cusort_expert_products_grad_weights(
                         temp, bytes, type, rows.data_ptr(), rows.stride(0), grad.data_ptr(), grad.stride(0),
                         ptr<int32_t>(counts), ptr<int32_t>(offsets), result.data_ptr(), in_last, capacity, in, out,
                         (int)experts, s);
                   });
  return wrap(in_last ? result.transpose(1, 2) : std::move(result));
}

// weights
PyObject* weights_in_contiguous(PyObject* const* p) {
  const at::Tensor& weights = tensor(p[0], "weights");
  if (weights.dim() != 3)
    refuse(PyExc_ValueError, "weights must be [experts, in, out] (got shape ", shape_of(weights), ")");
  return PyBool_FromLong(in_contiguous(weights));
}

// cached_lens, new_lens, block_tables, block_size, num_tokens, free_blocks, num_free, separate
PyObject* page_plan(PyObject* const* p) {
  const at::Tensor &cached = tensor(p[0], "cached_lens"), &fresh = tensor(p[1], "new_lens"),
                   &tables = tensor(p[2], "block_tables");
  const int64_t block = whole(p[3]), tokens = whole(p[4]);
  const at::Tensor *blocks = maybe(p[5], "free_blocks"), *num_free = maybe(p[6], "num_free");
  const at::Device device = cached.device();
  if (cached.dim() != 1 || cached.numel() > kMaxRequests)
    refuse(PyExc_ValueError, "cached_lens must be 1-D with at most ", kMaxRequests, " requests (got shape ",
           shape_of(cached), ")");
  const int64_t requests = cached.numel();
  check(cached, "cached_lens", at::kInt, device, {requests});
  check(fresh, "new_lens", at::kInt, device, {requests});
  check_rows(tables, "block_tables");
  if (tables.scalar_type() != at::kInt || tables.device() != device || tables.size(0) != requests)
    refuse(PyExc_ValueError, "block_tables must be int32 with ", requests, " rows on ", device, " (got ",
           name_of(tables.scalar_type()), ", ", shape_of(tables), ", ", tables.device(), ")");
  const int64_t width = tables.size(1);
  if (requests > 1 && tables.numel() > 0 && tables.stride(0) < width)
    refuse(PyExc_ValueError, "block_tables' rows must not overlap (strides ", tables.strides(), ")");
  if (width > INT32_MAX) refuse(PyExc_ValueError, "block_tables must be at most 2^31 - 1 blocks wide");
  if (block < 1 || block > 1 << 20)
    refuse(PyExc_ValueError, "block_size must be between 1 and 2^20 (got ", block, ")");
  if (tokens < 0 || tokens > INT32_MAX)
    refuse(PyExc_ValueError, "num_tokens must be between 0 and 2^31 - 1 (got ", tokens, ")");
  if ((blocks == nullptr) != (num_free == nullptr)) refuse(PyExc_ValueError, "free_blocks and num_free go together");
  if (blocks != nullptr) {
    if (blocks->dim() != 1 || blocks->numel() > 1 << 30)
      refuse(PyExc_ValueError, "free_blocks must be 1-D with at most 2^30 blocks (got shape ", shape_of(*blocks), ")");
    check(*blocks, "free_blocks", at::kInt, device, {blocks->numel()});
    check(*num_free, "num_free", at::kInt, device, {1});
  }
  check_cuda(cached, "cached_lens");
  Outputs out(device, truth(p[7]));
  const int slots = out.add({tokens}, at::kLong), positions = out.add({tokens}, at::kInt);
  const int starts = out.add({requests + 1}, at::kInt), served = out.add({requests}, at::kBool);
  const int left = num_free == nullptr ? -1 : out.add({1}, at::kInt);
  out.allocate();
  launch("cusort_page_plan", device, [&](cudaStream_t s) {
    return cusort_page_plan(ptr<int32_t>(cached), ptr<int32_t>(fresh), (int)requests, (int)block, ptr<int32_t>(tables),
                            std::max(tables.stride(0), width), (int)width, ptr<int32_t>(blocks),
                            blocks == nullptr ? 0 : (int)blocks->numel(), ptr<int32_t>(num_free), tokens,
                            out.ptr<int64_t>(slots), out.ptr<int32_t>(positions), out.ptr<int32_t>(starts),
                            out.ptr<uint8_t>(served), left < 0 ? nullptr : out.ptr<int32_t>(left), s);
  });
  return out.tuple(left < 0);
}

// Block tables [requests, width] of int32 whose rows do not overlap, and the requests' lengths.
void check_tables(const at::Tensor& tables, const at::Tensor& lens) {
  if (lens.dim() != 1 || lens.numel() > kMaxRequests)
    refuse(PyExc_ValueError, "lens must be 1-D with at most ", kMaxRequests, " requests (got shape ", shape_of(lens),
           ")");
  check(lens, "lens", at::kInt, lens.device(), {lens.numel()});
  check_rows(tables, "block_tables");
  if (tables.scalar_type() != at::kInt || tables.device() != lens.device() || tables.size(0) != lens.numel())
    refuse(PyExc_ValueError, "block_tables must be int32 with ", lens.numel(), " rows on ", lens.device(), " (got ",
           name_of(tables.scalar_type()), ", ", shape_of(tables), ", ", tables.device(), ")");
  if (tables.size(0) > 1 && tables.numel() > 0 && tables.stride(0) < tables.size(1))
    refuse(PyExc_ValueError, "block_tables' rows must not overlap (strides ", tables.strides(), ")");
  if (tables.size(1) > 1 << 30) refuse(PyExc_ValueError, "block_tables must be at most 2^30 blocks wide");
}

void check_block_size(int64_t block) {
  if (block < 1 || block > 1 << 20)
    refuse(PyExc_ValueError, "block_size must be between 1 and 2^20 (got ", block, ")");
}

// A pool's free list, its length and its blocks' shares; the number of blocks.
int64_t check_pool(const at::Tensor& free, const at::Tensor& num_free, const at::Tensor& shares, at::Device device) {
  if (shares.dim() != 1 || shares.numel() > 1 << 30)
    refuse(PyExc_ValueError, "shares must be 1-D with at most 2^30 blocks (got shape ", shape_of(shares), ")");
  check(shares, "shares", at::kInt, device, {shares.numel()});
  check(free, "free_blocks", at::kInt, device, {shares.numel()});
  check(num_free, "num_free", at::kInt, device, {1});
  return shares.numel();
}

int64_t stride_of(const at::Tensor& tables) { return std::max(tables.stride(0), tables.size(1)); }

// block_tables, lens, parents, block_size, free_blocks, num_free, shares, separate
PyObject* page_fork(PyObject* const* p) {
  const at::Tensor &tables = tensor(p[0], "block_tables"), &lens = tensor(p[1], "lens"),
                   &parents = tensor(p[2], "parents"), &free = tensor(p[4], "free_blocks"),
                   &num_free = tensor(p[5], "num_free"), &shares = tensor(p[6], "shares");
  const int64_t block = whole(p[3]);
  check_tables(tables, lens);
  check_block_size(block);
  const at::Device device = lens.device();
  if (parents.dim() != 1 || parents.numel() > kMaxRequests)
    refuse(PyExc_ValueError, "parents must be 1-D with at most ", kMaxRequests, " requests (got shape ",
           shape_of(parents), ")");
  const int64_t children = parents.numel(), width = tables.size(1);
  check(parents, "parents", at::kInt, device, {children});
  const int64_t blocks = check_pool(free, num_free, shares, device);
  check_cuda(lens, "lens");
  Outputs out(device, truth(p[7]));
  const int new_tables = out.add({children, width}, at::kInt), new_lens = out.add({children}, at::kInt);
  const int sources = out.add({children}, at::kInt), destinations = out.add({children}, at::kInt);
  const int served = out.add({children}, at::kBool), new_shares = out.add({blocks}, at::kInt);
  const int new_free = out.add({blocks}, at::kInt), left = out.add({1}, at::kInt);
  out.allocate();
  launch_with_temp("cusort_page_fork", device, [&](void* temp, size_t* bytes, cudaStream_t s) {
    return cusort_page_fork(temp, bytes, ptr<int32_t>(tables), stride_of(tables), (int)width, ptr<int32_t>(lens),
                            (int)lens.numel(), ptr<int32_t>(parents), (int)children, (int)block, ptr<int32_t>(free),
                            ptr<int32_t>(num_free), ptr<int32_t>(shares), (int)blocks, out.ptr<int32_t>(new_tables),
                            out.ptr<int32_t>(new_lens), out.ptr<int32_t>(sources), out.ptr<int32_t>(destinations),
                            out.ptr<uint8_t>(served), out.ptr<int32_t>(new_shares), out.ptr<int32_t>(new_free),
                            out.ptr<int32_t>(left), s);
  });
  return out.tuple();
}

// block_tables, lens, keep_lens, block_size, free_blocks, num_free, shares, separate
PyObject* page_free(PyObject* const* p) {
  const at::Tensor &tables = tensor(p[0], "block_tables"), &lens = tensor(p[1], "lens"),
                   &keep = tensor(p[2], "keep_lens"), &free = tensor(p[4], "free_blocks"),
                   &num_free = tensor(p[5], "num_free"), &shares = tensor(p[6], "shares");
  const int64_t block = whole(p[3]);
  check_tables(tables, lens);
  check_block_size(block);
  const at::Device device = lens.device();
  check(keep, "keep_lens", at::kInt, device, {lens.numel()});
  const int64_t blocks = check_pool(free, num_free, shares, device);
  check_cuda(lens, "lens");
  Outputs out(device, truth(p[7]));
  const int new_shares = out.add({blocks}, at::kInt), new_free = out.add({blocks}, at::kInt);
  const int left = out.add({1}, at::kInt);
  out.allocate();
  launch_with_temp("cusort_page_free", device, [&](void* temp, size_t* bytes, cudaStream_t s) {
    return cusort_page_free(temp, bytes, ptr<int32_t>(tables), stride_of(tables), (int)tables.size(1),
                            ptr<int32_t>(lens), ptr<int32_t>(keep), (int)lens.numel(), (int)block, ptr<int32_t>(free),
                            ptr<int32_t>(num_free), ptr<int32_t>(shares), (int)blocks, out.ptr<int32_t>(new_shares),
                            out.ptr<int32_t>(new_free), out.ptr<int32_t>(left), s);
  });
  return out.tuple();
}

// block_tables, lens, block_size, num_blocks, separate
PyObject* page_compact(PyObject* const* p) {
  const at::Tensor &tables = tensor(p[0], "block_tables"), &lens = tensor(p[1], "lens");
  const int64_t block = whole(p[2]), blocks = whole(p[3]);
  check_tables(tables, lens);
  check_block_size(block);
  if (blocks < 0 || blocks > 1 << 30)
    refuse(PyExc_ValueError, "num_blocks must be between 0 and 2^30 (got ", blocks, ")");
  check_cuda(lens, "lens");
  const at::Device device = lens.device();
  Outputs out(device, truth(p[4]));
  const int new_tables = out.add(tables.sizes(), at::kInt), sources = out.add({blocks / 2}, at::kInt);
  const int destinations = out.add({blocks / 2}, at::kInt), shares = out.add({blocks}, at::kInt);
  const int free = out.add({blocks}, at::kInt), left = out.add({1}, at::kInt);
  out.allocate();
  launch_with_temp("cusort_page_compact", device, [&](void* temp, size_t* bytes, cudaStream_t s) {
    return cusort_page_compact(temp, bytes, ptr<int32_t>(tables), stride_of(tables), (int)tables.size(1),
                               ptr<int32_t>(lens), (int)lens.numel(), (int)block, (int)blocks,
                               out.ptr<int32_t>(new_tables), out.ptr<int32_t>(sources), out.ptr<int32_t>(destinations),
                               out.ptr<int32_t>(shares), out.ptr<int32_t>(free), out.ptr<int32_t>(left), s);
  });
  return out.tuple();
}

// caches (a list or tuple), sources, destinations
PyObject* page_copy(PyObject* const* p) {
  if (!PyList_Check(p[0]) && !PyTuple_Check(p[0])) refuse(PyExc_TypeError, "caches must be a list or tuple of tensors");
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(p[0]);
  const at::Tensor &sources = tensor(p[1], "sources"), &destinations = tensor(p[2], "destinations");
  const at::Device device = sources.device();
  check(sources, "sources", at::kInt, device, {sources.numel()});
  check(destinations, "destinations", at::kInt, device, {sources.numel()});
  if (sources.numel() > INT32_MAX) refuse(PyExc_ValueError, "at most 2^31 - 1 pairs are supported");
  std::vector<void*> data;
  std::vector<int64_t> strides;
  std::vector<size_t> bytes;
  int64_t blocks = 0;
  for (Py_ssize_t i = 0; i < count; ++i) {
    const at::Tensor& t = tensor(PySequence_Fast_GET_ITEM(p[0], i), "every cache");
    if (t.dim() < 1) refuse(PyExc_ValueError, "every cache must be [blocks, ...] (got shape ", shape_of(t), ")");
    if (i == 0) blocks = t.size(0);
    int64_t of = 1;
    bool dense = t.device() == device && t.size(0) == blocks && blocks <= 1 << 30;
    for (int64_t d = t.dim() - 1; d > 0; --d) {
      dense = dense && (t.size(d) == 1 || t.stride(d) == of || t.numel() == 0);
      of *= t.size(d);
    }
    if (!dense || (blocks > 1 && t.stride(0) < of && t.numel() > 0))
      refuse(PyExc_ValueError, "every cache must be on ", device, " with ", blocks,
             " blocks (2^30 at most), each contiguous in itself, that do not overlap (got shape ", shape_of(t),
             ", strides ", t.strides(), ", ", t.device(), ")");
    data.push_back(t.data_ptr());
    strides.push_back(t.stride(0) * (int64_t)t.element_size());
    bytes.push_back((size_t)(t.numel() == 0 ? 0 : of) * t.element_size());
  }
  check_cuda(sources, "sources");
  launch("cusort_page_copy", device, [&](cudaStream_t s) {
    return cusort_page_copy(data.data(), strides.data(), bytes.data(), (int)count, (int)blocks, ptr<int32_t>(sources),
                            ptr<int32_t>(destinations), sources.numel(), s);
  });
  Py_RETURN_NONE;
}

// The boundary: no C++ exception leaves through it.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  try {
    if (count != N) refuse(PyExc_TypeError, N, " arguments are expected (got ", count, ")");
    return F(args);
  } catch (const Refused& r) {
    if (r.type != nullptr) PyErr_SetString(r.type, r.what.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    set_error("torch", "OutOfMemoryError", Py_BuildValue("(s)", e.what_without_backtrace()));
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

#define ENTRY(name, n) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {ENTRY(route, 9),   ENTRY(route_backward, 7), ENTRY(plan_dispatch, 4),
                          ENTRY(dispatch, 3), ENTRY(combine, 5),       ENTRY(combine_backward, 5),
                          ENTRY(expert_products, 6), ENTRY(expert_products_grad_weights, 5),
                          ENTRY(weights_in_contiguous, 1), ENTRY(page_plan, 8),
                          ENTRY(page_fork, 8), ENTRY(page_free, 8),
                          ENTRY(page_compact, 5), ENTRY(page_copy, 3), {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_cusort_torch", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__cusort_torch() { return PyModule_Create(&kModule); }
