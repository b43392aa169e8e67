// What the operators on torch tensors share (rows_torch.cpp, layer_torch.cpp): argument checks, launches on torch's
// current stream of the tensors' device, and what their autograd nodes hold.
#pragma once
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include "../../include/tace_hip.h"
#include "../../include/tace_rows.h"

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t MAX_ROW = 32768, MAX_INDEX = INT32_MAX - 8192;

inline int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return TACE_ROW_F32;
    case at::kDouble: return TACE_ROW_F64;
    case at::kBFloat16: return TACE_ROW_BF16;
    case at::kHalf: return TACE_ROW_F16;
    default: return -1;
  }
}

inline at::ScalarType sum_type(const Tensor& t) { return t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

// (a transform's wrapper, without storage, is refused by autograd or where its address is asked for)
inline void want_memory(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(!t.has_storage() || t.numel() == 0 || t.const_data_ptr(), name, " holds no memory (a fake tensor)");
}

inline void want_rows(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a GPU tensor (got ", t.device(), ")");
  TORCH_CHECK_VALUE(type_code(t.scalar_type()) >= 0, name, " has dtype ", t.scalar_type(),
                    ", expected float32, float64, bfloat16 or float16");
  want_memory(t, name);
}

inline void want_indices(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " has dtype ", t.scalar_type(),
                    ", expected int32 or int64");
  want_memory(t, name);
}

inline void want_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", expected ", like.device());
  want_memory(t, name);
}

inline void want_int32(const Tensor& t, int64_t n, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.is_contiguous() && !t.is_neg() && t.dim() == 1 && t.size(0) == n, name,
                    " must be a contiguous int32 tensor of ", n);
  want_device(t, like, name);
}

// what a kernel reads: rows one after the other, their signs in memory
inline Tensor signed_values(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
inline Tensor dense(const Tensor& t) { return signed_values(t).contiguous(); }

inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline int* ints(const Tensor& t) { return t.defined() ? t.data_ptr<int>() : nullptr; }

// Brackets a launch by ops.TIMER's events where the forward call was timed.
struct Launch {
  static inline PyObject* start = nullptr;   // ops._t0, ops._t1
  static inline PyObject* stop = nullptr;
  c10::DeviceGuard guard;
  void* stream;
  const char* name;
  py::object token;

  Launch(const Tensor& t, const char* name, bool timed)
      : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()), name(name) {
    if (timed) {
      py::gil_scoped_acquire gil;
      token = py::reinterpret_borrow<py::object>(start)(name);
    }
  }
  ~Launch() {
    if (token) {   // (left by an error)
      py::gil_scoped_acquire gil;
      token = py::object();
    }
  }
  void done(int rc, std::initializer_list<int64_t> sizes) {
    if (token) {
      py::gil_scoped_acquire gil;
      py::tuple info(sizes.size());
      size_t i = 0;
      for (int64_t v : sizes) info[i++] = py::int_(v);
      py::reinterpret_borrow<py::object>(stop)(token, info);
      token = py::object();
    }
    TORCH_CHECK(rc == 0, "tace_", name, " failed (", rc, "): ", tace_last_error());
  }
};

// whether autograd has to see this call
inline bool tracked(const Tensor& t) {
  return t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined());
}

// a node's plain arguments
template <typename T>
struct Held : torch::CustomClassHolder {
  T v;
  explicit Held(T x) : v(std::move(x)) {}
};
template <typename T>
void hold(AutogradContext* ctx, const T& v) {
  ctx->saved_data["args"] = c10::IValue::make_capsule(c10::make_intrusive<Held<T>>(v));
}
template <typename T>
const T& held(AutogradContext* ctx) {
  return static_cast<Held<T>*>(ctx->saved_data["args"].toCapsule().get())->v;
}

// A grouping's or plan's tensor beside the saved variables (which would refuse
// one made in inference mode, where there are no versions): a backward that
// finds it written to since raises, as for a saved variable.
struct Pinned {
  Tensor t;
  uint32_t version = 0;

  Pinned() = default;
  Pinned(const Tensor& x) : t(x), version(x.is_inference() ? 0 : x._version()) {}
  const Tensor& get(const char* name) const {
    TORCH_CHECK(t.is_inference() || t._version() == version, "one of the variables needed for gradient computation has "
                "been modified by an inplace operation: ", name, " is at version ", t._version(), ", expected ", version);
    return t;
  }
};

inline optional<Tensor> maybe(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

void bind_layer(py::module_& mod);   // layer_torch.cpp
