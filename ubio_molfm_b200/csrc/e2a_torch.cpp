// Host code against PyTorch's C++ interface, for calls whose Python side costs more than their kernels: the
// optimiser's tables of tensors (a model has hundreds) and the layer norm's autograd nodes (forward and backward
// of 2,560 x 16 values: 123 us through a Python autograd.Function, kernels of 6 us).  Loaded with ctypes.PyDLL (the
// caller holds the interpreter's lock); nothing is kept between calls.  The kernels are those of the library whose
// entry points e2a_torch_bind is given.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <optional>

#include "../../include/e2a.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int type_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

// One device, type and plain layout for all: what the optimiser's fast path needs.
struct Common {
  int type = -2, device = -2;
  bool take(const Tensor& t) {
    if (t.layout() != at::kStrided || !t.is_cuda() || !t.is_contiguous()) return false;
    const int k = type_code(t), d = t.get_device();
    if (k < 0 || (type != -2 && (k != type || d != device))) return false;
    type = k;
    device = d;
    return true;
  }
};

// ---- layer norm ------------------------------------------------------------------------------------
struct Entries {
  decltype(&e2a_layer_norm_fwd) fwd;
  decltype(&e2a_layer_norm_bwd_workspace_bytes) bwd_bytes;
  decltype(&e2a_layer_norm_bwd) bwd;
  decltype(&e2a_layer_norm_bwd2_workspace_bytes) bwd2_bytes;
  decltype(&e2a_layer_norm_bwd2) bwd2;
  decltype(&e2a_status_string) status;
  decltype(&e2a_last_cuda_error) cuda_error;
} entries{};

void check(int status, const char* what) {
  TORCH_CHECK(status == E2A_OK, what, " failed: ", entries.status(status), " (status ", status, ", cudaError ",
              entries.cuda_error(), ")");
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// t as rows of `width` with unit inner stride (a copy only where no such view exists; rows that repeat, stride 0,
// are read in place) and their stride.
struct Rows {
  Tensor t;
  int64_t ld, count;
  Rows(const Tensor& x, int64_t width) : t(x.dim() == 2 ? x : x.reshape({-1, width})) {
    if (width > 1 && t.stride(1) != 1) t = t.contiguous();
    ld = t.stride(0);
    count = t.size(0);
  }
};

// A contiguous fp32 vector, or NULL for an undefined tensor.
struct Vector {
  Tensor t;
  explicit Vector(const Tensor& v) : t(v.defined() ? v.contiguous().to(at::kFloat) : v) {}
  const float* data() const { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
};

Tensor rows_like(const Tensor& x) { return at::empty_like(x, x.options(), at::MemoryFormat::Contiguous); }

Tensor cast(const Tensor& t, const Tensor& like) {
  return t.defined() && like.defined() ? t.to(like.scalar_type()) : Tensor();
}

// {dx in x's type, dw, db in fp32}; undefined where not asked for.
variable_list backward_rows(const Tensor& x, const Tensor& g, const Tensor& weight, const Tensor& bias,
                            const Tensor& stats, int64_t act, bool need_x, bool need_cols) {
  c10::DeviceGuard guard(x.device());
  const int64_t width = x.size(-1);
  const Rows xr(x, width), gr(g, width);
  const Vector w(weight), b(bias);
  Tensor dx, dw, db, ws;
  if (need_x) dx = rows_like(x);
  size_t bytes = 0;
  if (need_cols) {
    dw = at::empty({width}, stats.options());
    db = at::empty({width}, stats.options());
    bytes = entries.bwd_bytes(xr.count, width);
    ws = at::empty({(int64_t)bytes}, stats.options().dtype(at::kByte));
  }
  const float* st = stats.const_data_ptr<float>();
  check(entries.bwd(xr.t.const_data_ptr(), xr.ld, gr.t.const_data_ptr(), gr.ld, type_code(x), w.data(), b.data(), st,
                    st + xr.count, xr.count, width, (int)act, need_x ? dx.mutable_data_ptr() : nullptr,
                    need_cols ? dw.mutable_data_ptr<float>() : nullptr,
                    need_cols ? db.mutable_data_ptr<float>() : nullptr, need_cols ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(x)),
        "e2a_layer_norm_bwd");
  return {dx, dw, db};
}

// Autograd numbers the inputs that are there: an absent weight or bias must not be passed as an undefined tensor.
using MaybeTensor = std::optional<Tensor>;
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

// Saves `always` and then the weight and the bias that are there (autograd saves no undefined tensor).
void save(AutogradContext* ctx, variable_list always, const Tensor& weight, const Tensor& bias) {
  ctx->saved_data["weight"] = weight.defined();
  ctx->saved_data["bias"] = bias.defined();
  if (weight.defined()) always.push_back(weight);
  if (bias.defined()) always.push_back(bias);
  ctx->save_for_backward(always);
}
// What save() saved, weight and bias last, undefined where absent.
variable_list saved(AutogradContext* ctx) {
  variable_list v = ctx->get_saved_variables();
  if (!ctx->saved_data["weight"].toBool()) v.insert(v.end() - (ctx->saved_data["bias"].toBool() ? 1 : 0), Tensor());
  if (!ctx->saved_data["bias"].toBool()) v.push_back(Tensor());
  return v;
}

// Whether this backward reaches the weight or the bias, whose edges are `first` and the next of those there.
bool needs_columns(const AutogradContext* ctx, size_t first, const Tensor& weight, const Tensor& bias) {
  bool any = false;
  for (const Tensor* t : {&weight, &bias})
    if (t->defined()) any |= ctx->needs_input_grad(first++);
  return any;
}

// (dx, dw, db) of the layer norm at upstream gradient g as a differentiable op.
struct LayerNormBackward : torch::autograd::Function<LayerNormBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& g, const Tensor& x, const MaybeTensor& weight_,
                               const MaybeTensor& bias_, const Tensor& stats, int64_t act, bool need_cols) {
    const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
    ctx->set_materialize_grads(false);
    save(ctx, {g, x, stats}, weight, bias);
    ctx->saved_data["act"] = act;
    variable_list out = backward_rows(x, g, weight, bias, stats, act, true, need_cols);
    if (!need_cols) return {out[0]};      // an op's outputs are all there
    return {out[0], weight.defined() ? cast(out[1], weight) : out[1], bias.defined() ? cast(out[2], bias) : out[2]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm: gradients of third and higher order are not supported");
    const variable_list v = saved(ctx);
    const Tensor &g = v[0], &x = v[1], &stats = v[2], &weight = v[3], &bias = v[4];
    grads.resize(3);
    Tensor u = grads[0];
    variable_list out(7);
    if (!u.defined() && !grads[1].defined() && !grads[2].defined()) return out;
    c10::DeviceGuard guard(x.device());
    if (!u.defined()) u = at::zeros({}, x.options()).expand_as(x);
    const int64_t width = x.size(-1);
    const Rows xr(x, width), gr(g, width), ur(u, width);
    const Vector w(weight), b(bias), p(grads[1]), q(grads[2]);
    const Tensor d_g = rows_like(x), d_x = rows_like(x);
    const bool need_cols = needs_columns(ctx, 2, weight, bias);
    Tensor dw, db;
    if (need_cols) {
      dw = at::empty({width}, stats.options());
      db = at::empty({width}, stats.options());
    }
    const size_t bytes = entries.bwd2_bytes(xr.count, width);
    const Tensor ws = at::empty({(int64_t)bytes}, stats.options().dtype(at::kByte));
    const float* st = stats.const_data_ptr<float>();
    check(entries.bwd2(xr.t.const_data_ptr(), xr.ld, gr.t.const_data_ptr(), gr.ld, ur.t.const_data_ptr(), ur.ld,
                       type_code(x), w.data(), b.data(), st, st + xr.count, p.data(), q.data(), xr.count, width,
                       (int)ctx->saved_data["act"].toInt(), d_g.mutable_data_ptr(), d_x.mutable_data_ptr(),
                       need_cols ? dw.mutable_data_ptr<float>() : nullptr,
                       need_cols ? db.mutable_data_ptr<float>() : nullptr, ws.mutable_data_ptr(), bytes, stream_of(x)),
          "e2a_layer_norm_bwd2");
    out[0] = d_g;
    out[1] = d_x;
    out[2] = cast(dw, weight);
    out[3] = cast(db, bias);
    return out;
  }
};

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_,
                        double eps, int64_t act) {
    const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
    c10::DeviceGuard guard(x.device());
    const int64_t width = x.size(-1);
    const Rows xr(x, width);
    const Vector w(weight), b(bias);
    const Tensor y = rows_like(x), stats = at::empty({2, xr.count}, x.options().dtype(at::kFloat));
    float* st = stats.mutable_data_ptr<float>();
    check(entries.fwd(xr.t.const_data_ptr(), xr.ld, type_code(x), w.data(), b.data(), xr.count, width, (float)eps,
                      (int)act, y.mutable_data_ptr(), st, st + xr.count, stream_of(x)),
          "e2a_layer_norm_fwd");
    save(ctx, {x, stats}, weight, bias);
    ctx->saved_data["act"] = act;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = saved(ctx);
    const Tensor &x = v[0], &stats = v[1], &weight = v[2], &bias = v[3];
    const int64_t act = ctx->saved_data["act"].toInt();
    const bool cols = needs_columns(ctx, 1, weight, bias);
    variable_list out;
    if (at::GradMode::is_enabled()) {
      // create_graph: the backward as an op of its own, with the second-order kernel behind it
      out = LayerNormBackward::apply(grads[0], x, maybe(weight), maybe(bias), stats, act, cols);
      out.resize(3);
    } else {
      out = backward_rows(x, grads[0], weight, bias, stats, act, ctx->needs_input_grad(0), cols);
      out[1] = cast(out[1], weight);
      out[2] = cast(out[2], bias);
    }
    return {out[0], weight.defined() ? out[1] : Tensor(), bias.defined() ? out[2] : Tensor(), Tensor(), Tensor()};
  }
};

// The tensor behind a Python object, undefined for None.
Tensor tensor_of(PyObject* o, const char* name) {
  if (o == Py_None) return Tensor();
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}

void check_affine(const Tensor& t, const Tensor& x, const char* name) {
  if (!t.defined()) return;
  const int64_t width = x.size(-1), dims = t.dim(), count = t.numel();
  TORCH_CHECK_VALUE(dims == 1 && count == width, name, " must be [", width, "], got ", count, " values in ", dims,
                    " dimensions");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type(), name,
                   " must be float32 or the input's type, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", the input on ", x.device());
}

}  // namespace

extern "C" {

// Addresses and numbers of elements of `tensors` (a list of n > 0).  Returns 0 with *type and *device where all are
// strided, contiguous CUDA tensors of one supported type on one device; 1 where not, or on any error: the caller
// then looks at them one by one and says what is wrong.
__attribute__((visibility("default"))) int e2a_tensor_table(PyObject* tensors, int64_t n, uint64_t* address,
                                                            int64_t* numel, int32_t* type, int32_t* device) {
  try {
    if (!PyList_CheckExact(tensors) || PyList_GET_SIZE(tensors) != n || n == 0) return 1;
    Common all;
    for (int64_t j = 0; j < n; ++j) {
      PyObject* o = PyList_GET_ITEM(tensors, j);
      if (!THPVariable_Check(o)) return 1;
      const Tensor& t = THPVariable_Unpack(o);
      if (!all.take(t)) return 1;
      address[j] = reinterpret_cast<uint64_t>(t.data_ptr());
      numel[j] = t.numel();
    }
    *type = all.type;
    *device = all.device;
    return 0;
  } catch (...) {
    return 1;
  }
}

// Whether a dict of dicts, an optimiser's state, is as it was noted: `held` is the list of n objects (key, entry, tuple
// of the entry's values) of every item, in the dict's order.  Compared by identity; returns 0 where all are the same.
__attribute__((visibility("default"))) int e2a_state_is_held(PyObject* state, PyObject* held, int64_t n) {
  if (!PyDict_Check(state) || !PyList_CheckExact(held) || PyList_GET_SIZE(held) != n) return 1;
  PyObject *key, *entry, *value;
  int64_t i = 0;
  for (Py_ssize_t at = 0; PyDict_Next(state, &at, &key, &entry); i += 3) {
    if (i + 3 > n || PyList_GET_ITEM(held, i) != key || PyList_GET_ITEM(held, i + 1) != entry) return 1;
    PyObject* values = PyList_GET_ITEM(held, i + 2);
    if (!PyDict_Check(entry) || !PyTuple_CheckExact(values)) return 1;
    Py_ssize_t k = 0;
    for (Py_ssize_t in = 0; PyDict_Next(entry, &in, nullptr, &value); ++k)
      if (k >= PyTuple_GET_SIZE(values) || PyTuple_GET_ITEM(values, k) != value) return 1;
    if (k != PyTuple_GET_SIZE(values)) return 1;
  }
  return i == n ? 0 : 1;
}

// The optimiser's table of a list of n parameters, which have to be those of the list `held`: for those that have a
// gradient, in order, the addresses of both, their number of elements (that of held_numel, or 1 is returned), their
// held_offset and their place in the list (int32), each from a multiple of n on in `table`; behind 5 n, type << 32 |
// device and their number.  Counts a new version of each, since the kernels write behind autograd's back.  Returns as
// above, with the number 0 and no type where no parameter has a gradient.
__attribute__((visibility("default"))) int e2a_step_table(PyObject* params, PyObject* held, int64_t n,
                                                          const int64_t* held_numel, const int64_t* held_offset,
                                                          int64_t* table) {
  try {
    if (!PyList_CheckExact(params) || PyList_GET_SIZE(params) != n) return 1;
    if (!PyList_CheckExact(held) || PyList_GET_SIZE(held) != n) return 1;
    int32_t* slot = reinterpret_cast<int32_t*>(table + 4 * n);
    Common all;
    int64_t k = 0;
    for (int64_t j = 0; j < n; ++j) {
      PyObject* o = PyList_GET_ITEM(params, j);
      if (o != PyList_GET_ITEM(held, j) || !THPVariable_Check(o)) return 1;
      const Tensor& t = THPVariable_Unpack(o);
      const Tensor& g = t.grad();
      if (!g.defined()) continue;
      if (!all.take(t) || !all.take(g) || t.numel() != held_numel[j] || g.numel() != held_numel[j]) return 1;
      table[k] = reinterpret_cast<int64_t>(t.data_ptr());
      table[n + k] = reinterpret_cast<int64_t>(g.data_ptr());
      table[2 * n + k] = held_numel[j];
      table[3 * n + k] = held_offset[j];
      slot[k++] = (int32_t)j;
    }
    for (int64_t i = 0; i < k; ++i)
      torch::autograd::impl::bump_version(THPVariable_Unpack(PyList_GET_ITEM(params, slot[i])));
    table[5 * n] = k ? (int64_t)all.type << 32 | all.device : 0;
    table[5 * n + 1] = k;
    return 0;
  } catch (...) {
    return 1;
  }
}

// The entry points of the kernels' library, in the order of Entries.
__attribute__((visibility("default"))) void e2a_torch_bind(void* const* at) {
  entries.fwd = reinterpret_cast<decltype(entries.fwd)>(at[0]);
  entries.bwd_bytes = reinterpret_cast<decltype(entries.bwd_bytes)>(at[1]);
  entries.bwd = reinterpret_cast<decltype(entries.bwd)>(at[2]);
  entries.bwd2_bytes = reinterpret_cast<decltype(entries.bwd2_bytes)>(at[3]);
  entries.bwd2 = reinterpret_cast<decltype(entries.bwd2)>(at[4]);
  entries.status = reinterpret_cast<decltype(entries.status)>(at[5]);
  entries.cuda_error = reinterpret_cast<decltype(entries.cuda_error)>(at[6]);
}

// norm.layer_norm: x a tensor, weight and bias tensors or None, act 0 or 1.  Raises as its documentation says.
__attribute__((visibility("default"))) PyObject* e2a_layer_norm(PyObject* x_, PyObject* weight_, PyObject* bias_,
                                                                double eps, int act) {
  HANDLE_TH_ERRORS
  const Tensor x = tensor_of(x_, "x"), weight = tensor_of(weight_, "weight"), bias = tensor_of(bias_, "bias");
  TORCH_CHECK_TYPE(x.defined(), "x must be a tensor");
  TORCH_CHECK_VALUE(x.is_cuda(), "ubio_molfm_b200 kernels need CUDA tensors (there is no CPU path)");
  TORCH_CHECK_TYPE(x.layout() == at::kStrided && type_code(x) >= 0,
                   "layer_norm takes float32, bfloat16 or float16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm needs a last dimension of at least one value");
  check_affine(weight, x, "weight");
  check_affine(bias, x, "bias");
  return THPVariable_Wrap(LayerNorm::apply(x, maybe(weight), maybe(bias), eps, (int64_t)act));
  END_HANDLE_TH_ERRORS
}

}  // extern "C"
