// What the optimiser's launches need to know of a list of tensors, read in one call: a model has hundreds, and
// asking each for its address, size, type, device and layout through Python costs several times the kernels.
// Loaded with ctypes.PyDLL (the caller holds the interpreter's lock); nothing is kept.
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

namespace {

int type_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

// One device, type and plain layout for all: what the fast path needs.
struct Common {
  int type = -2, device = -2;
  bool take(const at::Tensor& t) {
    if (t.layout() != at::kStrided || !t.is_cuda() || !t.is_contiguous()) return false;
    const int k = type_code(t), d = t.get_device();
    if (k < 0 || (type != -2 && (k != type || d != device))) return false;
    type = k;
    device = d;
    return true;
  }
};

}  // namespace

extern "C" {

// Addresses and numbers of elements of `tensors` (a list of n).  With `grads` also those of each one's .grad.
// Returns 0 with *type and *device where all are strided, contiguous CUDA tensors of one supported type on one
// device (and every gradient exists, as long as its parameter); 1 where not, or on any error: the caller then
// looks at them one by one and says what is wrong.
__attribute__((visibility("default"))) int e2a_tensor_table(PyObject* tensors, int64_t n, uint64_t* address,
                                                            int64_t* numel, uint64_t* grads, int32_t* type,
                                                            int32_t* device) {
  try {
    if (!PyList_CheckExact(tensors) || PyList_GET_SIZE(tensors) != n || n == 0) return 1;
    Common all;
    for (int64_t j = 0; j < n; ++j) {
      PyObject* o = PyList_GET_ITEM(tensors, j);
      if (!THPVariable_Check(o)) return 1;
      const at::Tensor& t = THPVariable_Unpack(o);
      if (!all.take(t)) return 1;
      address[j] = reinterpret_cast<uint64_t>(t.data_ptr());
      numel[j] = t.numel();
      if (grads) {
        const at::Tensor& g = t.grad();
        if (!g.defined() || !all.take(g) || g.numel() != numel[j]) return 1;
        grads[j] = reinterpret_cast<uint64_t>(g.data_ptr());
      }
    }
    *type = all.type;
    *device = all.device;
    return 0;
  } catch (...) {
    return 1;
  }
}

}  // extern "C"
