// Host fast path of the FP8 block-scaled operators (tokenforge_b200/fp8.py): one C++ call that looks
// at the tensors, allocates the outputs and calls the C ABI of the kernel library.
//
// The operators' kernels take 2 to 6 us at decode sizes, less than Python needs for the same
// checks, allocations and a ctypes call (10 to 14 us on the measured host; 4 to 6 here). Each
// function returns None for anything but the plain case (a subclass, a CPU or misplaced tensor, a
// wrong type, shape, stride or alignment, another current device, a status that is not 0); the
// Python function then goes its own way, which makes every check and raises every error.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/tokenforge_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

constexpr int64_t kGroup = 128;

// A plain CUDA tensor on the current device, or null.
const Tensor* plain(PyObject* o, int device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == device ? &t : nullptr;
}

// The first operand, which says the device: null unless that is the current one. The driver is
// not asked about anything before a CUDA tensor shows that it is there.
const Tensor* leading(PyObject* o, int* device) {
  if (!THPVariable_CheckExact(o) || !THPVariable_Unpack(o).is_cuda()) return nullptr;
  *device = c10::cuda::current_device();
  return plain(o, *device);
}

int stream_dtype(ScalarType t) {
  return t == ScalarType::Half ? TF_DTYPE_FP16 : t == ScalarType::BFloat16 ? TF_DTYPE_BF16 : -1;
}

bool codes(ScalarType t) { return t == ScalarType::Float8_e4m3fn || t == ScalarType::Byte; }

Tensor empty(at::IntArrayRef sizes, ScalarType type, int device) {
  return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, static_cast<int8_t>(device)),
                                std::nullopt);
}

// sizes with the last one replaced.
c10::SmallVector<int64_t, 5> with_last(const Tensor& t, int64_t last) {
  c10::SmallVector<int64_t, 5> s(t.sizes().begin(), t.sizes().end());
  s.back() = last;
  return s;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<int8_t>(device)).stream(); }

template <typename T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}

PyObject* none() { Py_RETURN_NONE; }

PyObject* pack(std::initializer_list<Tensor> ts) {
  PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) {
      Py_DECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

// Runs `body`, with C++ exceptions turned into Python's as PyTorch's own bindings do it (an output
// that does not fit is a torch.OutOfMemoryError).
template <typename F>
PyObject* guarded(F body) {
  try {
    return body();
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

// The interpreter lock is given up while outputs are allocated and the kernel is launched, either of
// which may wait (for memory, for a place in the launch queue).
class Unlocked {
 public:
  Unlocked() : state_(PyEval_SaveThread()) {}
  ~Unlocked() { PyEval_RestoreThread(state_); }
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;

 private:
  PyThreadState* state_;
};

bool group_arg(PyObject* o, int* group) {
  int overflow = 0;  // a number past a long is refused later, like any other wrong one
  const long g = PyLong_Check(o) ? PyLong_AsLongAndOverflow(o, &overflow) : -1;
  *group = static_cast<int>(g);
  return g == 0 || g == kGroup;
}

// (x, residual or None, weight, eps, group_size) -> (q, scale, sum) or None
PyObject* add_rmsnorm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int group;
    if (n != 5 || !group_arg(args[4], &group) || !PyFloat_Check(args[3])) return none();
    int device;
    const Tensor* x = leading(args[0], &device);
    if (!x) return none();
    const Tensor* w = plain(args[2], device);
    const Tensor* r = args[1] == Py_None ? nullptr : plain(args[1], device);
    if (!w || (args[1] != Py_None && !r) || x->dim() == 0) return none();
    const ScalarType type = x->scalar_type();
    const int dtype = stream_dtype(type);
    const int64_t h = x->size(-1);
    if (dtype < 0 || h == 0 || x->numel() == 0 || !x->is_contiguous()) return none();
    if (w->scalar_type() != type || w->dim() != 1 || w->size(0) != h || !w->is_contiguous())
      return none();
    if (r && (r->scalar_type() != type || r->sizes() != x->sizes() || !r->is_contiguous()))
      return none();
    const int64_t rows = x->numel() / h, groups = group ? (h + kGroup - 1) / kGroup : 1;
    const float eps = static_cast<float>(PyFloat_AS_DOUBLE(args[3]));
    Tensor q, scale, sum;
    int st;
    {
      Unlocked unlocked;
      q = empty(x->sizes(), ScalarType::Float8_e4m3fn, device);
      scale = empty(with_last(*x, groups), ScalarType::Float, device);
      if (r) sum = empty(x->sizes(), type, device);
      st = tf_add_rmsnorm_fp8_quant(
          ptr<uint16_t>(*x), rows, h, h, r ? ptr<uint16_t>(*r) : nullptr, r ? h : 0,
          ptr<uint16_t>(*w), eps, dtype, group, ptr<uint8_t>(q), ptr<float>(scale),
          r ? ptr<uint16_t>(sum) : nullptr, h, stream_of(device));
    }
    if (st != TF_OK) return none();
    if (r) return pack({q, scale, sum});
    PyObject* out = pack({q, scale, q});
    if (out) {  // without a residual the third output is the caller's x itself
      Py_INCREF(args[0]);
      PyObject* old = PyTuple_GET_ITEM(out, 2);
      PyTuple_SET_ITEM(out, 2, args[0]);
      Py_DECREF(old);
    }
    return out;
  });
}

// (gate_up, group_size) -> (q, scale) or None
PyObject* silu_mul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int group;
    if (n != 2 || !group_arg(args[1], &group)) return none();
    int device;
    const Tensor* x = leading(args[0], &device);
    if (!x || x->dim() == 0) return none();
    const int dtype = stream_dtype(x->scalar_type());
    const int64_t width = x->size(-1);
    if (dtype < 0 || x->numel() == 0 || width % 2 || !x->is_contiguous()) return none();
    const int64_t i = width / 2, rows = x->numel() / width;
    Tensor q, scale;
    int st;
    {
      Unlocked unlocked;
      q = empty(with_last(*x, i), ScalarType::Float8_e4m3fn, device);
      scale = empty(with_last(*x, group ? (i + kGroup - 1) / kGroup : 1), ScalarType::Float,
                    device);
      st = tf_silu_mul_fp8_quant(ptr<uint16_t>(*x), rows, i, width, dtype, group, ptr<uint8_t>(q),
                                 ptr<float>(scale), stream_of(device));
    }
    return st == TF_OK ? pack({q, scale}) : none();
  });
}

// (x,) -> (q, scale) or None
PyObject* quant_groups(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 1) return none();
    int device;
    const Tensor* x = leading(args[0], &device);
    if (!x || x->dim() == 0) return none();
    const int dtype = stream_dtype(x->scalar_type());
    if (dtype < 0 || x->numel() == 0 || !x->is_contiguous()) return none();
    const int64_t c = x->size(-1), rows = x->numel() / c;
    Tensor q, scale;
    int st;
    {
      Unlocked unlocked;
      q = empty(x->sizes(), ScalarType::Float8_e4m3fn, device);
      scale = empty(with_last(*x, (c + kGroup - 1) / kGroup), ScalarType::Float, device);
      st = tf_e4m3_quant_groups(ptr<uint16_t>(*x), rows, c, c, dtype, ptr<uint8_t>(q),
                                ptr<float>(scale), stream_of(device));
    }
    return st == TF_OK ? pack({q, scale}) : none();
  });
}

// (xq, x_scale, wq, w_scale, bias or None, out_dtype) -> y or None
PyObject* block_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || !THPDtype_Check(args[5])) return none();
    int device;
    const Tensor* x = leading(args[0], &device);
    if (!x) return none();
    const Tensor* xs = plain(args[1], device);
    const Tensor *w = plain(args[2], device), *ws = plain(args[3], device);
    const Tensor* b = args[4] == Py_None ? nullptr : plain(args[4], device);
    if (!xs || !w || !ws || (args[4] != Py_None && !b)) return none();
    const ScalarType type = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
    const int dtype = stream_dtype(type);
    if (dtype < 0 || !codes(x->scalar_type()) || !codes(w->scalar_type()) ||
        xs->scalar_type() != ScalarType::Float || ws->scalar_type() != ScalarType::Float)
      return none();
    if (w->dim() != 2 || x->dim() == 0 || x->numel() == 0 || xs->dim() != x->dim()) return none();
    const int64_t rows_w = w->size(0), k = w->size(1), kb = (k + kGroup - 1) / kGroup;
    if (rows_w == 0 || k == 0 || k % 16 || x->size(-1) != k || ws->dim() != 2 ||
        ws->size(0) != (rows_w + kGroup - 1) / kGroup || ws->size(1) != kb)
      return none();
    const auto scale_sizes = with_last(*x, kb);
    if (xs->sizes() != at::IntArrayRef(scale_sizes)) return none();
    if (!x->is_contiguous() || !xs->is_contiguous() || !w->is_contiguous() || !ws->is_contiguous())
      return none();
    if (b && (b->scalar_type() != type || b->dim() != 1 || b->size(0) != rows_w ||
              !b->is_contiguous()))
      return none();
    const int64_t m = x->numel() / k;
    Tensor y;
    int st;
    {
      Unlocked unlocked;
      y = empty(with_last(*x, rows_w), type, device);
      st = tf_w8a8_block_linear(
          ptr<uint8_t>(*x), m, k, k, ptr<float>(*xs), kb, ptr<uint8_t>(*w), ptr<float>(*ws),
          b ? ptr<uint16_t>(*b) : nullptr, rows_w, dtype, ptr<uint16_t>(y), rows_w,
          stream_of(device));
    }
    return st == TF_OK ? THPVariable_Wrap(y) : none();
  });
}

PyMethodDef kMethods[] = {
    {"add_rmsnorm", reinterpret_cast<PyCFunction>(add_rmsnorm), METH_FASTCALL, nullptr},
    {"silu_mul", reinterpret_cast<PyCFunction>(silu_mul), METH_FASTCALL, nullptr},
    {"quant_groups", reinterpret_cast<PyCFunction>(quant_groups), METH_FASTCALL, nullptr},
    {"block_linear", reinterpret_cast<PyCFunction>(block_linear), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "fp8_host", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fp8_host(void) { return PyModule_Create(&kModule); }
