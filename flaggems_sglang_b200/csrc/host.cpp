// The short way from Python into the operators of ops/norm.py and ops/linear.py: arguments as they usually come (CUDA tensors on the
// current device, dense, 16-byte aligned, of the expected types and shapes) are checked, results and workspaces allocated and the C entry
// point called without going back to the interpreter.  Anything else is answered with None, and the Python function does the work: it
// also has the words for what is refused.  A call on a few rows takes the GPU 3 to 7 us; from Python alone the host needed 10 to 12 us for
// it (17 for the MLP), of which the launch is 2.
#include <Python.h>

#include <cstring>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/fmoe_b200.h"

namespace {

struct {
  decltype(&fmoe_rms_norm_quant) norm;
  decltype(&fmoe_fp8_linear) linear;
  decltype(&fmoe_fp8_linear_workspace_bytes) linear_bytes;
  decltype(&fmoe_fp8_mlp) mlp;
  decltype(&fmoe_fp8_mlp_workspace_bytes) mlp_bytes;
} entry = {};

// The tensor behind a Python object; null for anything but a plain torch.Tensor (subclasses may mean something else by their methods).
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool is(const at::Tensor* t, c10::Device device, at::ScalarType type, int64_t dims) {
  return t && t->is_cuda() && t->device() == device && t->scalar_type() == type && t->dim() == dims && t->is_contiguous() && !t->is_neg() &&
         (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15) == 0;
}
bool is(const at::Tensor* t, c10::Device device, at::ScalarType type, int64_t rows, int64_t cols) {
  return is(t, device, type, 2) && t->size(0) == rows && t->size(1) == cols;
}

// Other Python threads run meanwhile: allocations and launches may wait (for memory, for room in the stream's queue), perhaps for what
// another thread has yet to launch.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// past the dispatcher, where no mode wants to see the call
at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, c10::Device device) {
  if (c10::impl::dispatch_mode_enabled()) return at::empty(sizes, at::TensorOptions().dtype(type).device(device));
  return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}

int code_of(at::ScalarType t) { return t == at::kBFloat16 ? FMOE_BF16 : (t == at::kFloat ? FMOE_F32 : -1); }

// What an operator's operands are, or null fields where the call is not a usual one.
struct Operands {
  const at::Tensor *x, *x_scale, *w, *w_scale, *w2 = nullptr, *w2_scale = nullptr, *bias = nullptr, *addend = nullptr;
  fmoe_fp8_args a = {};
  bool ok = false;
};

constexpr auto kE4M3 = at::kFloat8_e4m3fn;

Operands rows_and_weight(PyObject* x, PyObject* x_scale, PyObject* w, PyObject* w_scale) {
  Operands o;
  o.x = tensor(x);
  o.w = tensor(w);
  o.w_scale = tensor(w_scale);
  o.x_scale = nullptr;
  if (!o.x || !o.w || !o.x->is_cuda() || o.x->device().index() != c10::cuda::current_device()) return o;
  const auto dev = o.x->device();
  const auto type = o.x->scalar_type();
  if (type != kE4M3 && type != at::kBFloat16) return o;
  if (!is(o.x, dev, type, 2) || !is(o.w, dev, kE4M3, 2)) return o;
  const int64_t T = o.x->size(0), K = o.x->size(1), rows = o.w->size(0);
  if (T == 0 || K == 0 || K % 128 || o.w->size(1) != K || rows == 0) return o;
  if (!is(o.w_scale, dev, at::kFloat, (rows + 127) / 128, K / 128)) return o;
  if (type == kE4M3) {
    o.x_scale = tensor(x_scale);
    if (!is(o.x_scale, dev, at::kFloat, T, K / 128)) return o;
  } else if (x_scale != Py_None) {
    return o;
  }
  o.a.struct_size = sizeof(fmoe_fp8_args);
  o.a.x_dtype = type == kE4M3 ? FMOE_E4M3 : FMOE_BF16;
  o.a.T = T;
  o.a.K = K;
  o.a.x = o.x->const_data_ptr();
  o.a.x_scale = o.x_scale ? static_cast<const float*>(o.x_scale->const_data_ptr()) : nullptr;
  o.a.w = o.w->const_data_ptr();
  o.a.w_scale = static_cast<const float*>(o.w_scale->const_data_ptr());
  o.ok = true;
  return o;
}

// addend and output of a call that is otherwise complete, its workspace, the call: the output, or an error code
template <typename Run, typename Bytes>
PyObject* finish(Operands& o, PyObject* addend, Run run, Bytes bytes) {
  const auto dev = o.x->device();
  if (addend != Py_None) {
    o.addend = tensor(addend);
    if (!is(o.addend, dev, at::kBFloat16, o.a.T, o.a.N)) Py_RETURN_NONE;
    o.a.addend = o.addend->const_data_ptr();
  }
  at::Tensor out, ws;
  int64_t need;
  int rc = FMOE_OK;
  {
    Unlocked other_threads_run;
    out = make({o.a.T, o.a.N}, at::kBFloat16, dev);
    o.a.out = out.mutable_data_ptr();
    need = bytes(&o.a);
    if (need > 0) {
      ws = make({need}, at::kByte, dev);
      o.a.workspace = ws.mutable_data_ptr();
      o.a.workspace_bytes = need;
    }
    if (need >= 0) rc = run(&o.a, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  }
  if (need < 0) Py_RETURN_NONE;  // the Python function says why
  if (rc != FMOE_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
}

// linear(x, w, w_scale, x_scale, bias, addend)
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  Operands o = rows_and_weight(args[0], args[3], args[1], args[2]);
  if (!o.ok || o.w->size(0) % 8) Py_RETURN_NONE;
  o.a.N = o.w->size(0);
  if (args[4] != Py_None) {
    o.bias = tensor(args[4]);
    if (!is(o.bias, o.x->device(), at::kFloat, 1) || o.bias->size(0) != o.a.N) Py_RETURN_NONE;
    o.a.bias = static_cast<const float*>(o.bias->const_data_ptr());
  }
  return finish(o, args[5], entry.linear, entry.linear_bytes);
  END_HANDLE_TH_ERRORS
}

// mlp(x, w13, w13_scale, w2, w2_scale, x_scale, activation code, addend)
PyObject* mlp(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !PyLong_Check(args[6])) Py_RETURN_NONE;
  Operands o = rows_and_weight(args[0], args[5], args[1], args[2]);
  if (!o.ok || o.w->size(0) % 256) Py_RETURN_NONE;
  o.a.I = o.w->size(0) / 2;
  o.a.activation = (int)PyLong_AsLong(args[6]);
  const auto dev = o.x->device();
  o.w2 = tensor(args[3]);
  o.w2_scale = tensor(args[4]);
  if (!is(o.w2, dev, kE4M3, 2) || o.w2->size(1) != o.a.I || o.w2->size(0) == 0 || o.w2->size(0) % 8) Py_RETURN_NONE;
  o.a.N = o.w2->size(0);
  if (!is(o.w2_scale, dev, at::kFloat, (o.a.N + 127) / 128, o.a.I / 128)) Py_RETURN_NONE;
  o.a.w2 = o.w2->const_data_ptr();
  o.a.w2_scale = static_cast<const float*>(o.w2_scale->const_data_ptr());
  return finish(o, args[7], entry.mlp, entry.mlp_bytes);
  END_HANDLE_TH_ERRORS
}

// norm(x, weight, eps, residual, per_token, return_norm)
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !PyFloat_Check(args[2]) || !PyBool_Check(args[4]) || !PyBool_Check(args[5])) Py_RETURN_NONE;
  const at::Tensor *x = tensor(args[0]), *weight = tensor(args[1]), *residual = args[3] == Py_None ? nullptr : tensor(args[3]);
  if (!x || !weight || (args[3] != Py_None && !residual) || !x->is_cuda() || x->device().index() != c10::cuda::current_device()) Py_RETURN_NONE;
  const auto dev = x->device();
  const auto type = x->scalar_type();
  const int code = code_of(type), w_code = code_of(weight->scalar_type());
  const bool per_token = args[4] == Py_True, keep = args[5] == Py_True;
  if (code < 0 || w_code < 0 || !is(x, dev, type, 2) || !is(weight, dev, weight->scalar_type(), 1)) Py_RETURN_NONE;
  const int64_t rows = x->size(0), K = x->size(1);
  if (rows == 0 || K == 0 || K > 16384 || K % (per_token ? 8 : 128) || weight->size(0) != K) Py_RETURN_NONE;
  if (residual && !is(residual, dev, type, rows, K)) Py_RETURN_NONE;
  const void *x_data = x->const_data_ptr(), *weight_data = weight->const_data_ptr();
  void* residual_data = residual ? residual->mutable_data_ptr() : nullptr;
  const float eps = (float)PyFloat_AS_DOUBLE(args[2]);
  at::Tensor q, s, out;
  int rc;
  {
    Unlocked other_threads_run;
    q = make({rows, K}, kE4M3, dev);
    s = per_token ? make({rows}, at::kFloat, dev) : make({rows, K / 128}, at::kFloat, dev);
    if (keep) out = make({rows, K}, type, dev);
    rc = entry.norm(x_data, K, residual_data, K, code, weight_data, w_code, rows, K, eps, per_token, q.mutable_data_ptr(),
                    static_cast<float*>(s.mutable_data_ptr()), keep ? out.mutable_data_ptr() : nullptr,
                    c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  }
  if (rc != FMOE_OK) return PyLong_FromLong(rc);
  PyObject* result = PyTuple_New(keep ? 3 : 2);
  if (!result) return nullptr;
  PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(s)));
  if (keep) PyTuple_SET_ITEM(result, 2, THPVariable_Wrap(std::move(out)));
  return result;
  END_HANDLE_TH_ERRORS
}

// bind(addresses of fmoe_rms_norm_quant, fmoe_fp8_linear, .._workspace_bytes, fmoe_fp8_mlp, .._workspace_bytes): the library that is loaded
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  void* p[5];
  if (n != 5) return PyErr_Format(PyExc_TypeError, "bind takes five addresses");
  for (int i = 0; i < 5; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (!p[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "a null address");
  }
  entry.norm = reinterpret_cast<decltype(entry.norm)>(p[0]);
  entry.linear = reinterpret_cast<decltype(entry.linear)>(p[1]);
  entry.linear_bytes = reinterpret_cast<decltype(entry.linear_bytes)>(p[2]);
  entry.mlp = reinterpret_cast<decltype(entry.mlp)>(p[3]);
  entry.mlp_bytes = reinterpret_cast<decltype(entry.mlp_bytes)>(p[4]);
  Py_RETURN_NONE;
}

#define TEXT_OF(x) #x
#define TEXT(x) TEXT_OF(x)
#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"bind", FAST(bind), nullptr},
                         {"norm", FAST(norm), nullptr},
                         {"linear", FAST(linear), nullptr},
                         {"mlp", FAST(mlp), nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__host() {
  constexpr char built[] = TEXT(PY_MAJOR_VERSION) "." TEXT(PY_MINOR_VERSION) ".";
  if (strncmp(Py_GetVersion(), built, sizeof built - 1) != 0) return PyErr_Format(PyExc_ImportError, "built for another version of Python");
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", BUILT_FOR_TORCH) < 0) Py_CLEAR(m);
  return m;
}
