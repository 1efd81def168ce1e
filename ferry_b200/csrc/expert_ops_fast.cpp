// expert_ops_fast.cpp -- the short way from Python into route_experts,
// quantize_mxfp4, dequantize_mxfp4 and execute_experts_mxfp4.
//
// A decode step calls them with kernels of a few microseconds, and checking the
// arguments, allocating the outputs and converting to C types in Python takes
// longer than that (route_experts 11 us a call, 5 this way; a quantise and a
// dequantise 24, 8; execute_experts_mxfp4 19, 9).  Each function here answers the
// plain case (tensors on the current device, rows as the kernels take them) and
// returns None for anything else, bad arguments and errors of the library
// included: ferry_b200/expert_ops.py then goes through its own checks, which copy,
// switch devices or raise.  So a case left out here costs time, never behaviour.
//
// The reference reaches its native module the same way, as a compiled extension
// (ferry/csrc/expert_ops.cpp:144-157).
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cfloat>
#include <cmath>

#include "ferryb.h"

namespace {

// libferryb's entry points (the library is loaded by ferry_b200/_lib.py)
decltype(&ferryb_route_experts) route_fn;
decltype(&ferryb_quantize_mxfp4) quantize_fn;
decltype(&ferryb_dequantize_mxfp4) dequantize_fn;
decltype(&ferryb_execute_experts_mxfp4_workspace) workspace_fn;
decltype(&ferryb_execute_experts_mxfp4) experts_fn;

int element_type(at::ScalarType t) {
  return t == at::kBFloat16 ? FERRYB_BF16 : t == at::kHalf ? FERRYB_FP16 : t == at::kFloat ? FERRYB_FP32 : -1;
}

// A plain tensor on CUDA device `device`, else null.
const at::Tensor* cuda_tensor(PyObject* o, int device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == device ? &t : nullptr;
}
const at::Tensor* index_vector(PyObject* o, int device) {
  const at::Tensor* t = cuda_tensor(o, device);
  return t && t->scalar_type() == at::kLong && t->dim() == 1 && t->is_contiguous() ? t : nullptr;
}
bool to_int(PyObject* o, int64_t low, int64_t high, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow && *v >= low && *v <= high;
}
int which(PyObject* o, const char* a, const char* b) {
  if (!PyUnicode_CheckExact(o)) return -1;
  return PyUnicode_CompareWithASCIIString(o, a) == 0 ? 0 : PyUnicode_CompareWithASCIIString(o, b) == 0 ? 1 : -1;
}
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int device) {
  return at::Tensor(at::detail::empty_cuda(size, type, c10::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)),
                                           std::nullopt));
}
cudaStream_t stream_of(int device) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}

PyObject* init(PyObject*, PyObject* args) {
  unsigned long long f[5];
  if (!PyArg_ParseTuple(args, "KKKKK", f, f + 1, f + 2, f + 3, f + 4)) return nullptr;
  route_fn = reinterpret_cast<decltype(route_fn)>(f[0]);
  quantize_fn = reinterpret_cast<decltype(quantize_fn)>(f[1]);
  dequantize_fn = reinterpret_cast<decltype(dequantize_fn)>(f[2]);
  workspace_fn = reinterpret_cast<decltype(workspace_fn)>(f[3]);
  experts_fn = reinterpret_cast<decltype(experts_fn)>(f[4]);
  Py_RETURN_NONE;
}

// (logits, topk, score, bias, n_group, topk_group, group_score, norm, scaling, weights_dtype)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !THPVariable_CheckExact(a[0])) Py_RETURN_NONE;
  const at::Tensor& logits = THPVariable_Unpack(a[0]);
  if (!logits.is_cuda()) Py_RETURN_NONE;
  const int device = logits.get_device();
  int64_t topk, n_group, topk_group;
  ferryb_route_args r{};
  if (device != c10::cuda::current_device() || logits.layout() != at::kStrided || logits.dim() != 2 ||
      !to_int(a[1], 1, logits.size(1), &topk) || !to_int(a[4], 1, 32, &n_group) ||
      !to_int(a[5], 1, 32, &topk_group) || !PyBool_Check(a[7]) || !PyFloat_CheckExact(a[8]) ||
      !THPDtype_Check(a[9]))
    Py_RETURN_NONE;
  const double scaling = PyFloat_AS_DOUBLE(a[8]);
  if (std::isfinite(scaling) && std::fabs(scaling) > FLT_MAX) Py_RETURN_NONE;  // refused if it rounds to infinity
  r.tokens = logits.size(0);
  r.experts = static_cast<int32_t>(logits.size(1) > 1024 ? 1025 : logits.size(1));
  r.row_stride = logits.stride(0);
  r.logits_type = element_type(logits.scalar_type());
  const at::ScalarType out_type = reinterpret_cast<THPDtype*>(a[9])->scalar_type;
  r.weights_type = element_type(out_type);
  r.score = which(a[2], "softmax", "sigmoid");
  r.group_score = which(a[6], "max", "top2");
  if (r.logits_type < 0 || r.weights_type < 0 || r.score < 0 || r.group_score < 0 || logits.stride(1) != 1 ||
      (r.tokens > 1 && r.row_stride < r.experts))
    Py_RETURN_NONE;
  if (a[3] != Py_None) {
    const at::Tensor* bias = cuda_tensor(a[3], device);
    if (!bias || bias->scalar_type() != at::kFloat || bias->dim() != 1 || bias->size(0) != r.experts ||
        !bias->is_contiguous())
      Py_RETURN_NONE;
    r.bias = bias->const_data_ptr<float>();
  }
  at::Tensor selected = empty({r.tokens, topk}, at::kLong, device), weights = empty({r.tokens, topk}, out_type, device);
  r.logits = logits.const_data_ptr();
  r.topk = static_cast<int32_t>(topk);
  r.n_group = static_cast<int32_t>(n_group);
  r.topk_group = static_cast<int32_t>(topk_group);
  r.norm_topk = a[7] == Py_True;
  r.scaling = static_cast<float>(scaling);
  r.selected = selected.mutable_data_ptr<int64_t>();
  r.weights = weights.mutable_data_ptr();
  if (route_fn(&r, stream_of(device))) Py_RETURN_NONE;
  PyObject* first = THPVariable_Wrap(std::move(selected));
  PyObject* second = first ? THPVariable_Wrap(std::move(weights)) : nullptr;
  PyObject* both = second ? PyTuple_Pack(2, first, second) : nullptr;
  Py_XDECREF(first);
  Py_XDECREF(second);
  return both;
  END_HANDLE_TH_ERRORS
}

// (x): codes and scales in new tensors
PyObject* quantize(PyObject*, PyObject* o) {
  HANDLE_TH_ERRORS
  if (!THPVariable_CheckExact(o)) Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(o);
  if (!x.is_cuda()) Py_RETURN_NONE;
  const int device = x.get_device(), type = element_type(x.scalar_type());
  if (device != c10::cuda::current_device() || x.layout() != at::kStrided || type < 0 || x.dim() < 1 || x.numel() == 0)
    Py_RETURN_NONE;
  const int64_t width = x.size(-1), rows = x.numel() / width;
  int64_t stride = width;
  if (width % 32) Py_RETURN_NONE;
  if (!x.is_contiguous()) {
    if (x.dim() != 2 || x.stride(1) != 1 || x.stride(0) < width) Py_RETURN_NONE;
    stride = x.stride(0);
  }
  c10::SmallVector<int64_t, 6> size(x.sizes().begin(), x.sizes().end());
  size.back() = width / 2;
  at::Tensor codes = empty(size, at::kByte, device);
  size.back() = width / 32;
  at::Tensor scales = empty(size, at::kByte, device);
  if (quantize_fn(x.const_data_ptr(), type, rows, width, stride, codes.mutable_data_ptr(), width / 2,
                  scales.mutable_data_ptr(), width / 32, stream_of(device)))
    Py_RETURN_NONE;
  PyObject* first = THPVariable_Wrap(std::move(codes));
  PyObject* second = first ? THPVariable_Wrap(std::move(scales)) : nullptr;
  PyObject* both = second ? PyTuple_Pack(2, first, second) : nullptr;
  Py_XDECREF(first);
  Py_XDECREF(second);
  return both;
  END_HANDLE_TH_ERRORS
}

// (codes, scales, dtype): the values in a new tensor
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !THPVariable_CheckExact(a[0]) || !THPDtype_Check(a[2])) Py_RETURN_NONE;
  const at::Tensor& codes = THPVariable_Unpack(a[0]);
  if (!codes.is_cuda()) Py_RETURN_NONE;
  const int device = codes.get_device();
  const at::Tensor* scales = cuda_tensor(a[1], device);
  const at::ScalarType out_type = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
  const int type = element_type(out_type);
  if (device != c10::cuda::current_device() || !scales || codes.layout() != at::kStrided || type < 0 ||
      codes.scalar_type() != at::kByte || scales->scalar_type() != at::kByte || codes.dim() < 1 ||
      codes.numel() == 0 || scales->dim() != codes.dim() || !codes.is_contiguous() || !scales->is_contiguous())
    Py_RETURN_NONE;
  const int64_t width = 2 * codes.size(-1), rows = codes.numel() / codes.size(-1);
  if (width % 32 || scales->size(-1) != width / 32) Py_RETURN_NONE;
  for (int64_t i = 0; i + 1 < codes.dim(); ++i)
    if (scales->size(i) != codes.size(i)) Py_RETURN_NONE;
  c10::SmallVector<int64_t, 6> size(codes.sizes().begin(), codes.sizes().end());
  size.back() = width;
  at::Tensor out = empty(size, out_type, device);
  if (dequantize_fn(codes.const_data_ptr(), width / 2, scales->const_data_ptr(), width / 32, rows, width,
                    out.mutable_data_ptr(), type, width, stream_of(device)))
    Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (cache, input, routing_weights, slots, starts, rows, cols, hidden, intermediate, out, err)
PyObject* experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || !THPVariable_CheckExact(a[1])) Py_RETURN_NONE;
  const at::Tensor& input = THPVariable_Unpack(a[1]);
  if (!input.is_cuda()) Py_RETURN_NONE;
  const int device = input.get_device();
  if (device != c10::cuda::current_device()) Py_RETURN_NONE;
  const at::Tensor *cache = cuda_tensor(a[0], device), *weights = cuda_tensor(a[2], device),
                   *slots = index_vector(a[3], device), *starts = index_vector(a[4], device),
                   *rows = index_vector(a[5], device), *cols = index_vector(a[6], device),
                   *err = cuda_tensor(a[10], device);
  ferryb_mxfp4_experts_args e{};
  if (!cache || !weights || !slots || !starts || !rows || !cols || !err ||
      !to_int(a[7], 128, 65536, &e.hidden) || !to_int(a[8], 128, 65536, &e.intermediate) || e.hidden % 128 ||
      e.intermediate % 128)
    Py_RETURN_NONE;
  const int64_t row_bytes = 3 * e.hidden * e.intermediate / 32 * 17;
  e.weights_type = element_type(weights->scalar_type());
  e.n_groups = slots->size(0);
  e.routes = rows->size(0);
  e.n_input = input.size(0);
  if (cache->scalar_type() != at::kByte || cache->dim() != 2 || cache->size(1) != row_bytes || cache->size(0) < 1 ||
      !cache->is_contiguous() || reinterpret_cast<uintptr_t>(cache->const_data_ptr()) % 32 ||
      input.scalar_type() != at::kBFloat16 || input.layout() != at::kStrided || input.dim() != 2 ||
      input.size(1) != e.hidden || input.stride(1) != 1 ||
      reinterpret_cast<uintptr_t>(input.const_data_ptr()) % 16 ||
      (e.n_input > 1 && (input.stride(0) % 8 || input.stride(0) < e.hidden)) || e.weights_type < 0 ||
      weights->dim() != 2 || weights->size(0) != e.n_input || !weights->is_contiguous() ||
      starts->size(0) != e.n_groups + 1 || cols->size(0) != e.routes || e.routes == 0 || e.n_groups == 0 ||
      err->scalar_type() != at::kInt || err->numel() != 1)
    Py_RETURN_NONE;
  const at::Tensor* given = nullptr;
  if (a[9] != Py_None) {
    given = cuda_tensor(a[9], device);
    if (!given || given->scalar_type() != at::kBFloat16 || given->dim() != 2 || given->size(0) != e.routes ||
        given->size(1) != e.hidden || !given->is_contiguous() ||
        reinterpret_cast<uintptr_t>(given->const_data_ptr()) % 4)
      Py_RETURN_NONE;
  }
  e.workspace_bytes = workspace_fn(e.routes, e.n_groups, e.hidden, e.intermediate);
  if (e.workspace_bytes < 0) Py_RETURN_NONE;
  at::Tensor workspace = empty({e.workspace_bytes}, at::kByte, device);
  at::Tensor out = given ? *given : empty({e.routes, e.hidden}, at::kBFloat16, device);
  e.cache = cache->const_data_ptr();
  e.cache_slots = cache->size(0);
  e.input = input.const_data_ptr();
  e.input_stride = input.stride(0);
  e.routing_weights = weights->const_data_ptr();
  e.topk = weights->size(1);
  e.slots = slots->const_data_ptr<int64_t>();
  e.starts = starts->const_data_ptr<int64_t>();
  e.rows = rows->const_data_ptr<int64_t>();
  e.cols = cols->const_data_ptr<int64_t>();
  e.out = out.mutable_data_ptr();
  e.workspace = workspace.mutable_data_ptr();
  e.err = err->mutable_data_ptr<int32_t>();
  if (experts_fn(&e, stream_of(device))) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"init", init, METH_VARARGS, nullptr},
    {"route_experts", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(route)), METH_FASTCALL, nullptr},
    {"quantize_mxfp4", quantize, METH_O, nullptr},
    {"dequantize_mxfp4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dequantize)), METH_FASTCALL, nullptr},
    {"execute_experts_mxfp4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(experts)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__fast() {
  PyObject* m = PyModule_Create(&kModule);
  // what it was compiled against; _lib.fast() leaves it aside under anything else
  if (m && (PyModule_AddStringConstant(m, "torch_version", FERRYB_TORCH_VERSION) ||
            PyModule_AddStringConstant(m, "python_version", PY_VERSION))) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
