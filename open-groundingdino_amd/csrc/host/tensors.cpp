// gdino_amd._tensors: what the multi-tensor entry points need to know of a
// list of tensors, in one call.  A model's optimizer step hands over thousands
// of tensors (weights, gradients and moments of hundreds of parameters); asking
// each for its address, size, type and layout from Python costs about 0.1 us a
// question, more than the step takes on the device.
//
// describe(tensors, written=False) -> (addresses, sizes, type, device, dense)
//   addresses, sizes  bytes: the tensors' data pointers (uint64) and element
//                     counts (int64), as the C-ABI takes them
//   type              the dtype code they share (TYPES), -1: another, -2: mixed
//   device            the device index they share, -1: host, -2: mixed
//   dense             every tensor is strided and contiguous, none is None
//   written=True      also refuses (ValueError) tensors that overlap in memory
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <utility>
#include <vector>

namespace {

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kDouble: return 1;
    case at::kBFloat16: return 2;
    case at::kHalf: return 3;
    case at::kByte: return 4;
    case at::kFloat8_e4m3fn: return 5;
    case at::kFloat8_e8m0fnu: return 6;
    default: return -1;
  }
}

PyObject* describe_list(PyObject* list, int written) {
  const Py_ssize_t n = PyList_GET_SIZE(list);
  std::vector<uint64_t> addr(n + 1);  // (never empty: a null pointer would become None)
  std::vector<int64_t> size(n + 1);
  std::vector<std::pair<uint64_t, uint64_t>> spans;
  int type = -1, device = -1;
  bool dense = true;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "item %zd is not a tensor but %.100s", i, Py_TYPE(o)->tp_name);
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    const bool strided = t.layout() == at::kStrided;
    dense = dense && strided && t.is_contiguous();
    size[i] = t.numel();
    addr[i] = strided && size[i] ? reinterpret_cast<uint64_t>(t.data_ptr()) : 0;
    const int ty = type_code(t.scalar_type());
    const int dv = t.is_cuda() ? int(t.get_device()) : (t.device().is_cpu() ? -1 : -3);
    type = i == 0 || ty == type ? ty : -2;
    device = i == 0 || dv == device ? dv : -2;
    if (written && size[i]) spans.emplace_back(addr[i], addr[i] + uint64_t(size[i]) * t.element_size());
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) {
      PyErr_SetString(PyExc_ValueError, "tensors that are updated overlap in memory (or one is listed twice)");
      return nullptr;
    }
  return Py_BuildValue("y#y#iiO", reinterpret_cast<const char*>(addr.data()), Py_ssize_t(n * sizeof(uint64_t)),
                       reinterpret_cast<const char*>(size.data()), Py_ssize_t(n * sizeof(int64_t)), type, device,
                       dense ? Py_True : Py_False);
}

PyObject* describe(PyObject*, PyObject* args, PyObject* kw) {
  static const char* names[] = {"tensors", "written", nullptr};
  PyObject* list;
  int written = 0;
  if (!PyArg_ParseTupleAndKeywords(args, kw, "O!|p", const_cast<char**>(names), &PyList_Type, &list, &written))
    return nullptr;
  try {
    return describe_list(list, written);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"describe", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(describe)), METH_VARARGS | METH_KEYWORDS,
     "describe(tensors, written=False) -> (addresses, sizes, type, device, dense)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddObject(m, "TYPES", Py_BuildValue("(sssssss)", "float32", "float64", "bfloat16", "float16", "uint8",
                                                        "float8_e4m3fn", "float8_e8m0fnu")) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
