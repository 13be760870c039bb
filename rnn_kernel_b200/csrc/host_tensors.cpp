// What a call on many tensors asks of each of them, without an interpreted
// statement for each: the Python module rnn_kernel_b200._host.

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/rnn_kernel_b200.h"

namespace {

bool as_given(const at::Tensor& t, int64_t n, at::ScalarType type, int64_t device) {
  return t.layout() == at::kStrided && t.is_cuda() && t.device().index() == device && t.scalar_type() == type &&
         t.numel() == n && t.is_contiguous();
}

// adamw_addresses(parameters, address of their gru_adamw_tensor array, GRU_F32 or GRU_BF16, device):
// fills in `param` and `grad`.  False, with some of them filled in, where a parameter
// or its gradient is not a contiguous tensor of the entry's size, the type and the
// device, or there is no gradient.
PyObject* adamw_addresses(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* params;
  unsigned long long address;
  int dtype;
  long long device;
  if (!PyArg_ParseTuple(args, "O!KiL", &PyList_Type, &params, &address, &dtype, &device)) return nullptr;
  auto* entries = reinterpret_cast<gru_adamw_tensor*>(address);
  const at::ScalarType type = dtype == GRU_F32 ? at::kFloat : at::kBFloat16;
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); ++i) {
    PyObject* object = PyList_GET_ITEM(params, i);
    if (!THPVariable_Check(object)) Py_RETURN_FALSE;
    const at::Tensor& p = THPVariable_Unpack(object);
    if (!as_given(p, entries[i].n, type, device)) Py_RETURN_FALSE;
    const at::Tensor& g = p.grad();
    if (!g.defined() || !as_given(g, entries[i].n, type, device)) Py_RETURN_FALSE;
    entries[i].param = p.mutable_data_ptr();
    entries[i].grad = g.const_data_ptr();
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"adamw_addresses", adamw_addresses, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
