// gp_tensors.cpp — whether torch tensors still are what a plan over their memory
// was made of: the same address, length, type and order of values.  A Python
// module of its own (geeps_amd.native.tensor_facts), since a call of a plan asks
// for every tensor that it lists: 152 tensors take 0.83 us here, 6.7 through
// Tensor.data_ptr(), of a call of 10.6 us.  Host code, no HIP.

#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <exception>

namespace {

struct Fact {
  const void *data;
  int64_t values;
  int32_t type;
  int32_t in_order;
};

bool fact_of(PyObject *object, Fact *fact) {
  if (!THPVariable_Check(object)) {
    PyErr_SetString(PyExc_TypeError, "not a tensor");
    return false;
  }
  try {
    const at::Tensor &t = THPVariable_Unpack(object);
    std::memset(fact, 0, sizeof *fact);  // compared as bytes
    fact->data = t.const_data_ptr();
    fact->values = t.numel();
    fact->type = (int32_t)t.scalar_type();
    fact->in_order = t.is_contiguous();
    return true;
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return false;
  }
}

PyObject *facts(PyObject *, PyObject *tensors) {
  if (!PyTuple_Check(tensors)) {
    PyErr_SetString(PyExc_TypeError, "facts(tuple of tensors)");
    return nullptr;
  }
  const Py_ssize_t n = PyTuple_GET_SIZE(tensors);
  PyObject *bytes = PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(Fact));
  if (!bytes) return nullptr;
  char *to = PyBytes_AS_STRING(bytes);
  for (Py_ssize_t i = 0; i < n; ++i) {
    Fact fact;
    if (!fact_of(PyTuple_GET_ITEM(tensors, i), &fact)) {
      Py_DECREF(bytes);
      return nullptr;
    }
    std::memcpy(to + i * sizeof fact, &fact, sizeof fact);
  }
  return bytes;
}

PyObject *moved(PyObject *, PyObject *const *args, Py_ssize_t count) {
  if (count != 2 || !PyTuple_Check(args[0]) || !PyBytes_Check(args[1]) ||
      PyBytes_GET_SIZE(args[1]) != PyTuple_GET_SIZE(args[0]) * (Py_ssize_t)sizeof(Fact)) {
    PyErr_SetString(PyExc_TypeError, "moved(tuple of tensors, facts of as many)");
    return nullptr;
  }
  const char *was = PyBytes_AS_STRING(args[1]);
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[0]); ++i) {
    Fact fact;
    if (!fact_of(PyTuple_GET_ITEM(args[0], i), &fact)) return nullptr;
    if (std::memcmp(&fact, was + i * sizeof fact, sizeof fact) != 0) return PyLong_FromSsize_t(i);
  }
  return PyLong_FromLong(-1);
}

PyMethodDef methods[] = {
    {"facts", facts, METH_O, "facts(tensors): what moved() compares by, as bytes."},
    {"moved", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(moved)), METH_FASTCALL,
     "moved(tensors, facts): the first tensor that is not what it was, or -1."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "gp_tensors", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_gp_tensors(void) { return PyModule_Create(&module); }
