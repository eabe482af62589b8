// The only part of this package that reads torch's own structures: addresses of many tensors in one
// call, and the stream on which a leaf's gradient is added up.  An optimizer step needs the addresses of all weights and gradients and
// must see that each is still a dense, contiguous FP32 tensor of its size on its device: eleven Python
// attribute reads per tensor, 0.55 us, against 0.03 us here (42 tensors: a step's host time 45 -> 21 us).
// The kernels keep their plain C interface.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

namespace {

bool plain(const at::Tensor& t, int64_t size, int64_t device) {
  return t.layout() == at::kStrided && !t.is_neg() && t.scalar_type() == at::kFloat && t.is_cuda() && t.get_device() == device &&
         t.numel() == size && t.is_contiguous();
}

bool addresses(PyObject* const* args, Py_ssize_t from, Py_ssize_t count, unsigned long long* out) {
  for (Py_ssize_t i = 0; i < count; ++i) {
    out[i] = PyLong_AsUnsignedLongLong(args[from + i]);
    if (PyErr_Occurred()) return false;
  }
  return true;
}

// gather(params, sizes, device, weights, grads, empty): fills the host arrays at addresses `weights`
// and `grads` (uint64 [n]; 0 without a gradient, `empty` for one without values); `sizes`: address of
// int64 [n].  Returns how many have a gradient, or -1 - i where tensor i (with a gradient) is not what
// was expected.
PyObject* gather(PyObject*, PyObject* const* args, Py_ssize_t n) {
  unsigned long long a[5];
  if (n != 6 || !PyList_Check(args[0]) || !addresses(args, 1, 5, a)) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "gather takes a list and five integers");
    return nullptr;
  }
  const int64_t* sizes = reinterpret_cast<const int64_t*>(a[0]);
  const int64_t device = (int64_t)a[1];
  uint64_t* weights = reinterpret_cast<uint64_t*>(a[2]);
  uint64_t* grads = reinterpret_cast<uint64_t*>(a[3]);
  const Py_ssize_t count = PyList_GET_SIZE(args[0]);
  long live = 0;
  try {
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* item = PyList_GET_ITEM(args[0], i);
      if (!THPVariable_Check(item)) {
        PyErr_SetString(PyExc_TypeError, "gather takes tensors");
        return nullptr;
      }
      const at::Tensor& p = THPVariable_Unpack(item);
      const at::Tensor& g = p.grad();
      weights[i] = grads[i] = 0;
      if (!g.defined()) continue;
      if (!plain(p, sizes[i], device) || !plain(g, sizes[i], device)) return PyLong_FromLong(-1 - (long)i);
      weights[i] = reinterpret_cast<uint64_t>(p.data_ptr());
      grads[i] = sizes[i] ? reinterpret_cast<uint64_t>(g.data_ptr()) : (uint64_t)a[4];
      ++live;
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  return PyLong_FromLong(live);
}

// changed(params, grads): raises the version counter of every tensor whose entry in the host array at
// address `grads` is not 0.
PyObject* changed(PyObject*, PyObject* const* args, Py_ssize_t n) {
  unsigned long long at;
  if (n != 2 || !PyList_Check(args[0]) || !addresses(args, 1, 1, &at)) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "changed takes a list and an integer");
    return nullptr;
  }
  const uint64_t* grads = reinterpret_cast<const uint64_t*>(at);
  try {
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(args[0]); ++i) {
      PyObject* item = PyList_GET_ITEM(args[0], i);
      if (grads[i] && THPVariable_Check(item)) THPVariable_Unpack(item).unsafeGetTensorImpl()->bump_version();
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  Py_RETURN_NONE;
}

// holds(whole, from, part): whether the items of list `part` are those of list `whole` from `from` on.
PyObject* holds(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3 || !PyList_Check(args[0]) || !PyList_Check(args[2])) {
    PyErr_SetString(PyExc_TypeError, "holds takes a list, an integer and a list");
    return nullptr;
  }
  const Py_ssize_t from = PyLong_AsSsize_t(args[1]), count = PyList_GET_SIZE(args[2]);
  if (PyErr_Occurred()) return nullptr;
  bool same = from >= 0 && from <= PyList_GET_SIZE(args[0]) - count;
  for (Py_ssize_t i = 0; same && i < count; ++i) same = PyList_GET_ITEM(args[0], from + i) == PyList_GET_ITEM(args[2], i);
  return PyBool_FromLong(same);
}

// accumulates_on_default_stream(leaf): whether the leaf's gradient is added up on the device's default
// stream, as it is while a graph recorded there lives.
PyObject* accumulates_on_default_stream(PyObject*, PyObject* leaf) {
  if (!THPVariable_Check(leaf)) {
    PyErr_SetString(PyExc_TypeError, "accumulates_on_default_stream takes a tensor");
    return nullptr;
  }
  try {
    const auto node = torch::autograd::impl::try_get_grad_accumulator(THPVariable_Unpack(leaf));
    const auto stream = node ? node->stream() : std::nullopt;
    return PyBool_FromLong(stream.has_value() && stream->id() == 0);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gather)), METH_FASTCALL,
     "Addresses of tensors and their gradients."},
    {"changed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(changed)), METH_FASTCALL,
     "Raise the tensors' version counters."},
    {"holds", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(holds)), METH_FASTCALL,
     "Whether a list holds another one's items."},
    {"accumulates_on_default_stream", accumulates_on_default_stream, METH_O,
     "Whether a leaf's gradient is added up on the default stream."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: the torch whose structures this file was compiled for; with another one it must not be used.
PyMODINIT_FUNC PyInit__host_tensors() {
  PyObject* self = PyModule_Create(&module);
  if (self && PyModule_AddStringConstant(self, "torch_version", ICTC_TORCH_VERSION) < 0) {
    Py_DECREF(self);
    return nullptr;
  }
  return self;
}
