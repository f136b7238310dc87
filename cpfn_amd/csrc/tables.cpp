// Lists of tensors -> the address / length / type tables of the C ABI (include/cpfn_hip.h: cpfn_grad_norm, cpfn_grad_clip), checked, in
// one call: a model has hundreds of gradients, and reading five attributes of each from Python takes longer than the kernels.
// A CPython extension beside the C-ABI library: it only looks at tensors, it launches nothing.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <string>

namespace {

// elements fill one stretch of memory, in whatever order of the dimensions
bool dense(const at::Tensor &t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

std::string shape_of(const at::Tensor &t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// code of include/cpfn_hip.h (CPFN_F32 / BF16 / F16), -1: another type
int type_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

struct Columns {                                   // the tables while they are filled; given up on the way out unless taken
  PyObject *c[5] = {nullptr, nullptr, nullptr, nullptr, nullptr};
  ~Columns() { for (PyObject *o : c) Py_XDECREF(o); }
  PyObject *take(int i) { PyObject *o = c[i]; c[i] = nullptr; return o; }
};

// gradients(list, out list or None) -> (device, bytes moved, addresses, lengths, types, out addresses or None, out types or None)
PyObject *gradients(PyObject *, PyObject *args) {
  PyObject *list, *out;
  if (!PyArg_ParseTuple(args, "O!O", &PyList_Type, &list, &out)) return nullptr;
  const bool elsewhere = out != Py_None;
  if (elsewhere && !PyList_Check(out)) return PyErr_Format(PyExc_RuntimeError, "out must be a list of tensors");
  const Py_ssize_t n = PyList_GET_SIZE(list);
  if (elsewhere && PyList_GET_SIZE(out) != n)
    return PyErr_Format(PyExc_RuntimeError, "out must have a tensor for each gradient (got %zd for %zd)", PyList_GET_SIZE(out), n);
  Columns col;
  const Py_ssize_t width[5] = {8, 8, 4, 8, 4};
  for (int c = 0; c < (elsewhere ? 5 : 3); ++c)
  if (!(col.c[c] = PyBytes_FromStringAndSize(nullptr, n * width[c]))) return nullptr;
  void **src = (void **)PyBytes_AS_STRING(col.c[0]), **dst = elsewhere ? (void **)PyBytes_AS_STRING(col.c[3]) : nullptr;
  long long *len = (long long *)PyBytes_AS_STRING(col.c[1]), bytes = 0;
  int *type = (int *)PyBytes_AS_STRING(col.c[2]), *otype = elsewhere ? (int *)PyBytes_AS_STRING(col.c[4]) : nullptr;
  int device = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    for (int side = 0; side < (elsewhere ? 2 : 1); ++side) {
      const char *name = side ? "out" : "grads";
      PyObject *o = PyList_GET_ITEM(side ? out : list, i);
      if (!THPVariable_Check(o)) 
        return PyErr_Format(PyExc_RuntimeError, "%s must be tensors", name);
      const at::Tensor &t = THPVariable_Unpack(o);
      if (!t.is_cuda()) 
        return PyErr_Format(PyExc_RuntimeError, "%s must be CUDA(HIP) tensors: CPU not supported", name);
      if (device < 0) device = t.get_device();
      if (t.get_device() != device) 
        return PyErr_Format(PyExc_RuntimeError, "%s must be on one device (got %d and %d)", name, device, (int)t.get_device());
      const int code = type_code(t);
      if (code < 0) 
        return PyErr_Format(PyExc_RuntimeError, "%s must be float32, bfloat16 or float16 tensors (got %s)", name, c10::toString(t.scalar_type()));
      if (t.layout() != at::kStrided || !dense(t)) 
        return PyErr_Format(PyExc_RuntimeError, "%s must be dense and without overlap (got shape %s)", name,
                     t.layout() == at::kStrided ? shape_of(t).c_str() : "sparse");
      bytes += t.numel() * (code ? 2 : 4);
      if (side == 0) {
        src[i] = t.data_ptr();
        len[i] = t.numel();
        type[i] = code;
      } else {
        const at::Tensor &g = THPVariable_Unpack(PyList_GET_ITEM(list, i));
        if (t.sizes() != g.sizes() || (t.strides() != g.strides() && !(t.is_contiguous() && g.is_contiguous()))) 
          return PyErr_Format(PyExc_RuntimeError, "out must have the gradients' shapes and order of dimensions (got %s for %s)", shape_of(t).c_str(),
                       shape_of(g).c_str());
        if (code != type[i] && code != 0) 
          return PyErr_Format(PyExc_RuntimeError, "out must be of the gradient's type or float32 (got %s for %s)", c10::toString(t.scalar_type()),
                       c10::toString(g.scalar_type()));
        dst[i] = t.data_ptr();
        otype[i] = code;
      }
    }
  }
  if (!elsewhere) return Py_BuildValue("(iLNNNOO)", device, bytes, col.take(0), col.take(1), col.take(2), Py_None, Py_None);
  return Py_BuildValue("(iLNNNNN)", device, bytes, col.take(0), col.take(1), col.take(2), col.take(3), col.take(4));
}

// (nothing may leave an entry as a C++ exception)
PyObject *gradients_guarded(PyObject *self, PyObject *args) {
  try {
    return gradients(self, args);
  } catch (const std::exception &e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
}

PyMethodDef methods[] = {{"gradients", gradients_guarded, METH_VARARGS, "checked address / length / type tables of a list of gradients"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tables", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tables(void) { return PyModule_Create(&module); }
