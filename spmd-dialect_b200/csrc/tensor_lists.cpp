// tensor_lists.cpp -- reads a Python list of torch tensors into the host arrays
// that the list entries take (addresses, element counts, element types), with
// the checks those need.  One call per list: a hundred tensors take a few
// microseconds here and a hundred through attribute by attribute in Python,
// which is more than a small step takes on the GPU.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "../../include/spmd_b200.h"

namespace {

constexpr long kE4M3 = 3;  // bit of `kinds`, and type code, of an 8-bit state

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SPMDB200_F32;
    case at::kHalf: return SPMDB200_F16;
    case at::kBFloat16: return SPMDB200_BF16;
    case at::kFloat8_e4m3fn: return (int)kE4M3;
    default: return -1;
  }
}

// read(what, tensors, device, kinds, like) -> (addresses, sizes, types): bytes of
// uint64, int64 and int32.  `tensors` is a list of contiguous tensors on cuda
// device `device` whose types are among the bits of `kinds` (1 << type code); an
// entry may be None where bit 8 is set (address 0).  `like` is None or a list of
// as many tensors with the same shapes.
PyObject *read(PyObject *, PyObject *args) {
  const char *what;
  PyObject *tensors, *like;
  long device, kinds;
  if (!PyArg_ParseTuple(args, "sO!llO", &what, &PyList_Type, &tensors, &device, &kinds, &like)) return nullptr;
  if (like != Py_None && !PyList_Check(like)) return PyErr_Format(PyExc_TypeError, "%s: like is a list or None", what);
  const Py_ssize_t n = PyList_GET_SIZE(tensors);
  if (like != Py_None && PyList_GET_SIZE(like) != n)
    return PyErr_Format(PyExc_ValueError, "%s: %zd tensors for %zd parameters", what, n, PyList_GET_SIZE(like));
  PyObject *ptrs = PyBytes_FromStringAndSize(nullptr, n * 8), *sizes = PyBytes_FromStringAndSize(nullptr, n * 8),
           *types = PyBytes_FromStringAndSize(nullptr, n * 4), *out = nullptr;
  if (ptrs && sizes && types) {
    auto *p = reinterpret_cast<uint64_t *>(PyBytes_AS_STRING(ptrs));
    auto *s = reinterpret_cast<int64_t *>(PyBytes_AS_STRING(sizes));
    auto *t = reinterpret_cast<int32_t *>(PyBytes_AS_STRING(types));
    Py_ssize_t k = 0;
    try {
      for (; k < n; ++k) {
        PyObject *o = PyList_GET_ITEM(tensors, k);
        if (o == Py_None && (kinds & 256)) {
          p[k] = 0, s[k] = 0, t[k] = 0;
          continue;
        }
        if (!THPVariable_Check(o)) {
          PyErr_Format(PyExc_TypeError, "%s: entry %zd is not a tensor", what, k);
          break;
        }
        const at::Tensor &x = THPVariable_Unpack(o);
        if (!x.is_cuda() || x.get_device() != device || x.layout() != at::kStrided) {
          PyErr_Format(PyExc_ValueError, "%s: tensor %zd is not a plain tensor on cuda:%ld, as the first is", what, k, device);
          break;
        }
        const int code = code_of(x.scalar_type());
        if (code < 0 || !(kinds >> code & 1)) {
          PyErr_Format(PyExc_TypeError, "%s: tensor %zd has dtype %s", what, k, c10::toString(x.scalar_type()));
          break;
        }
        if (x.is_neg()) {  // its memory holds the negated values
          PyErr_Format(PyExc_ValueError, "%s: tensor %zd is negated lazily (resolve_neg gives its values)", what, k);
          break;
        }
        if (!x.is_contiguous()) {
          PyErr_Format(PyExc_ValueError, "%s: tensor %zd is not contiguous", what, k);
          break;
        }
        if (like != Py_None) {
          PyObject *l = PyList_GET_ITEM(like, k);
          if (!THPVariable_Check(l) || THPVariable_Unpack(l).sizes() != x.sizes()) {
            PyErr_Format(PyExc_ValueError, "%s: tensor %zd does not have its parameter's shape", what, k);
            break;
          }
        }
        p[k] = reinterpret_cast<uint64_t>(x.data_ptr());
        s[k] = x.numel();
        t[k] = code;
      }
    } catch (const std::exception &e) {
      PyErr_Format(PyExc_RuntimeError, "%s: tensor %zd: %s", what, k, e.what());
      k = -1;
    }
    if (k == n) out = PyTuple_Pack(3, ptrs, sizes, types);
  }
  Py_XDECREF(ptrs);
  Py_XDECREF(sizes);
  Py_XDECREF(types);
  return out;
}

// written(lists...): raises the version counter of every tensor of lists that a kernel
// has written, as in-place operations of torch do, so that autograd refuses what
// it saved of them.  A list, and an entry, may be None.
PyObject *written(PyObject *, PyObject *args) {
  for (Py_ssize_t a = 0; a < PyTuple_GET_SIZE(args); ++a) {
    PyObject *list = PyTuple_GET_ITEM(args, a);
    if (list == Py_None) continue;
    if (!PyList_Check(list)) return PyErr_Format(PyExc_TypeError, "written: argument %zd is no list", a);
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(list); ++k) {
      PyObject *o = PyList_GET_ITEM(list, k);
      if (!THPVariable_Check(o)) continue;
      const at::Tensor &x = THPVariable_Unpack(o);
      if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();  // inference tensors have no counter
    }
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"read", read, METH_VARARGS, "read(what, tensors, device, kinds, like)"},
                         {"written", written, METH_VARARGS, "written(lists...)"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists() { return PyModule_Create(&module); }
