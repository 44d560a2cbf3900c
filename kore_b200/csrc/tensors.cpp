// tensors.cpp — torch tensors described for the C entry points (kore_b200._tensors, a CPython module):
//   rows(address, tensor, name, device) fills the kore_cuda_rows at `address` from a [tokens][heads][head_dim]
//     tensor of CUDA device `device` and returns its tokens;
//   ints(tensor, name, device, dims, bytes, length) gives the address of a contiguous tensor of so many dimensions
//     of 4- or 8-byte integers, whose first dimension is `length` (-1: any).
// Both raise ValueError where the tensor does not fit. The same in Python (kore_b200/paged.py) takes 0.7 us a
// tensor, here it takes 0.1: a store of few tokens describes six and is otherwise bound by its launch.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/util/Exception.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cstring>

#include "kore_cuda.h"

namespace {

const at::Tensor *tensor_of(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_ValueError, "%s: expected a tensor, got %s", name, Py_TYPE(o)->tp_name);
        return nullptr;
    }
    return &THPVariable_Unpack(o);
}

int type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return KORE_CUDA_F32;
        case at::kHalf: return KORE_CUDA_F16;
        case at::kBFloat16: return KORE_CUDA_BF16;
        case at::kFloat8_e4m3fn: return KORE_CUDA_E4M3;
        default: return -1;
    }
}

// get_device() of a tensor that is on no CUDA device is -1, or a number of another kind of device
bool on_device(const at::Tensor &t, const char *name, long device) {
    if (t.is_cuda() && t.get_device() == device) return true;
    PyErr_Format(PyExc_ValueError, "%s is on %s, expected cuda:%ld", name, t.device().str().c_str(), device);
    return false;
}

PyObject *rows(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    if (n_args != 4) {
        PyErr_SetString(PyExc_TypeError, "rows(address, tensor, name, device)");
        return nullptr;
    }
    kore_cuda_rows *r = static_cast<kore_cuda_rows *>(PyLong_AsVoidPtr(a[0]));
    const char *name = PyUnicode_AsUTF8(a[2]);
    const long device = PyLong_AsLong(a[3]);
    if (PyErr_Occurred()) return nullptr;
    if (!r) {
        PyErr_SetString(PyExc_ValueError, "rows: the address is null");
        return nullptr;
    }
    const at::Tensor *t = tensor_of(a[1], name);
    if (!t) return nullptr;
    try {
        if (t->dim() != 3) {
            PyErr_Format(PyExc_ValueError, "%s: expected [tokens][heads][head_dim], got %ld dimensions", name, (long)t->dim());
            return nullptr;
        }
        const auto shape = t->sizes(), strides = t->strides();
        if (shape[0] > 0x7fffffffll || shape[1] > 0x7fffffffll || shape[2] > 0x7fffffffll) {
            PyErr_Format(PyExc_ValueError, "%s: %lld tokens are too many for one call", name, (long long)shape[0]);
            return nullptr;
        }
        if (strides[2] != 1 && shape[2] > 1) {
            PyErr_Format(PyExc_ValueError, "%s: the values of a head must be contiguous", name);
            return nullptr;
        }
        if (!on_device(*t, name, device)) return nullptr;
        std::memset(r, 0, sizeof(*r));   // (the hole before its strides too)
        r->data = t->data_ptr();
        r->type = type_of(t->scalar_type());
        r->n_head = (int)shape[1];
        r->head_dim = (int)shape[2];
        r->token_stride = strides[0];
        r->head_stride = strides[1];
        return PyLong_FromLongLong(shape[0]);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject *ints(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    if (n_args != 6) {
        PyErr_SetString(PyExc_TypeError, "ints(tensor, name, device, dims, bytes, length)");
        return nullptr;
    }
    const char *name = PyUnicode_AsUTF8(a[1]);
    const long device = PyLong_AsLong(a[2]), dims = PyLong_AsLong(a[3]), bytes = PyLong_AsLong(a[4]);
    const long long length = PyLong_AsLongLong(a[5]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor *t = tensor_of(a[0], name);
    if (!t) return nullptr;
    try {
        if (t->scalar_type() != (bytes == 8 ? at::kLong : at::kInt) || t->dim() != dims || !t->is_contiguous() || !t->is_cuda() ||
            t->get_device() != device) {
            PyErr_Format(PyExc_ValueError, "%s: expected a contiguous %ld-d int%ld tensor on cuda:%ld", name, dims, 8 * bytes, device);
            return nullptr;
        }
        if (length >= 0 && t->size(0) != length) {
            PyErr_Format(PyExc_ValueError, "%s: expected %lld values, got %lld", name, length, (long long)t->size(0));
            return nullptr;
        }
        return PyLong_FromVoidPtr(t->data_ptr());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {
    {"rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(rows)), METH_FASTCALL, "kore_cuda_rows of a tensor; its tokens"},
    {"ints", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(ints)), METH_FASTCALL, "address of a tensor of integers"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", "torch tensors described for the C entry points", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() {
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
