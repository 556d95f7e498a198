// Addresses, element counts and type codes of a list of torch tensors, for the entry points that
// take hundreds of them in a call (cflk_grad_sumsq, cflk_grad_clip). In Python each attribute of
// each tensor costs about 60 ns: 384 gradients and their outputs 200 us, more than the kernels run.
//
//   tensor_table(sequence) -> (addresses, counts, codes, device)
//
// the first three bytes objects of int64, int64 and int32 (0 float16, 1 bfloat16, 2 float32), the
// last the CUDA device's index, or -1 for no tensors. ValueError for anything that is not a
// contiguous tensor of those types on one CUDA device.
//
//   mark_written(sequence) -> None
//
// counts an in-place change of each tensor, as torch's own operators do, so that autograd refuses a
// backward pass over a saved tensor that has since been written.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>

namespace {

PyObject* refuse(const char* what) {
    PyErr_SetString(PyExc_ValueError, what);
    return nullptr;
}

// false with the error set
bool fill(PyObject* seq, Py_ssize_t n, int64_t* ptrs, int64_t* numel, int32_t* codes,
          int64_t& device) {
    PyObject** items = PySequence_Fast_ITEMS(seq);
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (!THPVariable_Check(items[i])) {
            refuse("gradients must be tensors");
            return false;
        }
        const at::Tensor& t = THPVariable_Unpack(items[i]);
        if (t.layout() != at::kStrided || !t.is_contiguous()) {
            refuse("tensors must be contiguous");
            return false;
        }
        switch (t.scalar_type()) {
            case at::kHalf: codes[i] = 0; break;
            case at::kBFloat16: codes[i] = 1; break;
            case at::kFloat: codes[i] = 2; break;
            default: refuse("gradients must be float16, bfloat16 or float32"); return false;
        }
        const int64_t d = t.is_cuda() ? t.get_device() : -1;
        if (d < 0 || (device >= 0 && d != device)) {
            refuse("tensors must be on one CUDA device");
            return false;
        }
        device = d;
        ptrs[i] = reinterpret_cast<int64_t>(t.data_ptr());
        numel[i] = t.numel();
    }
    return true;
}

PyObject* tensor_table(PyObject*, PyObject* arg) {
    PyObject* seq = PySequence_Fast(arg, "a sequence of tensors is wanted");
    if (seq == nullptr) {
        return nullptr;
    }
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    PyObject* ptrs = PyBytes_FromStringAndSize(nullptr, n * 8);
    PyObject* numel = PyBytes_FromStringAndSize(nullptr, n * 8);
    PyObject* codes = PyBytes_FromStringAndSize(nullptr, n * 4);
    PyObject* out = nullptr;
    if (ptrs != nullptr && numel != nullptr && codes != nullptr) {
        int64_t device = -1;
        bool ok = false;
        try {
            ok = fill(seq, n, reinterpret_cast<int64_t*>(PyBytes_AS_STRING(ptrs)),
                      reinterpret_cast<int64_t*>(PyBytes_AS_STRING(numel)),
                      reinterpret_cast<int32_t*>(PyBytes_AS_STRING(codes)), device);
        } catch (const std::exception& e) {  // torch's own errors must not cross into Python
            refuse(e.what());
        }
        if (ok) {
            out = Py_BuildValue("(OOOL)", ptrs, numel, codes, (long long)device);
        }
    }
    Py_XDECREF(ptrs);
    Py_XDECREF(numel);
    Py_XDECREF(codes);
    Py_DECREF(seq);
    return out;
}

PyObject* mark_written(PyObject*, PyObject* arg) {
    PyObject* seq = PySequence_Fast(arg, "a sequence of tensors is wanted");
    if (seq == nullptr) {
        return nullptr;
    }
    PyObject* out = Py_None;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    try {
        for (Py_ssize_t i = 0; out != nullptr && i < n; ++i) {
            PyObject* item = PySequence_Fast_GET_ITEM(seq, i);
            if (!THPVariable_Check(item)) {
                out = refuse("gradients must be tensors");
            } else if (const at::Tensor& t = THPVariable_Unpack(item); !t.is_inference()) {
                t.unsafeGetTensorImpl()->bump_version();  // (inference tensors have none)
            }
        }
    } catch (const std::exception& e) {
        out = refuse(e.what());
    }
    Py_DECREF(seq);
    Py_XINCREF(out);
    return out;
}

PyMethodDef methods[] = {
    {"tensor_table", tensor_table, METH_O,
     "Addresses, element counts, type codes and device of a list of tensors."},
    {"mark_written", mark_written, METH_O, "Count an in-place change of each tensor of a list."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_cflk_table", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cflk_table() {
    return PyModule_Create(&module);
}
