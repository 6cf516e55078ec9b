// Checks and unpacks two equally long lists of tensors (parameters, gradients) for the multi-tensor optimizer step: one pass
// in C++ instead of ten over Python objects (300 tensors: 172 us of host time for a step that takes 17 us on the GPU).
// Host code only; the C ABI of libunet_hip.so stays free of torch types.
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <vector>

namespace {

// Appends the list's addresses and sizes; false with a Python error where a tensor is not what the kernel takes.
bool unpack(PyObject* list, std::vector<uint64_t>& ptr, std::vector<int64_t>& numel, long& device) {
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
    ptr.reserve(n);
    numel.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* o = PySequence_Fast_GET_ITEM(list, i);
        if (!THPVariable_Check(o)) {
            PyErr_Format(PyExc_TypeError, "entry %zd is not a tensor", i);
            return false;
        }
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.layout() != at::kStrided || t.scalar_type() != at::kFloat || !t.is_contiguous()) {
            PyErr_SetString(PyExc_ValueError, "tensors must be dense contiguous fp32");
            return false;
        }
        const long d = t.is_cuda() ? (long)t.get_device() : -1;
        if (device == -2) device = d;
        if (d != device) {
            PyErr_SetString(PyExc_ValueError, "parameters, gradients and state must be on one device");
            return false;
        }
        ptr.push_back((uint64_t)(uintptr_t)t.const_data_ptr());
        numel.push_back(t.numel());
    }
    return true;
}

bool repeats(std::vector<uint64_t> ptr) {
    std::sort(ptr.begin(), ptr.end());
    for (size_t i = 1; i < ptr.size(); ++i)
        if (ptr[i] != 0 && ptr[i] == ptr[i - 1]) return true;       // (tensors without elements have no address)
    return false;
}

template <typename T> PyObject* bytes(const std::vector<T>& v) {
    return PyBytes_FromStringAndSize((const char*)v.data(), (Py_ssize_t)(v.size() * sizeof(T)));
}

// unpack_pair(params, grads, grads_written) -> (parameter addresses, gradient addresses, sizes, device or -1 for the CPU), host arrays as bytes
PyObject* unpack_pair(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 3) {
        PyErr_SetString(PyExc_TypeError, "unpack_pair(params, grads, grads_written)");
        return nullptr;
    }
    PyObject* a = PySequence_Fast(args[0], "params must be a sequence of tensors");
    PyObject* b = a ? PySequence_Fast(args[1], "grads must be a sequence of tensors") : nullptr;
    PyObject* result = nullptr;
    if (b) {
        try {
            std::vector<uint64_t> pa, pb;
            std::vector<int64_t> na, nb;
            long device = -2;
            const int written = PyObject_IsTrue(args[2]);
            if (PySequence_Fast_GET_SIZE(a) != PySequence_Fast_GET_SIZE(b)) PyErr_SetString(PyExc_ValueError, "list lengths differ");
            else if (written >= 0 && unpack(a, pa, na, device) && unpack(b, pb, nb, device)) {
                if (na != nb) PyErr_SetString(PyExc_ValueError, "parameter / gradient sizes differ");
                else if (repeats(pa) || (written && repeats(pb))) PyErr_SetString(PyExc_ValueError, "the same tensor is listed twice");
                else result = Py_BuildValue("(NNNl)", bytes(pa), bytes(pb), bytes(na), device < 0 ? -1L : device);
            }
        } catch (const std::exception& e) {
            PyErr_SetString(PyExc_RuntimeError, e.what());
        }
    }
    Py_XDECREF(a);
    Py_XDECREF(b);
    return result;
}

PyMethodDef methods[] = {{"unpack_pair", (PyCFunction)(void (*)(void))unpack_pair, METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_lists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_lists() { return PyModule_Create(&module); }
