// Lists of many torch tensors, looked at in one call: their addresses, sizes and types as arrays that the C ABI takes.
// From Python each attribute of each tensor costs 30 to 60 ns, and a call on a list needs six of them: 160 tensors took 41 us before
// the first kernel was launched, against 3 us here.  What is out of the ordinary (another type, layout, device; not a list of plain
// tensors) is not judged here: the answer is None, and the caller looks at the tensors one by one and says what is wrong.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <ATen/core/Tensor.h>
#include <algorithm>
#include <vector>

namespace {

// 0, 1, 2 as VCR_F32, VCR_BF16, VCR_F16; -1: not ordinary
int kind_of(const at::Tensor& t) {
    if (!t.defined() || t.layout() != at::kStrided || !t.device().is_cuda() || t.is_neg() || !t.is_contiguous()) return -1;
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}

const at::Tensor* plain(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

template <typename F> PyObject* guarded(F body) {          // (no C++ exception leaves a C entry)
    try {
        return body();
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// words(list) -> None or (device index, bytes, address of the bytes): n addresses, n sizes (64 bits each), n kinds (32 bits)
PyObject* words(PyObject*, PyObject* list) {
    return guarded([&]() -> PyObject* {
        if (!PyList_CheckExact(list) || PyList_GET_SIZE(list) == 0) Py_RETURN_NONE;
        const Py_ssize_t n = PyList_GET_SIZE(list);
        THPObjectPtr blob(PyBytes_FromStringAndSize(nullptr, n * 20));
        if (!blob) return nullptr;
        uint64_t* at_ = (uint64_t*)PyBytes_AS_STRING(blob.get());
        int64_t* numel = (int64_t*)(at_ + n);
        int32_t* kind = (int32_t*)(numel + n);
        int device = -1;
        for (Py_ssize_t i = 0; i < n; ++i) {
            const at::Tensor* t = plain(PyList_GET_ITEM(list, i));
            const int k = t ? kind_of(*t) : -1;
            if (k < 0 || (i > 0 && t->device().index() != device)) Py_RETURN_NONE;
            device = t->device().index();
            at_[i] = (uint64_t)(uintptr_t)t->const_data_ptr();
            numel[i] = t->numel();
            kind[i] = k;
        }
        return Py_BuildValue("iNK", device, blob.release(), (unsigned long long)(uintptr_t)at_);
    });
}

// gradients(params, flags) -> None or (device index, how many have a gradient, bytes, address of the bytes): n addresses of the
// gradients (0: none, or its byte in `flags` is 0; 1: one without elements), and what identifies the parameters: n objects, addresses, sizes, kinds.
// Every gradient is of its parameter's type, size and device.
PyObject* gradients(PyObject*, PyObject* args) {
    return guarded([&]() -> PyObject* {
        PyObject *list, *flags;
        if (!PyArg_ParseTuple(args, "OO", &list, &flags)) return nullptr;
        if (!PyList_CheckExact(list) || PyList_GET_SIZE(list) == 0) Py_RETURN_NONE;
        const Py_ssize_t n = PyList_GET_SIZE(list);
        const char* wanted = nullptr;
        if (flags != Py_None) {
            if (!PyBytes_Check(flags) || PyBytes_GET_SIZE(flags) != n) { PyErr_SetString(PyExc_ValueError, "gradients: one flag for each tensor"); return nullptr; }
            wanted = PyBytes_AS_STRING(flags);
        }
        THPObjectPtr blob(PyBytes_FromStringAndSize(nullptr, n * 36));
        if (!blob) return nullptr;
        uint64_t* grad = (uint64_t*)PyBytes_AS_STRING(blob.get());
        uint64_t *object = grad + n, *at_ = object + n;
        int64_t* numel = (int64_t*)(at_ + n);
        int32_t* kind = (int32_t*)(numel + n);
        int device = -1, live = 0;
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* o = PyList_GET_ITEM(list, i);
            const at::Tensor* t = plain(o);
            const int k = t ? kind_of(*t) : -1;
            bool good = k >= 0 && (i == 0 || t->device().index() == device);
            if (good) {
                device = t->device().index();
                object[i] = (uint64_t)(uintptr_t)o;
                at_[i] = (uint64_t)(uintptr_t)t->const_data_ptr();
                numel[i] = t->numel();
                kind[i] = k;
                grad[i] = 0;
                const at::Tensor& g = t->grad();
                if (g.defined() && (!wanted || wanted[i])) {
                    good = kind_of(g) == k && g.numel() == numel[i] && g.device().index() == device;
                    if (good) { grad[i] = numel[i] ? (uint64_t)(uintptr_t)g.const_data_ptr() : 1; ++live; }
                    good = good && grad[i];
                }
            }
            if (!good) Py_RETURN_NONE;
        }
        return Py_BuildValue("iiNK", device, live, blob.release(), (unsigned long long)(uintptr_t)grad);
    });
}

// What a tensor's memory is: address, elements, and type, device and layout.
struct Memory {
    uint64_t at;
    int64_t numel;
    int32_t type, device, dense, pad;
    explicit Memory(const at::Tensor& t)
        : at((uint64_t)(uintptr_t)t.const_data_ptr()), numel(t.numel()), type((int32_t)t.scalar_type()),
          device(t.is_cuda() ? (int32_t)t.device().index() : -1), dense(t.is_contiguous()), pad(0) {}
    bool operator!=(const Memory& o) const {
        return at != o.at || numel != o.numel || type != o.type || device != o.device || dense != o.dense;
    }
};

// memory(list) -> bytes: the Memory of each tensor
PyObject* memory(PyObject*, PyObject* list) {
    return guarded([&]() -> PyObject* {
        if (!PyList_CheckExact(list)) { PyErr_SetString(PyExc_TypeError, "memory: a list of tensors"); return nullptr; }
        const Py_ssize_t n = PyList_GET_SIZE(list);
        THPObjectPtr blob(PyBytes_FromStringAndSize(nullptr, n * sizeof(Memory)));
        if (!blob) return nullptr;
        Memory* m = (Memory*)PyBytes_AS_STRING(blob.get());
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* o = PyList_GET_ITEM(list, i);
            if (!THPVariable_Check(o)) { PyErr_SetString(PyExc_TypeError, "memory: a list of tensors"); return nullptr; }
            m[i] = Memory(THPVariable_Unpack(o));
        }
        return blob.release();
    });
}

// in_place(list, bytes) -> whether every tensor's memory is what `memory` of this list gave
PyObject* in_place(PyObject*, PyObject* args) {
    return guarded([&]() -> PyObject* {
        PyObject *list, *known;
        if (!PyArg_ParseTuple(args, "O!S", &PyList_Type, &list, &known)) return nullptr;
        const Py_ssize_t n = PyList_GET_SIZE(list);
        if (PyBytes_GET_SIZE(known) != n * (Py_ssize_t)sizeof(Memory)) Py_RETURN_FALSE;
        const Memory* m = (const Memory*)PyBytes_AS_STRING(known);
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* o = PyList_GET_ITEM(list, i);
            if (!THPVariable_Check(o) || Memory(THPVariable_Unpack(o)) != m[i]) Py_RETURN_FALSE;
        }
        Py_RETURN_TRUE;
    });
}

// sharing(lists...) -> None, or the numbers of two contiguous tensors, counted through all lists, that have memory in common: a launch
// over them would write it twice, in no order
PyObject* sharing(PyObject*, PyObject* lists) {
    return guarded([&]() -> PyObject* {
        struct Range { uint64_t at, end; Py_ssize_t number; };
        std::vector<Range> ranges;
        Py_ssize_t number = 0;
        bool ascending = true;
        for (Py_ssize_t l = 0; l < PyTuple_GET_SIZE(lists); ++l) {
            PyObject* list = PyTuple_GET_ITEM(lists, l);
            const Py_ssize_t n = PyList_CheckExact(list) ? PyList_GET_SIZE(list) : 0;
            if (l == 0) ranges.reserve(n * PyTuple_GET_SIZE(lists));
            bool good = PyList_CheckExact(list);
            for (Py_ssize_t i = 0; good && i < n; ++i, ++number) {
                PyObject* o = PyList_GET_ITEM(list, i);
                if (!(good = THPVariable_Check(o))) break;
                const at::Tensor& t = THPVariable_Unpack(o);
                const uint64_t at_ = (uint64_t)(uintptr_t)t.const_data_ptr();
                if (!at_ || t.numel() == 0) continue;
                ascending = ascending && (ranges.empty() || at_ >= ranges.back().at);
                ranges.push_back({at_, at_ + (uint64_t)t.numel() * t.element_size(), number});
            }
            if (!good) { PyErr_SetString(PyExc_TypeError, "sharing: lists of tensors"); return nullptr; }
        }
        if (!ascending) std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.at < b.at; });
        for (size_t k = 1, far = 0; k < ranges.size(); ++k) {               // `far`: the one so far that reaches furthest
            if (ranges[k].at < ranges[far].end) {
                const Py_ssize_t a = ranges[far].number, b = ranges[k].number;
                return Py_BuildValue("nn", std::min(a, b), std::max(a, b));
            }
            if (ranges[k].end > ranges[far].end) far = k;
        }
        Py_RETURN_NONE;
    });
}

// changed(list, words): the tensors (words: those whose 64-bit word in these bytes is not 0) have been written to behind torch's back:
// their version counters move, so that a backward that needs the old values says so instead of using the new ones
PyObject* changed(PyObject*, PyObject* args) {
    return guarded([&]() -> PyObject* {
        PyObject *list, *which;
        if (!PyArg_ParseTuple(args, "O!O", &PyList_Type, &list, &which)) return nullptr;
        const Py_ssize_t n = PyList_GET_SIZE(list);
        const uint64_t* w = nullptr;
        if (which != Py_None) {
            if (!PyBytes_Check(which) || PyBytes_GET_SIZE(which) < 8 * n) { PyErr_SetString(PyExc_ValueError, "changed: one word for each tensor"); return nullptr; }
            w = (const uint64_t*)PyBytes_AS_STRING(which);
        }
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* o = PyList_GET_ITEM(list, i);
            if (!THPVariable_Check(o) || (w && !w[i])) continue;
            const at::Tensor& t = THPVariable_Unpack(o);
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
        Py_RETURN_NONE;
    });
}

PyMethodDef methods[] = {{"words", words, METH_O, nullptr}, {"gradients", gradients, METH_VARARGS, nullptr},
                         {"memory", memory, METH_O, nullptr}, {"in_place", in_place, METH_VARARGS, nullptr},
                         {"sharing", sharing, METH_VARARGS, nullptr},
                         {"changed", changed, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_list", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_list(void) { return PyModule_Create(&module); }
