// Python module vc3d._tensors (host only): what an operator over hundreds of tensors asks of each of them, in one call.  A tensor's type,
// device, sizes, strides and address cost 40-70 ns each through Python; for AdamW over 100 tensors with 8-bit moments that was
// 140 of a step's 180 us (its kernels: 15).
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <string>
#include <vector>

#include "autograd.h"

namespace {

constexpr int64_t BLOCK = 256;  // VC_ADAMW_BLOCK
const char* const NAMES[6] = {"params", "grads", "exp_avg", "exp_avg_sq", "m_scale", "v_scale"};

struct Row {  // vc_adamw_tensor
    uint64_t p, g, m, v, m_scale, v_scale;
    int64_t n;
};

struct Sequence {
    PyObject* o = nullptr;
    ~Sequence() { Py_XDECREF(o); }
};

// addresses of what a launch writes: each may be there once (two workgroups would otherwise write one element)
struct Once {
    std::vector<uint64_t> slots;
    size_t mask;
    explicit Once(size_t most) {
        size_t n = 64;
        while (n < 2 * most) n *= 2;
        slots.assign(n, 0), mask = n - 1;
    }
    bool add(uint64_t a) {
        size_t i = (a * 0x9E3779B97F4A7C15ull >> 20) & mask;
        for (; slots[i] != 0; i = (i + 1) & mask)
            if (slots[i] == a) return false;
        slots[i] = a;
        return true;
    }
};

// fills `rows`; what is wrong, or "" (an exception is set where the lists hold something else than tensors)
std::string fill(Sequence* lists, int columns, Py_ssize_t n, Row* rows) {
    const bool eight = columns == 6;
    const at::Tensor* first = nullptr;
    at::ScalarType type{};
    Once written((size_t)n * (columns - 1));
    for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor* t[6];
        for (int c = 0; c < columns; ++c) {
            PyObject* const o = PySequence_Fast_GET_ITEM(lists[c].o, i);
            if (!THPVariable_Check(o)) return std::string(NAMES[c]) + "[" + std::to_string(i) + "] is no tensor";
            t[c] = &THPVariable_Unpack(o);
            if (t[c]->layout() != at::kStrided) return std::string(NAMES[c]) + "[" + std::to_string(i) + "] is not strided";
        }
        const at::Tensor& p = *t[0];
        if (first == nullptr) {
            first = &p, type = p.scalar_type();
            if (!p.is_cuda()) return "params[0] is not on the GPU";
            if (type != at::kFloat && type != at::kBFloat16) return std::string("params are ") + c10::toString(type) + "; fp32 or bf16 expected";
        }
        const at::ScalarType moment = eight ? at::kFloat8_e4m3fn : at::kFloat;
        const int64_t numel = p.numel();
        for (int c = 0; c < columns; ++c) {
            const at::ScalarType want = c < 2 ? type : c < 4 ? moment : at::kFloat;
            if (t[c]->scalar_type() != want)
                return std::string(NAMES[c]) + "[" + std::to_string(i) + "] is " + c10::toString(t[c]->scalar_type()) + "; " + c10::toString(want) + " expected";
            if (t[c]->device() != first->device()) return std::string(NAMES[c]) + "[" + std::to_string(i) + "] is not on " + first->device().str();
            if (c >= 4) {
                if (t[c]->numel() != (numel + BLOCK - 1) / BLOCK || !t[c]->is_contiguous())
                    return std::string(NAMES[c]) + " hold ceil(numel / 256) contiguous values each";
            } else if (c > 0 && t[c]->sizes() != p.sizes())
                return std::string(NAMES[c]) + " and params differ in shape";
        }
        if (!(p.is_contiguous() && t[1]->is_contiguous() && t[2]->is_contiguous() && t[3]->is_contiguous())) {
            bool same = p.is_non_overlapping_and_dense();
            for (int c = 1; c < 4; ++c) same = same && (numel <= 1 || t[c]->strides() == p.strides());
            if (!same) return "tensor " + std::to_string(i) + " and its gradient and moments must lie in memory in one dense order";
        }
        auto at = [](const at::Tensor& x) { return (uint64_t)(uintptr_t)x.mutable_data_ptr(); };
        rows[i] = {at(p), (uint64_t)(uintptr_t)t[1]->const_data_ptr(), at(*t[2]), at(*t[3]), eight ? at(*t[4]) : 0, eight ? at(*t[5]) : 0, numel};
        if (numel > 0 && !(written.add(rows[i].p) && written.add(rows[i].m) && written.add(rows[i].v) &&
                           (!eight || (written.add(rows[i].m_scale) && written.add(rows[i].v_scale)))))
            return "tensor " + std::to_string(i) + ", or one of its moments, is in the lists twice";
    }
    return "";
}

// adamw_table(lists, table): lists = (params, grads, exp_avg, exp_avg_sq[, m_scale, v_scale]), n tensors each; table = a writable
// buffer of 56 n bytes -> None, or what is wrong with the tensors
PyObject* adamw_table(PyObject*, PyObject* args) {
    PyObject *tuple, *buffer;
    if (!PyArg_ParseTuple(args, "O!O", &PyTuple_Type, &tuple, &buffer)) return nullptr;
    const Py_ssize_t columns = PyTuple_GET_SIZE(tuple);
    if (columns != 4 && columns != 6) return PyErr_Format(PyExc_ValueError, "4 or 6 lists expected"), nullptr;
    Sequence lists[6];
    Py_ssize_t n = 0;
    for (Py_ssize_t c = 0; c < columns; ++c) {
        lists[c].o = PySequence_Fast(PyTuple_GET_ITEM(tuple, c), "lists of tensors expected");
        if (lists[c].o == nullptr) return nullptr;
        const Py_ssize_t k = PySequence_Fast_GET_SIZE(lists[c].o);
        if (c == 0) n = k;
        else if (k != n) return PyUnicode_FromFormat("%zd %s for %zd params", k, NAMES[c], n);
    }
    Py_buffer view;
    if (PyObject_GetBuffer(buffer, &view, PyBUF_WRITABLE) != 0) return nullptr;
    PyObject* out = nullptr;
    if (view.len != (Py_ssize_t)(n * sizeof(Row))) PyErr_Format(PyExc_ValueError, "a table of %zd bytes expected", n * sizeof(Row));
    else
        out = [&]() -> PyObject* {
            HANDLE_TH_ERRORS
            const std::string wrong = fill(lists, (int)columns, n, (Row*)view.buf);
            return wrong.empty() ? Py_NewRef(Py_None) : PyUnicode_FromStringAndSize(wrong.data(), (Py_ssize_t)wrong.size());
            END_HANDLE_TH_ERRORS
        }();
    PyBuffer_Release(&view);
    return out;
}

// written(list, ...): counts a write in place for each tensor, as torch's own operators do
PyObject* written(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    for (Py_ssize_t c = 0; c < PyTuple_GET_SIZE(args); ++c) {
        Sequence list;
        list.o = PySequence_Fast(PyTuple_GET_ITEM(args, c), "lists of tensors expected");
        if (list.o == nullptr) return nullptr;
        for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(list.o); ++i) {
            PyObject* const o = PySequence_Fast_GET_ITEM(list.o, i);
            if (!THPVariable_Check(o)) return PyErr_Format(PyExc_TypeError, "tensors expected"), nullptr;
            const at::Tensor& t = THPVariable_Unpack(o);
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef METHODS[] = {{"adamw_table", adamw_table, METH_VARARGS, nullptr},
                         {"written", written, METH_VARARGS, nullptr},
                         {"bind", vc_bind, METH_VARARGS, nullptr},
                         {"gated_scan", vc_gated_scan_py, METH_VARARGS, nullptr},
                         {"gated_scan_step", vc_gated_scan_step_py, METH_VARARGS, nullptr},
                         {"linear_cross_entropy", vc_linear_cross_entropy_py, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&MODULE); }
