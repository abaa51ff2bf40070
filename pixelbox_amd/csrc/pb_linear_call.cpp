// pb_linear_call.cpp -- the short way from torch tensors to pb_quantize_rows, pb_linear_i8, pb_group_rows and pb_linear_grouped.
//
// One such call is a kernel of a few microseconds; checking a dozen tensor properties from Python and converting sixteen arguments
// through ctypes takes as long again (1 x 256 x 1280 in 8 bits, two calls: 14.3 us).  This module looks at the usual call -- right
// types, shapes and devices, contiguous tensors, no gradients or tangents -- and makes it; whatever it does not recognise it leaves alone (None), for
// pixelbox_amd/linear.py to check in full, to name the error or to make the call itself.  The library's functions are handed over by
// address (bind), so that this module uses the same copy of it as everything else in the process.
#define PY_SSIZE_T_CLEAN
#include <ATen/Functions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/pixelbox_hip.h"

namespace {

decltype(&pb_quantize_rows) f_quantize;
decltype(&pb_linear_i8) f_linear_i8;
decltype(&pb_group_rows) f_group;
decltype(&pb_linear_grouped) f_grouped;

using at::Tensor;

// a plain tensor argument; null where it is something else (a subclass, None)
const Tensor *tensor(PyObject *o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool usual(const Tensor *t, at::ScalarType type, int device, int dims) {
    return t && t->scalar_type() == type && t->is_cuda() && t->get_device() == device && t->dim() == dims && t->layout() == at::kStrided && t->is_contiguous() &&
           !(t->requires_grad() && at::GradMode::is_enabled()) && !t->is_neg() && !t->_is_zerotensor() && !t->_fw_grad(/*level=*/0).defined();
}
bool vector(const Tensor *t, at::ScalarType type, int device, int64_t n) { return usual(t, type, device, 1) && t->size(0) == n; }
bool matrix(const Tensor *t, at::ScalarType type, int device, int64_t m, int64_t n) { return usual(t, type, device, 2) && t->size(0) == m && t->size(1) == n; }

int float_type(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return PB_TYPE_F32;
        case at::kBFloat16: return PB_TYPE_BF16;
        case at::kHalf: return PB_TYPE_F16;
        default: return -1;
    }
}
bool float_matrix(const Tensor *t, int device, int64_t m, int64_t n) { return t && float_type(*t) >= 0 && matrix(t, t->scalar_type(), device, m, n); }

void *stream_of(int device) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }
const float *floats(const Tensor *t) { return t ? static_cast<const float *>(t->data_ptr()) : nullptr; }
const int *ints(const Tensor *t) { return t ? static_cast<const int *>(t->data_ptr()) : nullptr; }

// an output as a kernel argument: its version is counted up, so that a backward pass that saved the old values says so
void *written(const Tensor *t) {
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    return t->data_ptr();
}

// the call's status as a number; None for a call that is not the usual one
PyObject *status(int rc) { return PyLong_FromLong(rc); }
#define PB_USUAL(cond) \
    if (!(cond)) Py_RETURN_NONE

// (quantize_rows, linear_i8, group_rows, linear_grouped addresses)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 4 || !f_quantize) {
        if (n != 4) return PyErr_Format(PyExc_TypeError, "bind takes four addresses");
        f_quantize = reinterpret_cast<decltype(f_quantize)>(PyLong_AsVoidPtr(a[0]));
        f_linear_i8 = reinterpret_cast<decltype(f_linear_i8)>(PyLong_AsVoidPtr(a[1]));
        f_group = reinterpret_cast<decltype(f_group)>(PyLong_AsVoidPtr(a[2]));
        f_grouped = reinterpret_cast<decltype(f_grouped)>(PyLong_AsVoidPtr(a[3]));
    }
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// (x, codes, scale)
PyObject *quantize_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    PB_USUAL(n == 3 && f_quantize);
    const Tensor *x = tensor(a[0]), *codes = tensor(a[1]), *scale = tensor(a[2]);
    PB_USUAL(x && x->is_cuda() && x->dim() == 2);
    const int dev = (int)x->get_device();
    const int64_t m = x->size(0), k = x->size(1);
    PB_USUAL(float_matrix(x, dev, m, k) && matrix(codes, at::kChar, dev, m, k) && vector(scale, at::kFloat, dev, m) && k < (1ll << 31));
    return status(f_quantize(dev, stream_of(dev), x->data_ptr(), float_type(*x), (uint64_t)m, (uint32_t)k, (uint64_t)k, written(codes), (uint64_t)k,
                             static_cast<float *>(written(scale))));
}

// (x, x_scale, w, w_scale, bias or None, act, out)
PyObject *linear_i8(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    PB_USUAL(n_args == 7 && f_linear_i8);
    const Tensor *x = tensor(a[0]), *xs = tensor(a[1]), *w = tensor(a[2]), *ws = tensor(a[3]), *bias = a[4] == Py_None ? nullptr : tensor(a[4]), *out = tensor(a[6]);
    PB_USUAL(x && w && x->is_cuda() && x->dim() == 2 && w->dim() == 2 && (bias || a[4] == Py_None));
    const int dev = (int)x->get_device();
    const int64_t m = x->size(0), k = x->size(1), n = w->size(0);
    PB_USUAL(matrix(x, at::kChar, dev, m, k) && matrix(w, at::kChar, dev, n, k) && vector(xs, at::kFloat, dev, m) && vector(ws, at::kFloat, dev, n) &&
             (!bias || vector(bias, at::kFloat, dev, n)) && float_matrix(out, dev, m, n) && k < (1ll << 31) && n < (1ll << 31));
    const long act = PyLong_AsLong(a[5]);
    if (act == -1 && PyErr_Occurred()) return nullptr;
    return status(f_linear_i8(dev, stream_of(dev), x->data_ptr(), (uint64_t)k, floats(xs), w->data_ptr(), (uint64_t)k, floats(ws), floats(bias), (int)act,
                              written(out), float_type(*out), (uint64_t)n, (uint64_t)m, (uint32_t)n, (uint32_t)k));
}

// (group, groups, offsets, order)
PyObject *group_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    PB_USUAL(n == 4 && f_group);
    const Tensor *group = tensor(a[0]), *offsets = tensor(a[2]), *order = tensor(a[3]);
    PB_USUAL(group && group->is_cuda() && group->dim() == 1);
    const long groups = PyLong_AsLong(a[1]);
    if (groups == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    PB_USUAL(groups >= 1 && groups <= (long)PB_MAX_GROUPS);
    const int dev = (int)group->get_device();
    const int64_t m = group->size(0);
    PB_USUAL(vector(group, at::kInt, dev, m) && vector(offsets, at::kInt, dev, groups + 1) && vector(order, at::kInt, dev, m));
    return status(f_group(dev, stream_of(dev), ints(group), (uint64_t)m, (uint32_t)groups, static_cast<int *>(written(offsets)),
                          static_cast<int *>(written(order))));
}

// (x, w, offsets, x_rows or None, y_rows or None, x_scale or None, w_scale or None, bias or None, act, out)
PyObject *linear_grouped(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    PB_USUAL(n_args == 10 && f_grouped);
    const Tensor *x = tensor(a[0]), *w = tensor(a[1]), *offsets = tensor(a[2]), *out = tensor(a[9]);
    const Tensor *opt[5];  // x_rows, y_rows, x_scale, w_scale, bias
    for (int i = 0; i < 5; ++i) {
        opt[i] = a[3 + i] == Py_None ? nullptr : tensor(a[3 + i]);
        PB_USUAL(opt[i] || a[3 + i] == Py_None);
    }
    PB_USUAL(x && w && out && x->is_cuda() && x->dim() == 2 && w->dim() == 3 && out->dim() == 2);
    const int dev = (int)x->get_device();
    const bool i8 = x->scalar_type() == at::kChar;
    const int type = i8 ? PB_TYPE_I8 : float_type(*x);
    const int64_t x_total = x->size(0), k = x->size(1), groups = w->size(0), n = w->size(1), y_total = out->size(0);
    PB_USUAL(type >= 0 && matrix(x, x->scalar_type(), dev, x_total, k) && usual(w, x->scalar_type(), dev, 3) && w->size(2) == k && groups >= 1 &&
             groups <= (int64_t)PB_MAX_GROUPS && vector(offsets, at::kInt, dev, groups + 1) && float_matrix(out, dev, y_total, n));
    const int64_t m = opt[0] ? opt[0]->numel() : opt[1] ? opt[1]->numel() : x_total;
    PB_USUAL((!opt[0] || vector(opt[0], at::kInt, dev, m)) && (!opt[1] || vector(opt[1], at::kInt, dev, m)) && (opt[0] || m <= x_total) &&
             (opt[1] || m <= y_total));
    PB_USUAL(i8 ? vector(opt[2], at::kFloat, dev, x_total) && matrix(opt[3], at::kFloat, dev, groups, n) : !opt[2] && !opt[3]);
    PB_USUAL((!opt[4] || matrix(opt[4], at::kFloat, dev, groups, n)) && m > 0 && n > 0 && x_total > 0 && y_total > 0 && k < (1ll << 31) && n < (1ll << 31));
    const long act = PyLong_AsLong(a[8]);
    if (act == -1 && PyErr_Occurred()) return nullptr;
    return status(f_grouped(dev, stream_of(dev), type, x->data_ptr(), (uint64_t)x_total, (uint64_t)k, floats(opt[2]), w->data_ptr(), (uint64_t)k, floats(opt[3]),
                            floats(opt[4]), ints(offsets), (uint32_t)groups, ints(opt[0]), ints(opt[1]), (int)act, written(out), float_type(*out),
                            (uint64_t)y_total, (uint64_t)n, (uint64_t)m, (uint32_t)n, (uint32_t)k));
}

// a C++ exception does not leave a function that Python calls
template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    try {
        return F(self, a, n);
    } catch (const std::exception &e) {
        return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
    }
}

PyMethodDef methods[] = {{"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
                         {"quantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<quantize_rows>)), METH_FASTCALL, nullptr},
                         {"linear_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<linear_i8>)), METH_FASTCALL, nullptr},
                         {"group_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<group_rows>)), METH_FASTCALL, nullptr},
                         {"linear_grouped", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<linear_grouped>)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_linear_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__linear_call() {
    PyObject *m = PyModule_Create(&module);
    // torch's and Python's layouts are compiled in: linear.py takes this module only where they are the running ones
    if (m && PyModule_AddStringConstant(m, "built_for", PB_BUILT_FOR) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
