// tensor_list.cpp — a Python list of tensors as a gc_grads (include/gcodec.h).
//
// A model has hundreds of gradients, new ones every step, and each attribute
// read from Python costs about 70 ns: sizes, pointers, types, layouts and the
// .grad of 161 parameters took 85 us of a 105 us clip_grad_norm_.  Read here
// they take 5.  Host code only; the module is loaded beside libgcodec.so.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <stdint.h>

#include <vector>

#include "gcodec.h"

namespace {

typedef int (*plan_fn)(const uint64_t *, const void *const *, const uint32_t *, uint64_t, uint64_t *, uint32_t *, gc_grads *);

// the tensor, or (of_grads) its gradient, which may be undefined
const at::Tensor *item(PyObject *o, bool of_grads)
{
    if (!THPVariable_Check(o))
        return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    return of_grads ? &t.grad() : &t;
}

// gather(tensors, of_grads, ordered, written, plan, grads): fills the gc_grads at
// the address `grads` by the gc_grads_plan at the address `plan`
// -> (device index, host records, order); None without any gradient.
// ordered: a tensor's elements are taken row by row (else in any dense order)
// written: they may be written or kept, so a copy-on-write tensor gets its own memory
PyObject *gather(PyObject *, PyObject *args)
{
    PyObject *list;
    int of_grads, ordered, written;
    unsigned long long plan, out;
    if (!PyArg_ParseTuple(args, "OpppKK", &list, &of_grads, &ordered, &written, &plan, &out))
        return nullptr;
    PyObject *seq = PySequence_Fast(list, "not a list of dense tensors");
    if (!seq)
        return nullptr;
    const Py_ssize_t all = PySequence_Fast_GET_SIZE(seq);
    std::vector<uint64_t> sizes;
    std::vector<const void *> ptrs;
    std::vector<uint32_t> types;
    PyObject *result = nullptr, *host = nullptr, *order = nullptr;
    try {
        sizes.reserve(all);
        ptrs.reserve(all);
        types.reserve(all);
        c10::Device device(c10::kCPU);
        for (Py_ssize_t i = 0; i < all; ++i) {
            const at::Tensor *t = item(PySequence_Fast_GET_ITEM(seq, i), of_grads);
            if (!t) {
                PyErr_Format(PyExc_ValueError, "not a list of dense tensors (entry %zd)", i);
                goto done;
            }
            if (!t->defined())
                continue;
            if (t->layout() != c10::kStrided) {
                PyErr_Format(PyExc_ValueError, "not a list of dense tensors (entry %zd is sparse)", i);
                goto done;
            }
            if (!t->is_cuda()) {
                PyErr_Format(PyExc_LookupError, "tensor %zd is on %s", i, t->device().str().c_str());
                goto done;
            }
            if (types.empty())
                device = t->device();
            else if (t->device() != device) {
                PyErr_SetString(PyExc_ValueError, "the tensors are on different devices");
                goto done;
            }
            const auto type = t->scalar_type();
            if (type != at::kFloat && type != at::kHalf && type != at::kBFloat16) {
                PyErr_Format(PyExc_ValueError, "tensor %zd (%s) is not float32, float16 or bfloat16", i,
                             c10::toString(type));
                goto done;
            }
            if (!t->is_contiguous() && (ordered || !t->is_non_overlapping_and_dense())) {
                PyErr_Format(PyExc_ValueError, "tensor %zd is not %s", i, ordered ? "contiguous" : "dense");
                goto done;
            }
            if (t->is_conj() || t->is_neg()) {
                PyErr_Format(PyExc_ValueError, "tensor %zd is a lazily negated view", i);
                goto done;
            }
            sizes.push_back((uint64_t)t->numel());
            ptrs.push_back(written ? t->mutable_data_ptr() : t->const_data_ptr());
            types.push_back(type == at::kFloat ? GC_F32 : type == at::kHalf ? GC_F16 : GC_BF16);
        }
        if (types.empty()) {
            Py_INCREF(Py_None);
            result = Py_None;
            goto done;
        }
        const size_t count = types.size();
        host = PyBytes_FromStringAndSize(nullptr, (Py_ssize_t)(16 * (count + 1)));
        order = PyBytes_FromStringAndSize(nullptr, (Py_ssize_t)(4 * count));
        if (!host || !order)
            goto done;
        if (reinterpret_cast<plan_fn>(plan)(sizes.data(), ptrs.data(), types.data(), count,
                                            reinterpret_cast<uint64_t *>(PyBytes_AS_STRING(host)),
                                            reinterpret_cast<uint32_t *>(PyBytes_AS_STRING(order)),
                                            reinterpret_cast<gc_grads *>(out)) != GC_OK) {
            PyErr_SetString(PyExc_RuntimeError, "gc_grads_plan");
            goto done;
        }
        result = Py_BuildValue("iOO", (int)device.index(), host, order);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
done:
    Py_XDECREF(host);
    Py_XDECREF(order);
    Py_DECREF(seq);
    return result;
}

// written(tensors, of_grads): tells autograd of a write to them
PyObject *written(PyObject *, PyObject *args)
{
    PyObject *list;
    int of_grads;
    if (!PyArg_ParseTuple(args, "Op", &list, &of_grads))
        return nullptr;
    PyObject *seq = PySequence_Fast(list, "not a list of tensors");
    if (!seq)
        return nullptr;
    try {
        for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); ++i) {
            const at::Tensor *t = item(PySequence_Fast_GET_ITEM(seq, i), of_grads);
            if (t && t->defined() && !t->is_inference())  // inference tensors have no version
                t->unsafeGetTensorImpl()->bump_version();
        }
    } catch (const std::exception &e) {
        Py_DECREF(seq);
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    Py_DECREF(seq);
    Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {{"gather", gather, METH_VARARGS, nullptr},
                          {"written", written, METH_VARARGS, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tensor_list", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_list(void) { return PyModule_Create(&kModule); }
