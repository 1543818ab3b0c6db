// What the list entry points (gradient norm, clipping, optimizer step) need to know of a list of tensors, read in one
// pass.  From Python each attribute of each tensor costs 50 to 100 ns, about 0.3 us a tensor for a list that is only
// read and 2 us for an optimizer step's six lists: more than the kernels take on a network of some twenty tensors.
// Here it is about 10 ns a tensor, every call, with nothing remembered between calls.
//
//   describe(tensors)             -> (device index, pointers, element counts, types, dense): the middle three as bytes
//                                    objects that the C ABI takes as arrays; dense: every tensor fills its stretch of
//                                    memory without gaps or overlaps (in any order of dimensions)
//   match(tensors, like, fp32)    -> pointers of `tensors` (0 for None), each of the shape, device and order of its
//                                    partner in `like`, and of its type or, with fp32, float32; None if an order differs
//   is_dense(tensor)              -> bool
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

namespace {

// include/nerf_amd.h: NERF_F32, NERF_BF16, NERF_F16
int type_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}

bool dense(const at::Tensor& t) { return t.unsafeGetTensorImpl()->is_non_overlapping_and_dense_or_false(); }

// Whether the entries of two tensors of one shape lie in the same order (dimensions of one entry have no say in it).
bool same_order(const at::Tensor& a, const at::Tensor& b) {
    for (int64_t d = 0; d < a.dim(); ++d)
        if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return a.numel() == 0;
    return true;
}

const at::Tensor* tensor_at(PyObject* list, Py_ssize_t i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "expected a list of tensors");
        return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.layout() != at::kStrided || !t.has_storage() || t.is_neg()) {
        PyErr_SetString(PyExc_RuntimeError, "expected plain strided tensors (not sparse, no lazily negated views)");
        return nullptr;
    }
    return &t;
}

bool check_list(PyObject* list) {
    if (PyList_Check(list)) return true;
    PyErr_SetString(PyExc_TypeError, "expected a list of tensors");
    return false;
}

PyObject* describe(PyObject*, PyObject* list) {
    if (!check_list(list)) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(list);
    PyObject* ptrs = PyBytes_FromStringAndSize(nullptr, n * 8);
    PyObject* numels = PyBytes_FromStringAndSize(nullptr, n * 8);
    PyObject* types = PyBytes_FromStringAndSize(nullptr, n * 4);
    long device = -1;
    bool all_dense = true, ok = ptrs && numels && types;
    for (Py_ssize_t i = 0; i < n && ok; ++i) {
        const at::Tensor* t = tensor_at(list, i);
        if (!(ok = t != nullptr)) break;
        if (!t->is_cuda()) {
            PyErr_SetString(PyExc_RuntimeError, i ? "nerf_amd kernels need the tensors of a list on one HIP device"
                                                  : "nerf_amd kernels need tensors on a HIP device; got a CPU tensor");
            ok = false;
        } else if (i && t->get_device() != device) {
            PyErr_SetString(PyExc_RuntimeError, "nerf_amd kernels need the tensors of a list on one HIP device");
            ok = false;
        } else if (type_code(*t) < 0) {
            PyErr_Format(PyExc_RuntimeError, "expected float32, bfloat16 or float16 tensors, got %s", at::toString(t->scalar_type()));
            ok = false;
        } else {
            device = t->get_device();
            all_dense = all_dense && dense(*t);
            ((uint64_t*)PyBytes_AS_STRING(ptrs))[i] = (uint64_t)t->mutable_data_ptr();
            ((int64_t*)PyBytes_AS_STRING(numels))[i] = t->numel();
            ((int32_t*)PyBytes_AS_STRING(types))[i] = type_code(*t);
        }
    }
    PyObject* r = ok ? Py_BuildValue("lOOOO", device, ptrs, numels, types, all_dense ? Py_True : Py_False) : nullptr;
    Py_XDECREF(ptrs);
    Py_XDECREF(numels);
    Py_XDECREF(types);
    return r;
}

PyObject* match(PyObject*, PyObject* args) {
    PyObject *list, *like;
    int fp32;
    if (!PyArg_ParseTuple(args, "OOp", &list, &like, &fp32) || !check_list(list) || !check_list(like)) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(list);
    if (PyList_GET_SIZE(like) != n) {
        PyErr_SetString(PyExc_ValueError, "lists of different lengths");
        return nullptr;
    }
    PyObject* ptrs = PyBytes_FromStringAndSize(nullptr, n * 8);
    if (!ptrs) return nullptr;
    bool ordered = true;
    for (Py_ssize_t i = 0; i < n; ++i) {
        uint64_t* at = (uint64_t*)PyBytes_AS_STRING(ptrs) + i;
        if (PyList_GET_ITEM(list, i) == Py_None) {
            *at = 0;
            continue;
        }
        const at::Tensor *t = tensor_at(list, i), *l = tensor_at(like, i);
        if (!t || !l) {
            Py_DECREF(ptrs);
            return nullptr;
        }
        if (t->device() != l->device() || t->scalar_type() != (fp32 ? at::kFloat : l->scalar_type()) || t->sizes() != l->sizes()) {
            Py_DECREF(ptrs);
            return PyErr_Format(PyExc_RuntimeError, "expected %s tensors of their parameters' shape and device",
                                fp32 ? "fp32" : "same-type");
        }
        ordered = ordered && same_order(*t, *l);
        *at = (uint64_t)t->mutable_data_ptr();
    }
    if (!ordered) {
        Py_DECREF(ptrs);
        Py_RETURN_NONE;
    }
    return ptrs;
}

PyObject* is_dense(PyObject*, PyObject* o) {
    if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "expected a tensor");
        return nullptr;
    }
    return PyBool_FromLong(dense(THPVariable_Unpack(o)));
}

// No C++ exception may pass into the interpreter.
template <PyObject* (*F)(PyObject*, PyObject*)>
PyObject* guarded(PyObject* self, PyObject* arg) {
    try {
        return F(self, arg);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {
    {"describe", guarded<describe>, METH_O, nullptr},
    {"match", guarded<match>, METH_VARARGS, nullptr},
    {"is_dense", guarded<is_dense>, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists() { return PyModule_Create(&module); }
