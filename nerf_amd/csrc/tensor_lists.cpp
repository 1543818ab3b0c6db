// What the list entry points (gradient norm, clipping, optimizer step) need to know of a list of tensors, read in one
// pass.  From Python each attribute of each tensor costs 50 to 100 ns, about 0.3 us a tensor for a list that is only
// read and 2 us for an optimizer step's six lists: more than the kernels take on a network of some twenty tensors.
// Here it is 10 ns and 0.1 us, every call, with nothing remembered between calls.
//
//   describe(tensors)         -> (device index, pointers, element counts, types, dense): the middle three as bytes
//                                objects that the C ABI takes as arrays; dense: every tensor fills its stretch of
//                                memory without gaps or overlaps (in any order of dimensions)
//   optimizer(groups, state)  -> of the parameters of `groups` (a list of lists) that have a gradient: a list of those
//                                whose state (a dict of dicts) is not laid out yet; or, if there are none,
//                                (device index, parameters, tensors to keep until the launch, and as bytes objects the
//                                number per group and the nerf_adamw_tensors arrays param, grad, exp_avg, exp_avg_sq,
//                                master, step, numel, dtype)
//   is_dense(tensor)          -> bool
//   built_for                    versions of torch and Python whose headers the module was built with
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <vector>

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

// A Python object that is let go with its scope.
struct Held {
    PyObject* o;
    explicit Held(PyObject* x) : o(x) {}
    Held(const Held&) = delete;
    ~Held() { Py_XDECREF(o); }
};

PyObject* refuse(const char* what) {
    PyErr_SetString(PyExc_RuntimeError, what);
    return nullptr;
}

template <typename T>
PyObject* bytes_of(const std::vector<T>& v) {
    return PyBytes_FromStringAndSize((const char*)v.data(), v.size() * sizeof(T));
}

// The fp32 tensor `key` of a parameter's state, in the parameter's order -> its pointer; 0 with an error set.
uint64_t moment(PyObject* state, PyObject* key, const at::Tensor& p) {
    PyObject* o = PyDict_GetItemWithError(state, key);
    if (!o || !THPVariable_Check(o)) {
        PyErr_Format(PyExc_RuntimeError, "AdamW: the state of a parameter has no tensor %R", key);
        return 0;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() != at::kFloat || t.device() != p.device() || t.layout() != at::kStrided || t.sizes() != p.sizes() ||
        !same_order(t, p)) {
        PyErr_Format(PyExc_RuntimeError, "AdamW: state %R must be an fp32 tensor of its parameter's shape, order and device", key);
        return 0;
    }
    return t.numel() ? (uint64_t)t.mutable_data_ptr() : 1;      // (an empty tensor's pointer is never followed)
}

PyObject* optimizer(PyObject*, PyObject* args) {
    PyObject *groups, *state;
    if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &groups, &PyDict_Type, &state)) return nullptr;
    static PyObject *k_avg = PyUnicode_InternFromString("exp_avg"), *k_sq = PyUnicode_InternFromString("exp_avg_sq"),
                    *k_master = PyUnicode_InternFromString("master"), *k_step = PyUnicode_InternFromString("step");
    std::vector<uint64_t> p_, g_, m_, v_, w_, s_;
    std::vector<int64_t> numel;
    std::vector<int32_t> types, counts;
    long device = -1;
    bool half = false;
    Held params(PyList_New(0)), fresh(PyList_New(0)), keep(PyList_New(0));
    if (!params.o || !fresh.o || !keep.o) return nullptr;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(groups); ++k) {
        PyObject* group = PyList_GET_ITEM(groups, k);
        if (!check_list(group)) return nullptr;
        const size_t before = p_.size();
        size_t waiting = 0;
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(group); ++i) {
            PyObject* po = PyList_GET_ITEM(group, i);
            if (!THPVariable_Check(po)) return refuse("expected a list of tensors");
            const at::Tensor& grad = THPVariable_Unpack(po).grad();
            if (!grad.defined()) continue;
            const at::Tensor* pt = tensor_at(group, i);
            if (!pt) return nullptr;
            const at::Tensor& p = *pt;
            if (!p.is_cuda()) return refuse("nerf_amd kernels need tensors on a HIP device; got a CPU tensor");
            if (device >= 0 && p.get_device() != device) return refuse("nerf_amd kernels need the tensors of a list on one HIP device");
            device = p.get_device();
            const int type = type_code(p);
            if (type < 0)
                return PyErr_Format(PyExc_RuntimeError, "expected float32, bfloat16 or float16 tensors, got %s",
                                    at::toString(p.scalar_type()));
            if (!dense(p)) return refuse("AdamW: expected dense parameters (no gaps, no broadcast dimensions)");
            if (grad.layout() != at::kStrided || grad.is_neg() || grad.scalar_type() != p.scalar_type() ||
                grad.device() != p.device() || grad.sizes() != p.sizes())
                return refuse("AdamW: gradients must be strided tensors of their parameters' type, shape and device");
            PyObject* st = PyDict_GetItemWithError(state, po);
            if (!st && PyErr_Occurred()) return nullptr;
            if (st && !PyDict_Check(st)) return refuse("AdamW: the state of a parameter is no dict");
            if (!st || PyDict_GET_SIZE(st) == 0 || (type && !PyDict_GetItemWithError(st, k_master))) {
                if (PyList_Append(fresh.o, po)) return nullptr;
                ++waiting;
                continue;
            }
            const uint64_t m = moment(st, k_avg, p), v = m ? moment(st, k_sq, p) : 0;
            const uint64_t w = v && type ? moment(st, k_master, p) : 1;
            if (!m || !v || !w) return nullptr;
            PyObject* so = PyDict_GetItemWithError(st, k_step);
            if (!so || !THPVariable_Check(so)) return refuse("AdamW: the state of a parameter has no tensor 'step'");
            const at::Tensor& step = THPVariable_Unpack(so);
            if (step.scalar_type() != at::kFloat || step.device() != p.device() || step.layout() != at::kStrided || step.numel() != 1)
                return refuse("AdamW: state 'step' must be one fp32 number on its parameter's device");
            if (PyList_Append(params.o, po)) return nullptr;
            if (same_order(grad, p)) {
                g_.push_back((uint64_t)grad.mutable_data_ptr());
            } else {        // another order of the same entries: laid out as the parameter is
                c10::NoGradGuard no_grad;
                const at::Tensor copy = at::empty_like(p.detach(), at::TensorOptions(), at::MemoryFormat::Preserve).copy_(grad);
                if (!same_order(copy, p)) return refuse("AdamW: a gradient cannot be laid out as its parameter is");
                g_.push_back((uint64_t)copy.mutable_data_ptr());
                Held c(THPVariable_Wrap(copy));
                if (!c.o || PyList_Append(keep.o, c.o)) return nullptr;
            }
            p_.push_back((uint64_t)p.mutable_data_ptr());
            m_.push_back(m);
            v_.push_back(v);
            w_.push_back(type ? w : 0);
            s_.push_back((uint64_t)step.mutable_data_ptr());
            numel.push_back(p.numel());
            types.push_back(type);
            half = half || type;
        }
        counts.push_back((int32_t)(p_.size() - before + waiting));
    }
    if (PyList_GET_SIZE(fresh.o)) {
        Py_INCREF(fresh.o);
        return fresh.o;
    }
    Held c(bytes_of(counts)), p(bytes_of(p_)), g(bytes_of(g_)), m(bytes_of(m_)), v(bytes_of(v_)), w(bytes_of(w_)), s(bytes_of(s_)),
        n(bytes_of(numel)), t(bytes_of(types));
    if (!c.o || !p.o || !g.o || !m.o || !v.o || !w.o || !s.o || !n.o || !t.o) return nullptr;
    return Py_BuildValue("lOOOOOOOOOOO", device, params.o, keep.o, c.o, p.o, g.o, m.o, v.o, half ? w.o : Py_None, s.o, n.o, t.o);
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
    {"optimizer", guarded<optimizer>, METH_VARARGS, nullptr},
    {"is_dense", guarded<is_dense>, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists() {
    PyObject* m = PyModule_Create(&module);
    if (!m) return nullptr;
    PyObject* v = Py_BuildValue("(sN)", TORCH_VERSION, PyUnicode_FromFormat("%d.%d", PY_MAJOR_VERSION, PY_MINOR_VERSION));
    if (!v || PyModule_AddObject(m, "built_for", v)) {
        Py_XDECREF(v);
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
