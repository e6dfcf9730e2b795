// Host side of the small operators' Python calls: a decode step's kernels run for a few
// microseconds, and reading eight tensors' shapes, strides, types and devices from Python and
// handing 24 arguments to the C ABI one by one takes as long.
//
//   form(*tensors) -> bytes   what a call's checks depend on, as a dictionary key (None: no tensor)
//   kv_io, attn_q4, qk_norm_rope(plan, tensors..., numbers..., stream) -> status
//       the C function that the plan names, with the plan's sizes and the tensors' pointers
//
// A plan is the bytes of the struct below that fits the call, packed by the caller after its
// checks of the tensors' form; pointers are never part of one.
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <exception>
#include <limits>

namespace {

struct IoPlan {                    // "<Q6q6iIi"
    unsigned long long fn;
    long long strides[6];
    int dims[6];
    unsigned flags;
    int unused;
};
struct AttnPlan {                  // "<Q8iIi"
    unsigned long long fn;
    int dims[8];
    unsigned flags;
    int unused;
};
struct RopePlan {                  // "<Q12q6iIi"
    unsigned long long fn;
    long long strides[12];
    int dims[6];
    unsigned flags;
    int unused;
};

using IoFn = int (*)(const void*, const void*, const void*, const void*, int, int, int, int, int, int,
                     const long long*, unsigned, void*);
using AttnFn = int (*)(const void*, const void*, const int*, const int*, void*, float*, float*, int, int, int, int, int,
                       int, int, int, float, unsigned, void*, size_t, void*);
using RopeFn = int (*)(const void*, const void*, const void*, const void*, void*, void*, const int*, const float*, int,
                       int, int, int, int, int, float, float, float, const long long*, unsigned, void*);

struct PyFailure {};               // a Python exception is set

const at::Tensor& tensor(PyObject* o) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "expected a torch.Tensor, got %.100s", Py_TYPE(o)->tp_name);
        throw PyFailure();
    }
    return THPVariable_Unpack(o);
}
void* ptr(PyObject* o) { return o == Py_None ? nullptr : tensor(o).data_ptr(); }

template <class T>
T plan(PyObject* o) {
    char* s;
    Py_ssize_t n;
    T p;
    if (PyBytes_AsStringAndSize(o, &s, &n) < 0) throw PyFailure();
    if (n != static_cast<Py_ssize_t>(sizeof(T))) {
        PyErr_SetString(PyExc_ValueError, "not a plan of this call");
        throw PyFailure();
    }
    std::memcpy(&p, s, sizeof p);
    return p;
}
void* stream(PyObject* o) {
    void* s = PyLong_AsVoidPtr(o);
    if (PyErr_Occurred()) throw PyFailure();
    return s;
}
float number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (PyErr_Occurred()) throw PyFailure();
    return static_cast<float>(v);
}

// Runs f(args) with n arguments; C++ exceptions become Python's.
template <class F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
    try {
        if (want >= 0 && n != want) {
            PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
            return nullptr;
        }
        return f();
    } catch (const PyFailure&) {
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// The lock is free during a launch, which waits when the device's queue is full.
template <class F>
PyObject* status(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* form(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, -1, [&] {
        std::string key;
        key.reserve(1024);
        for (Py_ssize_t i = 0; i < n; ++i) {
            if (a[i] == Py_None) {
                key.push_back('-');
                continue;
            }
            const at::Tensor& t = tensor(a[i]);
            const char head[5] = {'t', static_cast<char>(t.scalar_type()), static_cast<char>(t.device().type()),
                                  static_cast<char>(t.device().index()), static_cast<char>(t.dim())};
            key.append(head, sizeof head);
            key.append(reinterpret_cast<const char*>(t.sizes().data()), t.dim() * sizeof(int64_t));
            key.append(reinterpret_cast<const char*>(t.strides().data()), t.dim() * sizeof(int64_t));
        }
        return PyBytes_FromStringAndSize(key.data(), static_cast<Py_ssize_t>(key.size()));
    });
}

// (plan, four tensors in the C function's order, stream)
PyObject* kv_io(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 6, [&] {
        const IoPlan p = plan<IoPlan>(a[0]);
        void *x[4], *s = stream(a[5]);
        for (int i = 0; i < 4; ++i) x[i] = ptr(a[1 + i]);
        return status([&] {
            return reinterpret_cast<IoFn>(p.fn)(x[0], x[1], x[2], x[3], p.dims[0], p.dims[1], p.dims[2], p.dims[3], p.dims[4],
                                                p.dims[5], p.strides, p.flags, s);
        });
    });
}

// (plan, q, cache, block_table, seq_lens, out, Mi, Li, scale, workspace, stream)
PyObject* attn_q4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&] {
        const AttnPlan p = plan<AttnPlan>(a[0]);
        void *x[7], *ws = ptr(a[9]), *s = stream(a[10]);
        for (int i = 0; i < 7; ++i) x[i] = ptr(a[1 + i]);
        const size_t ws_bytes = a[9] == Py_None ? 0 : tensor(a[9]).nbytes();
        // None is the C function's 0, the default; a number that is 0 in fp32 becomes its smallest one, with which every
        // score is as good as 0.
        float scale = 0.0f;
        if (a[8] != Py_None && (scale = number(a[8])) == 0.0f) scale = std::numeric_limits<float>::denorm_min();
        return status([&] {
            return reinterpret_cast<AttnFn>(p.fn)(x[0], x[1], static_cast<int*>(x[2]), static_cast<int*>(x[3]), x[4],
                                                  static_cast<float*>(x[5]), static_cast<float*>(x[6]), p.dims[0], p.dims[1],
                                                  p.dims[2], p.dims[3], p.dims[4], p.dims[5], p.dims[6], p.dims[7], scale,
                                                  p.flags, ws, ws_bytes, s);
        });
    });
}

// (plan, q, k, q_weight, k_weight, q_out, k_out, positions, inv_freq, theta, rot_scale, eps, stream)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 13, [&] {
        const RopePlan p = plan<RopePlan>(a[0]);
        void *x[8], *s = stream(a[12]);
        for (int i = 0; i < 8; ++i) x[i] = ptr(a[1 + i]);
        const float theta = number(a[9]), rot_scale = number(a[10]), eps = number(a[11]);
        return status([&] {
            return reinterpret_cast<RopeFn>(p.fn)(x[0], x[1], x[2], x[3], x[4], x[5], static_cast<int*>(x[6]),
                                                  static_cast<float*>(x[7]), p.dims[0], p.dims[1], p.dims[2], p.dims[3],
                                                  p.dims[4], p.dims[5], theta, rot_scale, eps, p.strides, p.flags, s);
        });
    });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<form>("form"), method<kv_io>("kv_io"), method<attn_q4>("attn_q4"),
                         method<qk_norm_rope>("qk_norm_rope"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kf_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kf_host() { return PyModule_Create(&module); }
