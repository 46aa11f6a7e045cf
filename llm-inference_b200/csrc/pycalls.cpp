// Python calls of the paged cache's entry points (include/b200attn.h) without
// ctypes: a call of 24 arguments spends 13 us in ctypes and in taking the
// tensors' addresses in Python, more than the smallest kernels run; here it
// takes about 2. The arguments are converted by the C declarations' types:
// device pointers from a tensor (its data_ptr(); host tensors are refused, so
// are those of another device than the current one, which the kernels could not
// read), an int or None; streams from a torch stream (its cuda_stream), an int
// or None.
//
// The module does not link the library: bind(name, address) gives it the
// functions of the one that _lib.py has loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <string_view>
#include <tuple>
#include <utility>

#include "b200attn.h"

namespace {

PyObject* s_is_cuda;
PyObject* s_get_device;
PyObject* s_data_ptr;
PyObject* s_cuda_stream;

int (*fn_current_device)(void) = nullptr;
constexpr int kNotAsked = -2;
thread_local int current_device = kNotAsked;  // in this call

// A host tensor is refused, so is one of another device. Objects that know neither pass.
bool on_current_device(PyObject* o) {
    PyObject* d = PyObject_CallMethodNoArgs(o, s_get_device);
    long device = -1;
    if (d != nullptr) {
        device = PyLong_AsLong(d);
        Py_DECREF(d);
        if (device == -1 && PyErr_Occurred()) return false;
    } else if (PyErr_ExceptionMatches(PyExc_AttributeError)) {
        PyErr_Clear();
        PyObject* cuda = PyObject_GetAttr(o, s_is_cuda);
        if (cuda == nullptr) {
            if (!PyErr_ExceptionMatches(PyExc_AttributeError)) return false;
            PyErr_Clear();
            return true;
        }
        const bool host = cuda == Py_False;
        Py_DECREF(cuda);
        if (!host) return true;
    } else {
        return false;
    }
    if (device < 0) {
        PyErr_SetString(PyExc_ValueError, "b200attn launchers take device buffers; got a host tensor");
        return false;
    }
    if (current_device == kNotAsked) current_device = fn_current_device ? fn_current_device() : -1;
    if (device == current_device) return true;
    PyErr_Format(PyExc_ValueError, "a tensor lies on device %ld, the current device is %d", device, current_device);
    return false;
}

bool convert(PyObject* o, void*& out) {
    if (o == Py_None) {
        out = nullptr;
        return true;
    }
    if (PyLong_Check(o)) {
        out = PyLong_AsVoidPtr(o);
        return out != nullptr || !PyErr_Occurred();
    }
    if (!on_current_device(o)) return false;
    PyObject* p = PyObject_CallMethodNoArgs(o, s_data_ptr);
    if (p == nullptr) {
        if (PyErr_ExceptionMatches(PyExc_AttributeError)) {
            PyErr_Clear();
            PyErr_Format(PyExc_TypeError, "expected a device tensor or int pointer, got %R", Py_TYPE(o));
        }
        return false;
    }
    out = PyLong_AsVoidPtr(p);
    Py_DECREF(p);
    return out != nullptr || !PyErr_Occurred();
}

template <typename T>
bool convert(PyObject* o, T*& out) {
    void* p = nullptr;
    if (!convert(o, p)) return false;
    out = static_cast<T*>(p);
    return true;
}

bool convert(PyObject* o, b2_stream_t& out) {
    if (o == Py_None || PyLong_Check(o)) {
        out = o == Py_None ? nullptr : static_cast<b2_stream_t>(PyLong_AsVoidPtr(o));
        return out != nullptr || !PyErr_Occurred();
    }
    PyObject* p = PyObject_GetAttr(o, s_cuda_stream);
    if (p == nullptr) return false;
    out = static_cast<b2_stream_t>(PyLong_AsVoidPtr(p));
    Py_DECREF(p);
    return out != nullptr || !PyErr_Occurred();
}

bool convert(PyObject* o, size_t& out) {
    out = PyLong_AsSize_t(o);
    return out != static_cast<size_t>(-1) || !PyErr_Occurred();
}

bool convert(PyObject* o, int32_t& out) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) return false;
    if (v < INT32_MIN || v > INT32_MAX) {
        PyErr_SetString(PyExc_OverflowError, "int32 argument out of range");
        return false;
    }
    out = static_cast<int32_t>(v);
    return true;
}

bool convert(PyObject* o, bool& out) {
    const int v = PyObject_IsTrue(o);
    out = v > 0;
    return v >= 0;
}

template <typename... A, size_t... I>
PyObject* call(int (*fn)(A...), const char* name, PyObject* const* args, Py_ssize_t n, std::index_sequence<I...>) {
    if (fn == nullptr) {
        PyErr_Format(PyExc_RuntimeError, "%s is not bound", name);
        return nullptr;
    }
    if (n != static_cast<Py_ssize_t>(sizeof...(A))) {
        PyErr_Format(PyExc_TypeError, "%s takes %d arguments (%d given)", name, static_cast<int>(sizeof...(A)),
                     static_cast<int>(n));
        return nullptr;
    }
    current_device = kNotAsked;
    std::tuple<A...> v{};
    if (!(convert(args[I], std::get<I>(v)) && ...)) return nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = fn(std::get<I>(v)...);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

template <typename... A>
PyObject* call(int (*fn)(A...), const char* name, PyObject* const* args, Py_ssize_t n) {
    return call(fn, name, args, n, std::index_sequence_for<A...>{});
}

#define B2_CALLS(X)                              \
    X(b2_launch_rope_and_store_kv_paged)         \
    X(b2_launch_causal_attention_decode_paged)   \
    X(b2_launch_decode_step_paged_fused)         \
    X(b2_launch_kv_pages_copy)                   \
    X(b2_launch_kv_pages_truncate)               \
    X(b2_launch_kv_pages_fork)                   \
    X(b2_launch_kv_pages_extend)                 \
    X(b2_launch_kv_pages_compact)

#define B2_CALL(name)                                                                \
    decltype(&::name) fn_##name = nullptr;                                           \
    PyObject* py_##name(PyObject*, PyObject* const* args, Py_ssize_t n) {            \
        return call(fn_##name, #name, args, n);                                      \
    }
B2_CALLS(B2_CALL)

PyObject* bind(PyObject*, PyObject* args) {
    const char* name = nullptr;
    PyObject* address = nullptr;
    if (!PyArg_ParseTuple(args, "sO", &name, &address)) return nullptr;
    void* p = PyLong_AsVoidPtr(address);
    if (p == nullptr) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null function");
        return nullptr;
    }
    if (std::string_view(name) == "b2_current_device") {
        fn_current_device = reinterpret_cast<int (*)(void)>(p);
        Py_RETURN_NONE;
    }
#define B2_BIND(f)                                          \
    if (std::string_view(name) == #f) {                     \
        fn_##f = reinterpret_cast<decltype(fn_##f)>(p);     \
        Py_RETURN_NONE;                                     \
    }
    B2_CALLS(B2_BIND)
    PyErr_Format(PyExc_KeyError, "%s", name);
    return nullptr;
}

#define B2_DEF(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##f)), METH_FASTCALL, nullptr},
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "bind(name, address): the function that calls of name go to"},
                         B2_CALLS(B2_DEF) {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "calls of libb200attn.so without ctypes", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) {
    s_is_cuda = PyUnicode_InternFromString("is_cuda");
    s_get_device = PyUnicode_InternFromString("get_device");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_cuda_stream = PyUnicode_InternFromString("cuda_stream");
    if (!s_is_cuda || !s_get_device || !s_data_ptr || !s_cuda_stream) return nullptr;
    PyObject* m = PyModule_Create(&module);
    if (m == nullptr) return nullptr;
    PyObject* names = Py_BuildValue("[" 
#define B2_S(f) "s"
        B2_CALLS(B2_S)
#undef B2_S
        "]"
#define B2_N(f) , #f
        B2_CALLS(B2_N)
#undef B2_N
    );
    if (names == nullptr || PyModule_AddObject(m, "NAMES", names) != 0) return nullptr;
    return m;
}
