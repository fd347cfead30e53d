// CPython entries for the operators on logits and beams, whose kernels can be shorter
// than a call through ctypes (2.4 us for the 14 arguments of rnet_beam_select, 0.16 us
// here). The other functions go through ctypes; a line in `entries` adds one. Each is
// derived from the C function's own type: pointers from int or None, integers from int,
// floats from float or int. With any other argument, or another number of them, an
// entry returns NotImplemented and calls nothing.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "rnet_capi.h"

namespace {

// Whether `o` fits a parameter of type T, and its value.
template <class T>
bool take(PyObject* o, T& v) {
  if constexpr (std::is_pointer<T>::value) {
    if (o == Py_None) {
      v = nullptr;
      return true;
    }
    if (!PyLong_CheckExact(o)) return false;
    v = (T)(size_t)PyLong_AsUnsignedLongLongMask(o);
    return true;
  } else if constexpr (std::is_floating_point<T>::value) {
    if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
    const double d = PyFloat_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
    v = (T)d;
    return true;
  } else {
    if (!PyLong_CheckExact(o)) return false;
    int beyond = 0;
    const long long n = PyLong_AsLongLongAndOverflow(o, &beyond);
    v = (T)n;
    return !beyond && (long long)v == n && (std::is_signed<T>::value || n >= 0);
  }
}

template <auto F>
struct Entry;
template <class... A, int (*F)(A...)>
struct Entry<F> {
  template <size_t... I>
  static PyObject* run(PyObject* const* args, std::index_sequence<I...>) {
    std::tuple<A...> v;
    if (!(take(args[I], std::get<I>(v)) && ...)) Py_RETURN_NOTIMPLEMENTED;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = F(std::get<I>(v)...);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  }
  static PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != (Py_ssize_t)sizeof...(A)) Py_RETURN_NOTIMPLEMENTED;
    return run(args, std::index_sequence_for<A...>());
  }
};

#define ENTRY(f) {#f, (PyCFunction)(void (*)(void))Entry<f>::call, METH_FASTCALL, nullptr}
PyMethodDef entries[] = {
    ENTRY(rnet_topk_logits_forward),
    ENTRY(rnet_distill_topk_forward),
    ENTRY(rnet_beam_select),
    ENTRY(rnet_beam_reorder),
    ENTRY(rnet_beam_backtrack),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, entries,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
