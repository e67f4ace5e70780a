#include "host.h"

#include <exception>

EntryPoints entry = {};

namespace {

PyObject* error_type = nullptr;

PyObject* set_error_type(PyObject*, PyObject* type) {
    Py_INCREF(type);
    Py_XDECREF(error_type);
    error_type = type;
    Py_RETURN_NONE;
}

// addresses in the order of EntryPoints
PyObject* set_entry_points(PyObject*, PyObject* args) {
    unsigned long long a[5];
    if (!PyArg_ParseTuple(args, "KKKKK", &a[0], &a[1], &a[2], &a[3], &a[4])) return nullptr;
    entry.gn_fwd_workspace = reinterpret_cast<decltype(entry.gn_fwd_workspace)>(a[0]);
    entry.gn_bwd_workspace = reinterpret_cast<decltype(entry.gn_bwd_workspace)>(a[1]);
    entry.gn_act_fwd = reinterpret_cast<decltype(entry.gn_act_fwd)>(a[2]);
    entry.gn_act_bwd = reinterpret_cast<decltype(entry.gn_act_bwd)>(a[3]);
    entry.last_error = reinterpret_cast<decltype(entry.last_error)>(a[4]);
    Py_RETURN_NONE;
}

// C++ exceptions become Python ones
template <PyObject* (*F)(PyObject*, PyObject*)>
PyObject* guarded(PyObject* self, PyObject* args) {
    try {
        return F(self, args);
    } catch (const std::exception& e) {
        return fail(e.what());
    }
}

PyMethodDef methods[] = {{"adamw_rows", guarded<adamw_rows>, METH_VARARGS, "addresses of parameters and gradients"},
                         {"clip_rows", guarded<clip_rows>, METH_O, "addresses and sizes of gradients"},
                         {"gn_act", guarded<gn_act>, METH_VARARGS, "group norm with an activation, with its gradient"},
                         {"set_error_type", set_error_type, METH_O, "exception type for refused tensors"},
                         {"set_entry_points", set_entry_points, METH_VARARGS, "addresses of the kernel library"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyObject* fail(const std::string& text) {
    PyErr_SetString(error_type ? error_type : PyExc_RuntimeError, text.c_str());
    return nullptr;
}

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
