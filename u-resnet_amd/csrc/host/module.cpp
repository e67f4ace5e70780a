#include "host.h"

#include <c10/util/Exception.h>
#include <torch/csrc/Exceptions.h>

#include <exception>
#include <stdexcept>
#include <type_traits>

EntryPoints entry = {};

namespace {

PyObject* error_type = nullptr;

PyObject* set_error_type(PyObject*, PyObject* type) {
    Py_INCREF(type);
    Py_XDECREF(error_type);
    error_type = type;
    Py_RETURN_NONE;
}

// entry points by name, as addresses
PyObject* set_entry_points(PyObject*, PyObject* found) {
    const auto take = [&](const char* name, auto& to) {
        PyObject* v = PyDict_GetItemString(found, name);
        if (!v) { PyErr_Format(PyExc_KeyError, "no entry point %s", name); return false; }
        to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(PyLong_AsUnsignedLongLong(v));
        return !PyErr_Occurred();
    };
    if (!PyDict_Check(found)) return fail("entry points: a dict is expected");
    if (!(take("ur_gn_fwd_workspace", entry.gn_fwd_workspace) && take("ur_gn_bwd_workspace", entry.gn_bwd_workspace) &&
          take("ur_gn_act_fwd", entry.gn_act_fwd) && take("ur_gn_act_bwd", entry.gn_act_bwd) &&
          take("ur_param_table_max_rows", entry.param_table_max_rows) && take("ur_param_table_bytes", entry.param_table_bytes) &&
          take("ur_param_table", entry.param_table) && take("ur_grad_sqnorm_max_parts", entry.grad_sqnorm_max_parts) &&
          take("ur_grad_sqnorm", entry.grad_sqnorm) && take("ur_grad_clip", entry.grad_clip) && take("ur_adamw_multi", entry.adamw_multi) &&
          take("ur_last_error", entry.last_error)))
        return nullptr;
    Py_RETURN_NONE;
}

// C++ exceptions become Python ones: Python's own (out of a saved-tensor hook; activation checkpointing stops by one) and torch's
// for memory as they are, others the package's
template <PyObject* (*F)(PyObject*, PyObject*)>
PyObject* guarded(PyObject* self, PyObject* args) {
    try {
        return F(self, args);
    } catch (python_error& e) {
        e.restore();
        return PyErr_Occurred() ? nullptr : fail("a Python callback failed");
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");
        PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        if (type) PyErr_SetString(type, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch);
        return nullptr;
    } catch (const std::exception& e) {
        return fail(e.what());
    }
}

PyMethodDef methods[] = {{"adamw_step", guarded<adamw_step>, METH_VARARGS, "one AdamW step over parameter groups"},
                         {"holds", guarded<holds>, METH_VARARGS, "whether a dict of dicts still holds the same objects"},
                         {"clip_grads", guarded<clip_grads>, METH_VARARGS, "gradients scaled to a norm"},
                         {"gn_act", guarded<gn_act>, METH_VARARGS, "group norm with an activation, with its gradient"},
                         {"set_error_type", set_error_type, METH_O, "exception type for refused tensors"},
                         {"set_entry_points", set_entry_points, METH_O, "addresses of the kernel library"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyObject* fail(const std::string& text) {
    PyErr_SetString(error_type ? error_type : PyExc_RuntimeError, text.c_str());
    return nullptr;
}

void check(int status, const char* what) {
    if (status) throw std::runtime_error(std::string(what) + " failed: " + entry.last_error());
}

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
