// The host module (_host): what a step does per tensor or per call outside the kernels, where the interpreter would cost more
// than the launch.  Host code only, against torch's C++ interface; the kernels are reached through the C ABI, whose addresses
// the loader hands over (set_entry_points), so that one library serves both.
#pragma once
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../../include/uresnet_hip.h"

struct EntryPoints {
    decltype(&ur_gn_fwd_workspace) gn_fwd_workspace;
    decltype(&ur_gn_bwd_workspace) gn_bwd_workspace;
    decltype(&ur_gn_act_fwd) gn_act_fwd;
    decltype(&ur_gn_act_bwd) gn_act_bwd;
    decltype(&ur_param_table_max_rows) param_table_max_rows;
    decltype(&ur_param_table_bytes) param_table_bytes;
    decltype(&ur_param_table) param_table;
    decltype(&ur_grad_sqnorm_max_parts) grad_sqnorm_max_parts;
    decltype(&ur_grad_sqnorm) grad_sqnorm;
    decltype(&ur_grad_clip) grad_clip;
    decltype(&ur_adamw_multi) adamw_multi;
    decltype(&ur_last_error) last_error;
};
extern EntryPoints entry;

PyObject* fail(const std::string& text);                   // raises the package's error type
void check(int status, const char* what);                  // throws with the entry point's message
PyObject* adamw_step(PyObject* self, PyObject* args);
PyObject* holds(PyObject* self, PyObject* args);
PyObject* clip_grads(PyObject* self, PyObject* args);
PyObject* gn_act(PyObject* self, PyObject* args);
