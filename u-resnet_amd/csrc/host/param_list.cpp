// Reads lists of parameters for the multi-tensor optimiser entry points: addresses and sizes of parameters and gradients as
// arrays, with the checks that the kernels rely on.  Host code only; a call per step instead of some ten interpreter calls per
// parameter (134 tensors: 130 us -> 3 us).
#include "host.h"

#include <algorithm>
#include <utility>
#include <vector>

namespace {

std::string told(const at::Tensor& t) {
    return std::string(c10::toString(t.layout())) + " " + c10::toString(t.scalar_type()) + " on " + t.device().str();
}

bool plain_gpu_f32(const at::Tensor& g, c10::Device device) {
    return g.layout() == c10::kStrided && g.scalar_type() == at::kFloat && g.device() == device && device.is_cuda();
}

PyObject* bytes_of(const std::vector<long long>& v) {
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(v.data()), (Py_ssize_t)(v.size() * sizeof(long long)));
}

bool get_tensor(PyObject* o, at::Tensor& out) {
    if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "a list of tensors is expected");
        return false;
    }
    out = THPVariable_Unpack(o);
    return true;
}

}  // namespace

// adamw_rows(params, sizes, grads or None) -> (params, grads, live, uneven): addresses as int64 arrays; a parameter without
// gradient has a zero.  live: how many have one.  uneven: whether a gradient is not contiguous (its address is left zero).
// sizes: int64 array of the element counts that the state was made for.
PyObject* adamw_rows(PyObject*, PyObject* args) {
    PyObject *params, *sizes, *grads;
    if (!PyArg_ParseTuple(args, "O!SO", &PyList_Type, &params, &sizes, &grads)) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(params);
    if (PyBytes_GET_SIZE(sizes) != (Py_ssize_t)(n * sizeof(long long)) || (grads != Py_None && (!PyList_Check(grads) || PyList_GET_SIZE(grads) != n)))
        return fail("AdamW: lists of different lengths");
    const long long* want = reinterpret_cast<const long long*>(PyBytes_AS_STRING(sizes));
    std::vector<long long> ps(n, 0), gs(n, 0);
    long long live = 0;
    bool uneven = false;
    for (Py_ssize_t i = 0; i < n; ++i) {
        at::Tensor p, g;
        if (!get_tensor(PyList_GET_ITEM(params, i), p)) return nullptr;
        if (grads == Py_None) g = p.grad();
        else if (PyList_GET_ITEM(grads, i) != Py_None && !get_tensor(PyList_GET_ITEM(grads, i), g)) return nullptr;
        if (!g.defined()) continue;
        if (!p.device().is_cuda()) return fail("AdamW: parameters must be on a GPU (got " + p.device().str() + ")");
        if (!plain_gpu_f32(g, p.device())) return fail("AdamW: gradients must be dense fp32 tensors on the parameter's GPU (got " + told(g) + ")");
        if (p.layout() != c10::kStrided || p.scalar_type() != at::kFloat || !p.is_contiguous() || p.numel() != want[i] || g.numel() != want[i])
            return fail("AdamW: a parameter changed its size, layout or type");
        ++live;
        if (!g.is_contiguous()) { uneven = true; continue; }
        ps[i] = (long long)p.data_ptr();
        gs[i] = (long long)g.data_ptr();
    }
    return Py_BuildValue("NNLO", bytes_of(ps), bytes_of(gs), live, uneven ? Py_True : Py_False);
}

// clip_rows(params) -> (grads, sizes, count, device index), the gradients that have elements; device index -1: no gradient
PyObject* clip_rows(PyObject*, PyObject* params) {
    if (!PyList_Check(params)) return fail("clip_grad_norm_: a list is expected");
    std::vector<long long> gs, ns;
    int device = -1;
    c10::Device first(c10::kCPU);
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); ++i) {
        at::Tensor p;
        if (!get_tensor(PyList_GET_ITEM(params, i), p)) return nullptr;
        const at::Tensor g = p.grad();
        if (!g.defined()) continue;
        if (device < 0) { first = g.device(); device = first.is_cuda() ? first.index() : 0; }
        if (!plain_gpu_f32(g, first)) return fail("clip_grad_norm_: gradients must be dense fp32 tensors on one GPU (got " + told(g) + ")");
        if (!g.is_non_overlapping_and_dense()) return fail("clip_grad_norm_: a gradient is not dense");
        if (!g.numel()) continue;
        gs.push_back((long long)g.data_ptr());
        ns.push_back((long long)g.numel());
    }
    std::vector<std::pair<long long, long long>> sorted;                       // {begin, end} in bytes
    for (size_t i = 0; i < gs.size(); ++i) sorted.emplace_back(gs[i], gs[i] + 4 * ns[i]);
    std::sort(sorted.begin(), sorted.end());
    for (size_t i = 1; i < sorted.size(); ++i)
        if (sorted[i].first < sorted[i - 1].second) {
            PyErr_SetString(PyExc_ValueError, sorted[i] == sorted[i - 1] ? "clip_grad_norm_: a gradient is listed twice" : "clip_grad_norm_: two gradients overlap");
            return nullptr;
        }
    return Py_BuildValue("NNni", bytes_of(gs), bytes_of(ns), (Py_ssize_t)gs.size(), device);
}
