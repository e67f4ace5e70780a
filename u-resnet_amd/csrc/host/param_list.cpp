// The optimiser step and gradient clipping over lists of tensors: reads the lists, checks what the kernels rely on and queues
// the launches.  One call per step instead of some ten interpreter calls per parameter and more per launch.
#include "host.h"

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

namespace {

std::string told(const at::Tensor& t) {
    return std::string(c10::toString(t.layout())) + " " + c10::toString(t.scalar_type()) + " on " + t.device().str();
}

bool plain_gpu_f32(const at::Tensor& g, c10::Device device) {
    return g.layout() == c10::kStrided && g.scalar_type() == at::kFloat && g.device() == device && device.is_cuda();
}

bool get_tensor(PyObject* o, at::Tensor& out) {
    if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "a list of tensors is expected");
        return false;
    }
    out = THPVariable_Unpack(o);
    return true;
}

// Tensors [at, at + count) of a list: what one table holds
struct Span {
    int at, count;
    long long chunks;
    char* table;
};

// the spans of a list in which a gradient has elements
std::vector<Span> spans_of(const std::vector<long long>& grads, const std::vector<long long>& sizes) {
    std::vector<Span> out;
    const int rows = entry.param_table_max_rows(), n = (int)grads.size();
    for (int at = 0; at < n; at += rows) {
        const Span s = {at, std::min(rows, n - at), 0, nullptr};
        bool any = false;
        for (int i = at; i < at + s.count; ++i) any = any || (grads[i] && sizes[i]);
        if (any) out.push_back(s);
    }
    return out;
}

size_t table_bytes(int count) { return (entry.param_table_bytes(count) + 15) / 16 * 16; }

// device memory for the tables of all spans and, behind them, the partial sums of the norm
struct Memory {
    at::Tensor buf;
    double* parts;
    Memory(const std::vector<Span*>& spans, bool norm, c10::Device device) {
        size_t bytes = 0;
        for (const Span* s : spans) bytes += table_bytes(s->count);
        const size_t sums = norm ? spans.size() * entry.grad_sqnorm_max_parts() * sizeof(double) : 0;
        buf = at::empty({(int64_t)(bytes + sums)}, at::TensorOptions().dtype(at::kByte).device(device));
        char* p = static_cast<char*>(buf.data_ptr());
        parts = reinterpret_cast<double*>(p + bytes);
        for (Span* s : spans) { s->table = p; p += table_bytes(s->count); }
    }
};

// Bytes [begin, end) of each tensor of four-byte elements at `addresses`, in order; empty and absent ones left out.
std::vector<std::pair<long long, long long>> ranges(const std::vector<long long>& addresses, const std::vector<long long>& sizes) {
    std::vector<std::pair<long long, long long>> out;
    out.reserve(addresses.size());
    for (size_t i = 0; i < addresses.size(); ++i)
        if (addresses[i] && sizes[i]) out.emplace_back(addresses[i], addresses[i] + 4 * sizes[i]);
    std::sort(out.begin(), out.end());
    return out;
}

struct Group {
    std::vector<long long> params, grads, sizes;
    std::vector<Span> spans;
    unsigned long long blocks, steps, m, v, ms, vs;
    int bits;
    double lr, beta1, beta2, eps, wd;
};

// The kernels write through addresses: without a count autograd would hand a graph that saved these tensors their new values.
void count_writes(const std::vector<at::Tensor>& written) {
    for (const at::Tensor& t : written)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct Written {                                               // counted when it goes, also by an exception
    const std::vector<at::Tensor>& tensors;
    explicit Written(const std::vector<at::Tensor>& t) : tensors(t) {}
    ~Written() { count_writes(tensors); }
};

at::Tensor scalar_on(c10::Device device) { return at::empty({}, at::TensorOptions().dtype(at::kFloat).device(device)); }

}  // namespace

// adamw_step(groups, max_norm or None, grad_scale) -> (whether anything was launched, norm or None).  A group: (parameters,
// element counts that the state was made for (int64 array), addresses of the first blocks and step counts, state_bits, addresses
// of the moments and their scales, lr, beta1, beta2, eps, weight decay).  Everything is checked before the first launch.
PyObject* adamw_step(PyObject*, PyObject* args) {
    PyObject *list, *limit;
    double grad_scale;
    if (!PyArg_ParseTuple(args, "O!Od", &PyList_Type, &list, &limit, &grad_scale)) return nullptr;
    const bool clip = limit != Py_None;
    const double max_norm = clip ? PyFloat_AsDouble(limit) : 0.0;
    if (PyErr_Occurred()) return nullptr;
    std::vector<Group> groups((size_t)PyList_GET_SIZE(list));
    std::vector<at::Tensor> held, written;                     // contiguous copies of gradients, until the launches are queued
    c10::Device device(c10::kCPU);
    bool live = false;
    for (size_t k = 0; k < groups.size(); ++k) {
        Group& q = groups[k];
        PyObject *params, *sizes;
        if (!PyArg_ParseTuple(PyList_GET_ITEM(list, (Py_ssize_t)k), "O!SKKiKKKKddddd", &PyList_Type, &params, &sizes, &q.blocks, &q.steps, &q.bits,
                              &q.m, &q.v, &q.ms, &q.vs, &q.lr, &q.beta1, &q.beta2, &q.eps, &q.wd))
            return nullptr;
        if (q.bits == 8 && q.beta1 > 17.0 / 18.0) return fail("AdamW: 8-bit moments need betas[0] <= 17/18 (got " + std::to_string(q.beta1) + ")");
        const Py_ssize_t n = PyList_GET_SIZE(params);
        if (PyBytes_GET_SIZE(sizes) != (Py_ssize_t)(n * sizeof(long long))) return fail("AdamW: lists of different lengths");
        const long long* want = reinterpret_cast<const long long*>(PyBytes_AS_STRING(sizes));
        q.sizes.assign(want, want + n);
        q.params.assign(n, 0);
        q.grads.assign(n, 0);
        for (Py_ssize_t i = 0; i < n; ++i) {
            at::Tensor p;
            if (!get_tensor(PyList_GET_ITEM(params, i), p)) return nullptr;
            at::Tensor g = p.grad();
            if (!g.defined()) continue;
            if (!p.device().is_cuda()) return fail("AdamW: parameters must be on a GPU (got " + p.device().str() + ")");
            if (!plain_gpu_f32(g, p.device())) return fail("AdamW: gradients must be dense fp32 tensors on the parameter's GPU (got " + told(g) + ")");
            if (p.layout() != c10::kStrided || p.scalar_type() != at::kFloat || !p.is_contiguous() || p.numel() != want[i] || g.numel() != want[i])
                return fail("AdamW: a parameter changed its size, layout or type");
            if (live && p.device() != device) return fail("AdamW: all parameters must be on one GPU");
            device = p.device();
            live = true;
            if (!g.is_contiguous()) {
                const at::NoGradGuard no_grad;
                const c10::DeviceGuard guard(device);
                g = g.contiguous();
                held.push_back(g);
            }
            q.params[i] = (long long)p.data_ptr();
            q.grads[i] = (long long)g.data_ptr();
            written.push_back(std::move(p));
        }
        const auto places = ranges(q.params, q.sizes);         // one launch writes them all: shared memory would be a race
        for (size_t i = 1; i < places.size(); ++i)
            if (places[i].first < places[i - 1].second) return fail("AdamW: two parameters of a group share memory");
        q.spans = spans_of(q.grads, q.sizes);
    }
    std::vector<Span*> spans;
    for (Group& q : groups)
        for (Span& s : q.spans) spans.push_back(&s);
    if (spans.empty()) return Py_BuildValue("OO", Py_False, Py_None);
    at::Tensor norm;
    {
        const pybind11::gil_scoped_release no_gil;
        const c10::DeviceGuard guard(device);
        void* stream = c10::hip::getCurrentHIPStream(device.index()).stream();
        const Memory mem(spans, clip, device);
        if (clip) norm = scalar_on(device);
        const Written count(written);
        for (Group& q : groups)
            for (Span& s : q.spans)
                check(entry.param_table(&q.params[s.at], &q.grads[s.at], &q.sizes[s.at], reinterpret_cast<const long long*>(q.blocks) + s.at, s.count,
                                        s.table, table_bytes(s.count), reinterpret_cast<int*>(q.steps) + s.at, q.lr, q.beta1, q.beta2, &s.chunks,
                                        stream),
                      "ur_param_table");
        int nparts = 0;
        if (clip)
            for (const Span* s : spans) {
                int got = 0;
                check(entry.grad_sqnorm(s->table, s->count, s->chunks, mem.parts + nparts, &got, stream), "ur_grad_sqnorm");
                nparts += got;
            }
        for (const Group& q : groups)
            for (const Span& s : q.spans)
                check(entry.adamw_multi(s.table, s.count, s.chunks, q.bits, reinterpret_cast<void*>(q.m), reinterpret_cast<void*>(q.v),
                                        reinterpret_cast<float*>(q.ms), reinterpret_cast<float*>(q.vs), q.lr, q.beta1, q.beta2, q.eps, q.wd,
                                        clip ? mem.parts : nullptr, nparts, (float)max_norm, (float)grad_scale,
                                        clip ? norm.data_ptr<float>() : nullptr, stream),
                      "ur_adamw_multi");
    }
    if (!clip) return Py_BuildValue("OO", Py_True, Py_None);
    return Py_BuildValue("ON", Py_True, THPVariable_Wrap(norm));
}

// holds(state, entries, contents): whether the values of the dict `state` are the dicts `entries` and their values, one after the
// other, the objects of the list `contents`
PyObject* holds(PyObject*, PyObject* args) {
    PyObject *state, *entries, *contents;
    if (!PyArg_ParseTuple(args, "O!O!O!", &PyDict_Type, &state, &PyList_Type, &entries, &PyList_Type, &contents)) return nullptr;
    if (PyDict_Size(state) != PyList_GET_SIZE(entries)) Py_RETURN_FALSE;
    Py_ssize_t at = 0, i = 0, k = 0;
    for (PyObject *key, *entry; PyDict_Next(state, &at, &key, &entry); ++i) {
        if (entry != PyList_GET_ITEM(entries, i) || !PyDict_Check(entry)) Py_RETURN_FALSE;
        Py_ssize_t in = 0;
        for (PyObject *name, *value; PyDict_Next(entry, &in, &name, &value); ++k)
            if (k >= PyList_GET_SIZE(contents) || value != PyList_GET_ITEM(contents, k)) Py_RETURN_FALSE;
    }
    return PyBool_FromLong(k == PyList_GET_SIZE(contents));
}

// clip_grads(parameters, max_norm, whether to raise on a norm that is not finite) -> norm, None without gradients
PyObject* clip_grads(PyObject*, PyObject* args) {
    PyObject* params;
    double max_norm;
    int raise;
    if (!PyArg_ParseTuple(args, "O!dp", &PyList_Type, &params, &max_norm, &raise)) return nullptr;
    std::vector<long long> gs, ns;
    std::vector<at::Tensor> written;
    bool live = false;
    c10::Device device(c10::kCPU);
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); ++i) {
        at::Tensor p;
        if (!get_tensor(PyList_GET_ITEM(params, i), p)) return nullptr;
        const at::Tensor g = p.grad();
        if (!g.defined()) continue;
        if (!live) device = g.device();
        live = true;
        if (!plain_gpu_f32(g, device)) return fail("clip_grad_norm_: gradients must be dense fp32 tensors on one GPU (got " + told(g) + ")");
        if (!g.is_non_overlapping_and_dense()) return fail("clip_grad_norm_: a gradient is not dense");
        if (!g.numel()) continue;
        gs.push_back((long long)g.data_ptr());
        ns.push_back((long long)g.numel());
        written.push_back(g);
    }
    if (!live) Py_RETURN_NONE;
    const auto sorted = ranges(gs, ns);
    for (size_t i = 1; i < sorted.size(); ++i)
        if (sorted[i].first < sorted[i - 1].second) {
            PyErr_SetString(PyExc_ValueError, sorted[i] == sorted[i - 1] ? "clip_grad_norm_: a gradient is listed twice" : "clip_grad_norm_: two gradients overlap");
            return nullptr;
        }
    std::vector<Span> list = spans_of(gs, ns);
    std::vector<Span*> spans;
    for (Span& s : list) spans.push_back(&s);
    at::Tensor norm;
    std::string error;
    {
        const pybind11::gil_scoped_release no_gil;
        const c10::DeviceGuard guard(device);
        norm = scalar_on(device);
        if (spans.empty()) norm.zero_();
        else {
            void* stream = c10::hip::getCurrentHIPStream(device.index()).stream();
            const Memory mem(spans, true, device);
            int nparts = 0;
            for (Span* s : spans) {
                int got = 0;
                check(entry.param_table(nullptr, &gs[s->at], &ns[s->at], nullptr, s->count, s->table, table_bytes(s->count), nullptr, 0.0, 0.0, 0.0,
                                        &s->chunks, stream),
                      "ur_param_table");
                check(entry.grad_sqnorm(s->table, s->count, s->chunks, mem.parts + nparts, &got, stream), "ur_grad_sqnorm");
                nparts += got;
            }
            if (raise) {
                const int64_t at = (reinterpret_cast<char*>(mem.parts) - static_cast<char*>(mem.buf.data_ptr())) / 8;
                const at::NoGradGuard no_grad;
                const double total = mem.buf.narrow(0, 8 * at, 8 * (int64_t)nparts).view(at::kDouble).sum().item<double>();
                if (!std::isfinite((float)std::sqrt(total))) error = "clip_grad_norm_: the total norm of the gradients is not finite";
            }
            if (error.empty())
                for (const Span* s : spans)
                    check(entry.grad_clip(s->table, s->count, s->chunks, mem.parts, nparts, (float)max_norm, norm.data_ptr<float>(), stream), "ur_grad_clip");
        }
    }
    if (!error.empty()) return fail(error);
    count_writes(written);
    return THPVariable_Wrap(norm);
}
