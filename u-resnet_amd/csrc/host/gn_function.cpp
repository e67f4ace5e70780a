// act(GroupNorm(x) (+ residual)) as a node of the autograd tape: ur_gn_act_fwd / ur_gn_act_bwd with their buffers.
#include "host.h"

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <climits>
#include <memory>
#include <stdexcept>

namespace {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

constexpr auto CL = at::MemoryFormat::ChannelsLast;

struct Shape {
    int dtype, n, c, groups, act;
    long long hw;
    float slope;
};

// channel pitch of a dense NHWC tensor or a channel window of one, 0 if t is neither (sizes of one leave strides without
// meaning: a dense tensor is recognised by its memory format)
int pitch(const at::Tensor& t) {
    if (t.is_contiguous(CL)) return (int)t.size(1);
    const int64_t c = t.size(1), h = t.size(2), w = t.size(3), ld = t.stride(3);
    return t.stride(1) == 1 && ld >= c && ld <= INT_MAX && t.stride(2) == w * ld && t.stride(0) == h * w * ld ? (int)ld : 0;
}

// whether two tensors with a pitch share an element; windows over different channels of one buffer do not
bool overlap(const at::Tensor& a, const at::Tensor& b) {
    const int64_t pa = pitch(a), pb = pitch(b), c = a.size(1), rows = a.size(0) * a.size(2) * a.size(3), size = (int64_t)a.element_size();
    const char *p = static_cast<const char*>(a.data_ptr()), *q = static_cast<const char*>(b.data_ptr());
    if (p + ((rows - 1) * pa + c) * size <= q || q + ((rows - 1) * pb + c) * size <= p) return false;
    if (pa != pb || (p - q) % size) return true;
    const int64_t off = (((p - q) / size) % pa + pa) % pa;
    return off < c || off > pa - c;
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const at::Tensor& t) { return static_cast<float*>(ptr(t)); }

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

struct GnBackward : public Node {
    SavedVariable x, gamma, beta, residual;
    at::Tensor stats;
    Shape s;
    bool passes_dy = false;              // a residual without activation: its gradient is dy itself

    std::string name() const override { return "GnActBackward"; }
    void release_variables() override {
        x.reset_data();
        gamma.reset_data();
        beta.reset_data();
        residual.reset_data();
        stats.reset();
    }

    int layout(at::Tensor& t, at::IntArrayRef sizes, const char* what) const {
        if (t.device() != stats.device() || t.scalar_type() != (s.dtype == UR_BF16 ? at::kBFloat16 : at::kFloat) || t.sizes() != sizes)
            throw std::runtime_error(std::string("gn_act: ") + what + " came back from its saved-tensor hook with another type, shape or device");
        if (const int ld = pitch(t)) return ld;
        t = t.contiguous(CL);
        return s.c;
    }
    at::Tensor channel_values(const at::Tensor& t) const {
        if (t.device() != stats.device() || t.scalar_type() != at::kFloat || t.numel() != s.c)
            throw std::runtime_error("gn_act: a parameter came back from its saved-tensor hook with another type, shape or device");
        return t.contiguous();
    }

    // A captured backward pass cannot hand a gradient on to the default stream, which does not take part in the capture: what
    // was recorded there eagerly and is still alive (a leaf's accumulator in another, live graph) would end the process
    void refuse_capture_into_eager_graph(c10::Device device) const {
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
        // by number: the graph's streams carry torch's device type, these HIP's, and so never compare equal
        const c10::StreamId eager = c10::hip::getDefaultHIPStream(device.index()).id();
        for (uint32_t i = 0; i < num_outputs(); ++i) {
            const auto& next = next_edge(i).function;
            if (!next || !task_should_compute_output(i)) continue;
            const auto on = next->stream();
            if (on && on->id() == eager)
                throw std::runtime_error("gn_act: the captured backward pass reaches a tensor whose graph was recorded outside the capture and "
                                         "is still alive: drop what an eager forward pass returned before capturing");
        }
    }

    variable_list apply(variable_list&& grads) override {
        variable_list out(4);
        at::Tensor dy = grads[0];
        if (!dy.defined()) return out;
        if (at::GradMode::is_enabled()) throw std::runtime_error("gn_act: no double backward (create_graph=True)");
        refuse_capture_into_eager_graph(dy.device());
        const bool want_x = task_should_compute_output(0), want_gamma = task_should_compute_output(1), want_beta = task_should_compute_output(2),
                   want_res = task_should_compute_output(3);
        if (passes_dy && want_res) out[3] = dy;
        const bool want_dres = !passes_dy && want_res;
        if (!(want_x || want_gamma || want_beta || want_dres)) return out;
        at::Tensor xs = x.unpack(), gs = gamma.unpack(), bs = beta.unpack(), rs = residual.unpack();
        if (!stats.defined()) throw std::runtime_error("gn_act: backward through the same graph a second time (retain_graph=True keeps it)");
        const c10::DeviceGuard guard(stats.device());
        // what comes back may be laid out in another way than what was saved (saved-tensor hooks)
        const int x_ld = layout(xs, dy.sizes(), "x"), res_ld = rs.defined() ? layout(rs, dy.sizes(), "the residual") : 0;
        for (at::Tensor* p : {&gs, &bs})
            if (p->defined()) *p = channel_values(*p);
        if (dy.scalar_type() != xs.scalar_type()) dy = dy.to(xs.scalar_type());
        int dy_ld = pitch(dy);
        if (!dy_ld) { dy = dy.contiguous(CL); dy_ld = s.c; }
        at::Tensor dres;
        if (want_x || want_dres) out[0] = at::empty(xs.sizes(), xs.options().memory_format(CL));
        if (want_dres) dres = at::empty(xs.sizes(), xs.options().memory_format(CL));
        if (want_gamma) out[1] = at::empty({s.c}, xs.options().dtype(at::kFloat));
        if (want_beta) out[2] = at::empty({s.c}, xs.options().dtype(at::kFloat));
        const size_t bytes = entry.gn_bwd_workspace(s.dtype, s.n, s.hw, s.c, s.groups);
        const at::Tensor ws = at::empty({(int64_t)bytes}, xs.options().dtype(at::kByte));
        check(entry.gn_act_bwd(ptr(dy), dy_ld, ptr(xs), x_ld, ptr(rs), res_ld, fptr(gs), fptr(bs), static_cast<double*>(ptr(stats)),
                               ptr(out[0]), ptr(dres), fptr(out[1]), fptr(out[2]), s.dtype, s.n, s.hw, s.c, s.groups, s.act, s.slope, ptr(ws),
                               bytes, stream_of(xs)),
              "ur_gn_act_bwd");
        if (want_dres) out[3] = dres;
        if (!want_x) out[0] = at::Tensor();
        return out;
    }
};

at::Tensor forward(const at::Tensor& x, const at::Tensor& gamma, const at::Tensor& beta, const at::Tensor& residual, at::Tensor z, int groups,
                   double eps, int act, double slope) {
    Shape s;
    s.dtype = x.scalar_type() == at::kBFloat16 ? UR_BF16 : UR_F32;
    s.n = (int)x.size(0);
    s.c = (int)x.size(1);
    s.groups = groups;
    s.act = act;
    s.hw = x.size(2) * x.size(3);
    s.slope = (float)slope;
    const c10::DeviceGuard guard(x.device());
    at::Tensor stats;
    {
        const at::NoGradGuard no_grad;
        if (!z.defined()) z = at::empty(x.sizes(), x.options().memory_format(CL));
        else if (!z.is_inference()) z.unsafeGetTensorImpl()->bump_version();       // written in place
        stats = at::empty({s.n, groups, 2}, x.options().dtype(at::kDouble));
        const size_t bytes = entry.gn_fwd_workspace(s.dtype, s.n, s.hw, s.c, groups);
        const at::Tensor ws = at::empty({(int64_t)(bytes ? bytes : 16)}, x.options().dtype(at::kByte));
        check(entry.gn_act_fwd(ptr(x), pitch(x), ptr(residual), residual.defined() ? pitch(residual) : 0, fptr(gamma), fptr(beta), ptr(z), pitch(z), static_cast<double*>(ptr(stats)),
                               s.dtype, s.n, s.hw, s.c, groups, (float)eps, act, s.slope, ptr(ws), bytes, stream_of(x)),
              "ur_gn_act_fwd");
    }
    if (at::GradMode::is_enabled() && torch::autograd::compute_requires_grad(x, gamma, beta, residual)) {
        auto node = std::shared_ptr<GnBackward>(new GnBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, gamma, beta, residual));
        node->x = SavedVariable(x, false);
        node->gamma = SavedVariable(gamma, false);
        node->beta = SavedVariable(beta, false);
        // without an activation nothing depends on the residual's values
        node->passes_dy = residual.defined() && act == UR_ACT_NONE;
        node->residual = SavedVariable(act == UR_ACT_NONE ? at::Tensor() : residual, false);
        node->stats = stats;
        node->s = s;
        torch::autograd::set_history(z, node);
    }
    return z;
}

bool optional_tensor(PyObject* o, at::Tensor& out) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "gn_act: a tensor or None is expected");
        return false;
    }
    out = THPVariable_Unpack(o);
    return true;
}

std::string shape_of(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

}  // namespace

// gn_act(x, weight, bias, residual, out, groups, channels, eps, act, slope): everything the kernels rely on is checked here
PyObject* gn_act(PyObject*, PyObject* args) {
    PyObject* o[5];
    int groups, channels, act;
    double eps, slope;
    if (!PyArg_ParseTuple(args, "OOOOOiidid", &o[0], &o[1], &o[2], &o[3], &o[4], &groups, &channels, &eps, &act, &slope)) return nullptr;
    at::Tensor x, gamma, beta, residual, out;
    at::Tensor* t[5] = {&x, &gamma, &beta, &residual, &out};
    for (int i = 0; i < 5; ++i)
        if (!optional_tensor(o[i], *t[i])) return nullptr;
    const auto refuse = [](PyObject* type, const std::string& text) -> PyObject* {
        PyErr_SetString(type, ("gn_act: " + text).c_str());
        return nullptr;
    };
    // neither sees what the kernels write through addresses: a tangent would be lost, a recorded call would return fresh memory
    for (const at::Tensor* p : t)
        if (p->defined() && p->_fw_grad(0).defined()) return refuse(PyExc_NotImplementedError, "no forward-mode gradient (an input carries a tangent)");
    if (torch::jit::tracer::isTracing()) return refuse(PyExc_NotImplementedError, "cannot be recorded by torch.jit.trace");
    if (!x.defined() || x.dim() != 4) return refuse(PyExc_ValueError, "expected a 4-D NCHW tensor" + (x.defined() ? ", got shape " + shape_of(x) : ""));
    if (act < UR_ACT_NONE || act > UR_ACT_SILU) return refuse(PyExc_ValueError, "unknown activation code " + std::to_string(act));
    if (!x.is_cuda()) return fail("u-resnet_amd operators run on the GPU only (got a " + x.device().str() + " tensor); there is no CPU fallback");
    if (x.scalar_type() != at::kFloat && x.scalar_type() != at::kBFloat16)
        return refuse(PyExc_TypeError, std::string("unsupported activation dtype ") + c10::toString(x.scalar_type()) + " (use torch.float32 or torch.bfloat16)");
    if (x.size(1) != channels) return refuse(PyExc_RuntimeError, std::to_string(x.size(1)) + " channels, the GroupNorm has " + std::to_string(channels));
    if (x.numel() == 0) return fail("gn_act: non-positive size in shape " + shape_of(x));
    for (const at::Tensor* p : {&gamma, &beta})
        if (p->defined() && (p->scalar_type() != at::kFloat || p->device() != x.device() || !p->is_contiguous() || p->numel() != channels))
            return fail(std::string("gn_act: the GroupNorm's ") + (p == &gamma ? "weight" : "bias") + " must be a contiguous fp32 tensor on " + x.device().str());
    if (residual.defined() && (residual.sizes() != x.sizes() || residual.device() != x.device() || residual.scalar_type() != x.scalar_type() || !pitch(residual)))
        return refuse(PyExc_RuntimeError, "the residual is " + shape_of(residual) + " on " + residual.device().str() + ", expected " + shape_of(x) +
                                              " on " + x.device().str() + ", of the same type and channels last");
    if (out.defined() && (out.dim() != 4 || out.sizes() != x.sizes() || out.device() != x.device() || out.scalar_type() != x.scalar_type() || !pitch(out)))
        return refuse(PyExc_RuntimeError, "`out` must be a channel window with x's shape, dtype and device");
    if (!pitch(x)) return refuse(PyExc_RuntimeError, "x must be channels last or a channel window");
    if (x.size(0) > INT_MAX) return refuse(PyExc_RuntimeError, std::to_string(x.size(0)) + " images");
    if (out.defined() && (overlap(out, x) || (residual.defined() && overlap(out, residual))))
        return refuse(PyExc_RuntimeError, "`out` shares elements with an input");
    if (out.defined() && out.requires_grad() && at::GradMode::is_enabled())
        return refuse(PyExc_RuntimeError, "`out` belongs to a graph or is a leaf that requires a gradient");
    at::Tensor z;
    {
        const pybind11::gil_scoped_release no_gil;
        z = forward(x, gamma, beta, residual, out, groups, eps, act, slope);
    }
    return THPVariable_Wrap(z);
}
