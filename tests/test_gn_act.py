"""GroupNorm + activation (ops.gn_act, nn.GroupNorm) against the formulas in 64 bits.

Tolerances.  The kernels keep statistics in fp64 and compute each element in fp32: pre = d * A + B (+ r) carries at most five
roundings of 2^-24 relative to |d A| + |B| + |r|, an activation at most another dozen (erf, exp, division), its slope is at
most 1.13.  TERMS = 20 of them bound an element of y, with the storage rounding (half a step: bf16 2^-8, fp32 2^-24) on top.
dx is a sum of three terms, each a product of such values; the group means P1, P2 come from fp32 sums of at most R pixels per
thread, so they are off by (R + 10) 2^-24 times the mean of |terms|.  The parameter gradients are the same sums themselves."""
import math

import pytest
import torch

import uresnet_amd
from uresnet_amd import _lib, nn as hnn, ops

DEV = "cuda:0"
E24 = 2.0 ** -24
TERMS = 20
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
ACTS = {"none": 0, "relu": 1, "relu6": 2, "leakyrelu": 3, "gelu": 4, "hswish": 5, "silu": 6}
SLOPE = 0.2
# n, c, h, w, groups
SHAPES = [
    (1, 1, 1, 1, 1),           # a group of one value
    (2, 8, 1, 1, 8),           # ... in every group
    (2, 3, 5, 7, 3),           # no vector accesses
    (1, 6, 9, 4, 2),
    (2, 64, 16, 16, 32),       # two channels to a group
    (3, 80, 7, 13, 20),        # ten vectors: threads of a workgroup stay idle
    (2, 24, 5, 5, 3),          # a group per vector
    (1, 48, 11, 3, 4),         # groups that end inside a vector of eight
    (1, 2056, 3, 2, 8),        # more channel vectors than threads, groups across the slabs
    (1, 300, 2, 3, 300),       # instance norm, element-wise in bf16 with two slabs
    (2, 512, 4, 5, 1),         # one group
    (70, 16, 2, 2, 4),         # more images than pixels
    (1, 32, 1, 700, 4),        # one long row
    (2, 40, 37, 53, 5),
]


def act_of(p, act):
    F = torch.nn.functional
    return {"none": lambda t: t, "relu": F.relu, "relu6": F.relu6, "leakyrelu": lambda t: F.leaky_relu(t, SLOPE), "gelu": F.gelu,
            "hswish": F.hardswish, "silu": F.silu}[act](p)


def make(shape, dtype, seed, mean=1.0, residual=False, affine=True):
    n, c, h, w, groups = shape
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, c, h, w, generator=g) * (0.5 + torch.rand(c, 1, 1, generator=g)) + mean * torch.randn(c, 1, 1, generator=g)).to(dtype)
    dy = (torch.randn(n, c, h, w, generator=g) + 0.3 * x.float()).to(dtype)
    r = torch.randn(n, c, h, w, generator=g).to(dtype) if residual else None
    gn = hnn.GroupNorm(groups, c, eps=1e-5, affine=affine)
    if affine:
        with torch.no_grad():
            gn.weight.copy_(1 + 0.3 * torch.randn(c, generator=g))
            gn.bias.copy_(0.3 * torch.randn(c, generator=g))
    return x, dy, r, gn


def reference(x, dy, r, gn, act):
    """y, gradients and, for the tolerances, the magnitudes of the terms: everything in 64 bits on the CPU."""
    n, c, h, w = x.shape
    G = gn.num_groups
    xd = x.double()
    w4 = (gn.weight.detach().double() if gn.affine else torch.ones(c).double()).view(1, c, 1, 1)
    b4 = (gn.bias.detach().double() if gn.affine else torch.zeros(c).double()).view(1, c, 1, 1)
    grouped = xd.reshape(n, G, -1)
    mean = grouped.mean(2)
    rstd = (grouped.var(2, unbiased=False) + gn.eps).rsqrt()
    m4, s4 = (t.repeat_interleave(c // G, 1).view(n, c, 1, 1) for t in (mean, rstd))
    xhat = (xd - m4) * s4
    pre = (xhat * w4 + b4 + (0 if r is None else r.double())).requires_grad_()
    y = act_of(pre, act)
    g = torch.autograd.grad(y, pre, dy.double())[0]
    pre, y = pre.detach(), y.detach()

    def over_group(t):
        return t.reshape(n, G, -1).mean(2).repeat_interleave(c // G, 1).view(n, c, 1, 1)
    dx = s4 * (w4 * g - over_group(w4 * g) - xhat * over_group(w4 * g * xhat))
    size_pre = (xhat * w4).abs() + b4.abs() + (0 if r is None else r.double().abs())
    size_dx = s4 * ((w4 * g).abs() + over_group((w4 * g).abs()) + xhat.abs() * over_group((w4 * g * xhat).abs()))
    return {"y": y, "dx": dx, "dres": g, "dgamma": (g * xhat).sum((0, 2, 3)), "dbeta": g.sum((0, 2, 3)), "size_pre": size_pre,
            "size_dx": size_dx, "size_g": dy.double().abs() * 1.2, "abs_dgamma": (g * xhat).abs().sum((0, 2, 3)),
            "abs_dbeta": g.abs().sum((0, 2, 3))}


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= tol).all(), "%s: off by %.3g where %.3g is allowed" % (what, (off - tol).max().item() + tol.flatten()[(off - tol).argmax()].item(), tol.flatten()[(off - tol).argmax()].item())


def check(x, dy, r, gn, act, got):
    ref, half = reference(x, dy, r, gn, act), HALF[x.dtype]
    rows = 4 * (x.shape[2] * x.shape[3])                        # more pixels than any thread sums
    within(got["y"], ref["y"], half * ref["y"].abs() + TERMS * E24 * (1.2 * ref["size_pre"] + 1e-3), "y")
    within(got["dx"], ref["dx"], half * ref["dx"].abs() + (rows + TERMS) * E24 * 1.2 * ref["size_dx"] + 1e-12, "dx")
    if gn.affine:
        for k in ("dgamma", "dbeta"):
            within(got[k], ref[k], (rows + TERMS) * E24 * ref["abs_" + k] + 1e-12, k)
    if r is not None:
        within(got["dres"], ref["dres"], half * ref["dres"].abs() + TERMS * E24 * (ref["size_g"] + 1e-3), "dres")


def run(x, dy, r, gn, act, layout=lambda t: t.to(DEV).contiguous(memory_format=torch.channels_last)):
    gn = gn.to(DEV)
    xd, rd = layout(x).detach().requires_grad_(), None if r is None else layout(r).detach().requires_grad_()
    y = ops.gn_act(xd, gn, residual=rd, act=ACTS[act], slope=SLOPE)
    wrt = [xd] + ([gn.weight, gn.bias] if gn.affine else []) + ([] if r is None else [rd])
    grads = list(torch.autograd.grad(y, wrt, layout(dy)))
    out = {"y": y, "dx": grads.pop(0)}
    if gn.affine:
        out["dgamma"], out["dbeta"] = grads.pop(0), grads.pop(0)
    if r is not None:
        out["dres"] = grads.pop(0)
    torch.cuda.synchronize()
    gn.cpu()
    return out


# ------------------------------------------------------------------------------ refusals (CPU)
def test_refusals_without_a_gpu():
    gn = hnn.GroupNorm(4, 8)
    with pytest.raises(_lib.UResNetHipError, match="no CPU fallback"):
        gn(torch.randn(1, 8, 4, 4))
    with pytest.raises(ValueError, match="4-D"):
        ops.gn_act(torch.randn(8, 8), gn)
    with pytest.raises(ValueError, match="activation"):
        ops.gn_act(torch.randn(1, 8, 4, 4), gn, act=9)
    with pytest.raises(ValueError):
        hnn.GroupNorm(3, 8)
    with pytest.raises(ValueError, match="positive"):
        hnn.to_group_norm(torch.nn.BatchNorm2d(8), 0)


@pytest.mark.parametrize("sizes, message", [((1, 0, 8, 4), "non-positive"), ((0, 16, 8, 4), "non-positive"), ((1, 16, 8, 0), "non-positive"),
                                            ((1, 16, 9, 4), "not divisible"), ((70000, 16, 8, 4), "limits")])
def test_entry_points_refuse_bad_sizes_before_any_launch(sizes, message):
    n, hw, c, groups = sizes
    assert _lib.query("ur_gn_fwd_workspace", _lib.UR_F32, n, hw, c, groups) == 0
    assert _lib.query("ur_gn_bwd_workspace", _lib.UR_F32, n, hw, c, groups) == 0
    with pytest.raises(_lib.UResNetHipError, match=message):
        _lib.call("ur_gn_act_fwd", 16, 0, None, 0, None, None, 16, 0, 16, _lib.UR_F32, n, hw, c, groups, 1e-5, 0, 0.0, 16, 1 << 30, None)
    with pytest.raises(_lib.UResNetHipError, match=message):
        _lib.call("ur_gn_act_bwd", 16, 0, 16, 0, None, 0, None, None, 16, 16, None, None, None, _lib.UR_F32, n, hw, c, groups, 0, 0.0, 16,
                  1 << 30, None)


def test_entry_points_refuse_bad_pointers_pitches_and_workspaces():
    def fwd(x=16, ld=0, y=16, dtype=_lib.UR_F32, act=0, ws=16, size=1 << 30):
        _lib.call("ur_gn_act_fwd", x, ld, None, 0, None, None, y, 0, 16, dtype, 1, 16, 8, 4, 1e-5, act, 0.0, ws, size, None)

    def bwd(res=None, dx=16, dres=None, size=1 << 30):
        _lib.call("ur_gn_act_bwd", 16, 0, 16, 0, res, 0, None, None, 16, dx, dres, None, None, _lib.UR_F32, 1, 16, 8, 4, 0, 0.0, 16, size, None)
    for f, kw, message in ((fwd, dict(x=None), "null"), (fwd, dict(y=None), "null"), (fwd, dict(ws=None), "null"), (fwd, dict(ld=7), "pitch"),
                           (fwd, dict(dtype=5), "dtype"), (fwd, dict(act=7), "activation"), (fwd, dict(size=8), "workspace"),
                           (bwd, dict(dres=16), "without a residual"), (bwd, dict(res=16, dx=None, dres=16), "without dx"),
                           (bwd, dict(size=8), "workspace")):
        with pytest.raises(_lib.UResNetHipError, match=message):
            f(**kw)


def test_to_group_norm_replaces_every_batch_norm_and_keeps_the_parameters():
    from uresnet_amd.modules.U_ResNet import UResNetNewEUCB
    m = UResNetNewEUCB(19, 3, 8).eval()
    names = [k for k, v in m.named_modules() if isinstance(v, torch.nn.BatchNorm2d)]
    weights = {k: m.get_submodule(k).weight for k in names}
    assert hnn.to_group_norm(m, 32) is m
    assert not any(isinstance(v, torch.nn.BatchNorm2d) for v in m.modules())
    for k in names:
        gn = m.get_submodule(k)
        assert isinstance(gn, hnn.GroupNorm) and gn.weight is weights[k] and not gn.training
        assert gn.num_channels % gn.num_groups == 0 and gn.num_groups <= 32
    assert m.out_conv[0].num_groups == 24                      # 24 channels (8 + 16): the largest divisor up to 32
    assert isinstance(hnn.to_group_norm(torch.nn.BatchNorm2d(6, affine=False), 4), hnn.GroupNorm)


def test_to_group_norm_keeps_a_shared_layer_shared():
    bn = torch.nn.BatchNorm2d(8)
    inner = torch.nn.Sequential(bn, torch.nn.ReLU(), bn)
    m = hnn.to_group_norm(torch.nn.Sequential(inner, bn, inner), 4)
    assert isinstance(m[1], hnn.GroupNorm) and m[0][0] is m[1] and m[0][2] is m[1] and m[2] is m[0]


def test_entry_points_refuse_more_channels_than_their_sums_are_laid_out_for():
    for query in ("ur_gn_fwd_workspace", "ur_gn_bwd_workspace"):
        assert _lib.query(query, _lib.UR_BF16, 1, 4, 16384, 32) > 0 and _lib.query(query, _lib.UR_BF16, 1, 4, 16392, 8) == 0


# ------------------------------------------------------------------------------ values (GPU)
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, dtype):
    x, dy, _, gn = make(shape, dtype, 1)
    check(x, dy, None, gn, "relu", run(x, dy, None, gn, "relu"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("act", list(ACTS))
def test_activations_and_residual(act, residual, dtype):
    for shape in ((2, 32, 9, 11, 8), (2, 5, 6, 7, 5)):
        x, dy, r, gn = make(shape, dtype, 2, residual=residual)
        check(x, dy, r, gn, act, run(x, dy, r, gn, act))


@pytest.mark.gpu
def test_without_weight_and_bias():
    x, dy, _, gn = make((2, 16, 5, 9, 4), torch.float32, 3, affine=False)
    check(x, dy, None, gn, "silu", run(x, dy, None, gn, "silu"))


@pytest.mark.gpu
def test_a_mean_far_from_zero_keeps_the_variance():
    """Mean 200 times the spread: fp32 sums of squares would lose 4e4 * 2^-24 of the variance; x - mean_hi is exact here."""
    g = torch.Generator().manual_seed(4)
    x = 100 + 0.5 * torch.randn(2, 16, 20, 20, generator=g)
    dy = torch.randn(x.shape, generator=g)
    gn = hnn.GroupNorm(4, 16)
    check(x, dy, None, gn, "relu", run(x, dy, None, gn, "relu"))


@pytest.mark.gpu
@pytest.mark.parametrize("act, at", [("relu", 0.0), ("leakyrelu", 0.0), ("relu6", 6.0), ("hswish", -3.0), ("hswish", 3.0)])
def test_elements_exactly_on_a_kink(act, at):
    """Inputs symmetric around zero (mean exactly 0) with many zeros, bias at the kink: pre is exactly `at` for those zeros."""
    g = torch.Generator().manual_seed(5)
    half = torch.randn(1, 8, 4, 32, generator=g)
    x = torch.cat([half, -half, torch.zeros(1, 8, 2, 32)], 2).to(torch.bfloat16)
    dy = torch.randn(x.shape, generator=g).to(torch.bfloat16)
    gn = hnn.GroupNorm(2, 8)
    with torch.no_grad():
        gn.bias.fill_(at)
    check(x, dy, None, gn, act, run(x, dy, None, gn, act))


@pytest.mark.gpu
def test_bf16_inputs_near_a_kink_are_all_on_its_right_side():
    """Biases chosen so that one bf16 value maps to within 1e-8 of the kink, a distance that fp32 cannot resolve there."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(1, 8, 64, 64, generator=g).to(torch.bfloat16)
    dy = torch.ones_like(x)
    gn = hnn.GroupNorm(1, 8)
    xd = x.double()
    mean, rstd = xd.mean(), (xd.var(unbiased=False) + gn.eps).rsqrt()
    with torch.no_grad():
        v = x[0, :, 0, 0].double()
        gn.bias.copy_(-(v - mean) * rstd)                       # rounded to fp32: the value's pre is that rounding
    check(x, dy, None, gn, "relu", run(x, dy, None, gn, "relu"))


@pytest.mark.gpu
@pytest.mark.parametrize("c0, wide", [(8, 24), (3, 19)])
def test_channel_windows_and_other_layouts(c0, wide):
    """x, the residual and dy as channel windows of wider tensors (aligned and not), NCHW tensors, and `out` windows."""
    x, dy, r, gn = make((2, 8, 6, 5, 4), torch.bfloat16, 7, residual=True)

    def window(t):
        buf = torch.full((2, wide, 6, 5), 7.0, dtype=t.dtype, device=DEV).contiguous(memory_format=torch.channels_last)
        win = ops.alias_window(buf, c0, 8)
        win.copy_(t.to(DEV))
        return win
    want = run(x, dy, r, gn, "gelu")
    check(x, dy, r, gn, "gelu", want)
    for layout in (window, lambda t: t.to(DEV).contiguous()):
        got = run(x, dy, r, gn, "gelu", layout)
        for k in want:                                          # the same values; sums may be grouped in another way
            assert torch.allclose(got[k].float(), want[k].float(), rtol=2.0 ** -7, atol=1e-5), k
        check(x, dy, r, gn, "gelu", got)
    gn = gn.to(DEV)
    buf = torch.full((2, wide, 6, 5), 7.0, dtype=torch.bfloat16, device=DEV).contiguous(memory_format=torch.channels_last)
    out = ops.alias_window(buf, c0, 8)
    xd = x.to(DEV).contiguous(memory_format=torch.channels_last)
    z = ops.gn_act(xd, gn, act=ACTS["relu"], out=out)
    assert z.data_ptr() == out.data_ptr() and torch.equal(out, ops.gn_act(xd, gn, act=ACTS["relu"]))
    rest = torch.ones(wide, dtype=torch.bool)
    rest[c0:c0 + 8] = False
    assert (buf[:, rest] == 7).all()                            # what lies beside the window stays


@pytest.mark.gpu
def test_an_output_window_shares_nothing_with_the_inputs():
    gn = hnn.GroupNorm(4, 8).to(DEV)
    buf = torch.randn(2, 24, 6, 5, device=DEV).contiguous(memory_format=torch.channels_last)
    x, y = ops.alias_window(buf, 0, 8), ops.alias_window(buf, 8, 8)
    want = ops.gn_act(x.clone(memory_format=torch.channels_last), gn)
    version = y._version
    with torch.no_grad():
        assert torch.equal(ops.gn_act(x, gn, out=y), want)      # neighbours in one buffer
    assert y._version > version
    for out, residual in ((x, None), (ops.alias_window(buf, 4, 8), None), (y, ops.alias_window(buf, 12, 8)), (ops.alias_window(buf, 7, 8), None)):
        with pytest.raises(RuntimeError, match="shares elements"):
            ops.gn_act(x, gn, residual=residual, out=out)
    first = ops.gn_act(x, gn, out=ops.alias_window(buf, 16, 8))
    with pytest.raises(RuntimeError, match="belongs to a graph"):
        ops.gn_act(x, gn, out=first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 1024, 3, 3, 1), (2, 2048, 3, 3, 1), (1, 4088, 2, 2, 8), (1, 4096, 1, 5, 4096), (3, 72, 90, 70, 8)])
def test_wide_groups(shape, dtype):
    """Groups as wide as a cell's sums allow and wider, and the widest slabs."""
    x, dy, r, gn = make(shape, dtype, 15, residual=True)
    check(x, dy, r, gn, "silu", run(x, dy, r, gn, "silu"))


@pytest.mark.gpu
def test_expanded_gradients_and_half_precision():
    x, _, _, gn = make((2, 16, 5, 7, 4), torch.float32, 8)
    gn = gn.to(DEV)
    xd = x.to(DEV).requires_grad_()
    y = ops.gn_act(xd, gn)
    y.sum().backward()                                          # an expanded gradient
    got = {"y": y, "dx": xd.grad, "dgamma": gn.weight.grad, "dbeta": gn.bias.grad}
    check(x, torch.ones_like(x), None, gn.cpu(), "relu", got)
    with pytest.raises(TypeError, match="float16"):
        ops.gn_act(xd.detach().half(), gn)


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_image_and_group():
    x, dy, _, gn = make((3, 16, 4, 4, 4), torch.float32, 9)
    x[1, 5, 2, 2] = float("nan")
    x[2, 12, 0, 0] = float("inf")
    got = run(x, dy, None, gn, "relu")
    bad = torch.zeros(3, 16, dtype=torch.bool)
    bad[1, 4:8] = bad[2, 12:16] = True
    for k in ("y", "dx"):
        v = got[k].detach().cpu()
        assert torch.isfinite(v[~bad]).all() and torch.isnan(v[bad]).any(1).any(1).all(), k
    assert torch.isnan(got["y"].detach().cpu()[1, 4:8]).all()   # relu hands NaN on


@pytest.mark.gpu
def test_only_the_gradients_that_are_asked_for():
    x, dy, r, gn = make((2, 16, 5, 7, 4), torch.bfloat16, 10, residual=True)
    want = run(x, dy, r, gn, "relu")
    gn = gn.to(DEV)

    def cl(t):
        return t.to(DEV).contiguous(memory_format=torch.channels_last)
    rd = cl(r).requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.gn_act(cl(x), gn, residual=rd), rd, cl(dy))[0], want["dres"])
    assert torch.equal(torch.autograd.grad(ops.gn_act(cl(x), gn, residual=cl(r)), gn.bias, cl(dy))[0], want["dbeta"])
    xd = cl(x).requires_grad_()
    with torch.no_grad():
        gn.requires_grad_(False)
    assert torch.equal(torch.autograd.grad(ops.gn_act(xd, gn, residual=cl(r)), xd, cl(dy))[0], want["dx"])
    gn.requires_grad_(True)
    # without an activation the residual's gradient is dy, and the residual may change in between
    rd = cl(r).requires_grad_()
    y = ops.gn_act(cl(x), gn, residual=rd, act=0)
    assert torch.equal(torch.autograd.grad(y, rd, cl(dy))[0], cl(dy))
    # the same tensor as input and residual: both gradients arrive
    xd = cl(x).requires_grad_()
    a = torch.autograd.grad(ops.gn_act(xd, gn, residual=xd), xd, cl(dy))[0]
    x2, r2 = cl(x).requires_grad_(), cl(x).requires_grad_()
    b, c = torch.autograd.grad(ops.gn_act(x2, gn, residual=r2), [x2, r2], cl(dy))
    assert torch.equal(a, b + c)


@pytest.mark.gpu
def test_double_backward_and_bad_arguments_are_refused():
    x, dy, r, gn = make((2, 16, 5, 7, 4), torch.float32, 11, residual=True)
    gn = gn.to(DEV)
    xd = x.to(DEV).requires_grad_()
    with pytest.raises(RuntimeError, match="double backward"):
        torch.autograd.grad(ops.gn_act(xd, gn, act=ACTS["silu"]).square().sum(), xd, create_graph=True)
    y = ops.gn_act(xd, gn)
    first = torch.autograd.grad(y.sum(), xd, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y.sum(), xd)[0], first)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y.sum(), xd)
    xc = xd.detach().contiguous(memory_format=torch.channels_last).requires_grad_()       # (NCHW inputs are saved as a copy)
    y = ops.gn_act(xc, gn)
    with torch.no_grad():
        xc.add_(1.0)                                            # a saved tensor that changed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="channels"):
        ops.gn_act(torch.randn(1, 8, 4, 4, device=DEV), gn)
    with pytest.raises(RuntimeError, match="residual"):
        ops.gn_act(xd, gn, residual=r.to(DEV)[:1])
    with pytest.raises(RuntimeError, match="residual"):
        ops.gn_act(xd, gn, residual=r)
    with pytest.raises(_lib.UResNetHipError, match="non-positive"):
        ops.gn_act(xd[:0], gn)
    with pytest.raises(_lib.UResNetHipError, match="weight"):
        ops.gn_act(xd, hnn.GroupNorm(4, 16).to(DEV).bfloat16())
    with pytest.raises(_lib.UResNetHipError, match="weight"):
        ops.gn_act(xd, hnn.GroupNorm(4, 16))
    with pytest.raises(RuntimeError, match="window"):
        ops.gn_act(xd, gn, out=torch.empty(2, 16, 5, 8, device=DEV))


@pytest.mark.gpu
def test_saved_tensors_may_come_back_in_another_layout():
    """Saved-tensor hooks: an offload to the host that returns channels-first tensors (of a channel window as well), and one
    that returns something else."""
    x, dy, r, gn = make((2, 8, 6, 5, 4), torch.bfloat16, 16, residual=True)
    buf = torch.randn(2, 24, 6, 5, device=DEV).to(torch.bfloat16).contiguous(memory_format=torch.channels_last)
    gn = gn.to(DEV)
    dyd = dy.to(DEV)

    def grads():
        a, b = ops.alias_window(buf, 8, 8).requires_grad_(), r.to(DEV).contiguous(memory_format=torch.channels_last).requires_grad_()
        return torch.autograd.grad(ops.gn_act(a, gn, residual=b), [a, b, gn.weight, gn.bias], dyd)
    ops.alias_window(buf, 8, 8).copy_(x.to(DEV))
    want = grads()
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        assert all(torch.equal(p, q) for p, q in zip(grads(), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t):
        assert all(torch.equal(p, q) for p, q in zip(grads(), want))
    for change in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:1]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change), pytest.raises(RuntimeError, match="saved-tensor hook"):
            grads()


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences in the fp32 kernel: truncation h^2 and rounding 2^-24 |y| sqrt(N) / h leave 1e-3 at h = 1e-2."""
    x, dy, r, gn = make((1, 8, 3, 5, 2), torch.float32, 12, residual=True)
    gn = gn.to(DEV)
    cl = lambda t: t.to(DEV).contiguous(memory_format=torch.channels_last)      # noqa: E731
    xd, rd = cl(x).requires_grad_(), cl(r).requires_grad_()
    dyd = cl(dy)

    def loss(a, b):
        return (ops.gn_act(a, gn, residual=b, act=ACTS["silu"]).double() * dyd.double()).sum()
    grads = torch.autograd.grad(loss(xd, rd), [xd, rd, gn.weight, gn.bias])
    gen, h = torch.Generator().manual_seed(13), 1e-2
    for t, g in zip((xd, rd, gn.weight, gn.bias), grads):
        v = torch.randn(t.shape, generator=gen).to(DEV)
        v /= v.norm()
        with torch.no_grad():
            t += h * v
            up = loss(xd, rd)
            t -= 2 * h * v
            down = loss(xd, rd)
            t += h * v
        assert abs(((up - down) / (2 * h)).item() - (g.double() * v.double()).sum().item()) < 2e-3 * max(1.0, g.norm().item())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 64, 16, 16, 32), (6, 64, 128, 96, 32), (1, 80, 200, 150, 20)])
def test_the_same_call_gives_the_same_bits_on_any_stream_and_in_a_replayed_graph(shape):
    x, dy, r, gn = make(shape, torch.bfloat16, 14, residual=True)
    gn = gn.to(DEV)
    cl = lambda t: t.to(DEV).contiguous(memory_format=torch.channels_last)      # noqa: E731
    xd, rd, dyd = cl(x), cl(r), cl(dy)

    def step():
        a, b = xd.detach().requires_grad_(), rd.detach().requires_grad_()
        y = ops.gn_act(a, gn, residual=b, act=ACTS["relu"])
        return (y.detach(),) + torch.autograd.grad(y, [a, gn.weight, gn.bias, b], dyd)
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                                          # two captured graphs, replayed in turn
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            out = step()
        graphs.append((graph, out))
    for k in range(4):
        x2 = (x.float() * (1 + k)).to(x.dtype)
        xd.copy_(x2.to(DEV))
        graphs[k % 2][0].replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(graphs[k % 2][1], eager)), k


@pytest.mark.gpu
def test_a_captured_backward_pass_beside_a_live_eager_graph_is_refused():
    x, dy, _, gn = make((2, 16, 9, 5, 4), torch.bfloat16, 17)
    gn = gn.to(DEV)
    xd, dyd = (t.to(DEV).contiguous(memory_format=torch.channels_last) for t in (x, dy))

    def step():
        a = xd.detach().requires_grad_()
        y = ops.gn_act(a, gn)
        return torch.autograd.grad(y, [a, gn.weight, gn.bias], dyd)
    want = [t.clone() for t in step()]
    alive = ops.gn_act(xd, gn)                                  # holds the accumulators of weight and bias, on the default stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            step()
    torch.cuda.synchronize()
    alive.backward(dyd)                                         # the eager graph is unharmed
    assert torch.equal(gn.weight.grad, want[1]) and torch.equal(gn.bias.grad, want[2])
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        out = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.gpu
def test_two_calls_at_once_on_two_streams():
    a = make((2, 64, 96, 80, 32), torch.bfloat16, 15)
    b = make((3, 32, 50, 60, 4), torch.float32, 16)
    want = [run(*t[:2], None, t[3], "relu") for t in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    cl = lambda t: t.to(DEV).contiguous(memory_format=torch.channels_last)      # noqa: E731
    ins = [(cl(t[0]).requires_grad_(), cl(t[1]), t[3].to(DEV)) for t in (a, b)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, dy, gn = ins[i]
                y = ops.gn_act(x, gn)
                got[i] = (y,) + torch.autograd.grad(y, [x, gn.weight, gn.bias], dy)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(p, w[k]) for p, k in zip(g, ("y", "dx", "dgamma", "dbeta")))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """2^31 + elements in one tensor (4.3 GB in bf16): the last image equals the same image by itself."""
    n, c, h, w = 33, 64, 1024, 1024
    x = torch.empty((n, h, w, c), dtype=torch.bfloat16, device=DEV).permute(0, 3, 1, 2)
    last = torch.randn((1, h, w, c), device=DEV).to(torch.bfloat16).permute(0, 3, 1, 2)
    x.zero_()
    x[-1:].copy_(last)
    gn = hnn.GroupNorm(32, c).to(DEV)
    with torch.no_grad():
        a = ops.gn_act(x, gn)
        b = ops.gn_act(last, gn)
    # another split of the pixels sums in another order (64 bits): one fp32 rounding of the constants, one of the result
    assert torch.allclose(a[-1:].float(), b.float(), rtol=2.0 ** -7, atol=1e-6)
    assert not a[:-1].any()


# ------------------------------------------------------------------------------ what a tape node cannot serve
def refused_transforms(x, gn):
    """Forward mode (a dual input, weight, residual or output window) and tracing: refused on any device, before the device is
    looked at."""
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        named = {"weight": fwd.make_dual(gn.weight.detach(), torch.ones_like(gn.weight)), "bias": gn.bias.detach()}
        for call in (lambda: gn(dual), lambda: ops.gn_act(x, gn, residual=dual), lambda: ops.gn_act(x, gn, out=dual),
                     lambda: torch.func.functional_call(gn, named, (x,))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    with pytest.raises(NotImplementedError, match="torch.jit.trace"):
        torch.jit.trace(gn, (x,), check_trace=False)


def test_forward_mode_and_tracing_are_refused_without_a_gpu():
    refused_transforms(torch.randn(1, 8, 4, 4).contiguous(memory_format=torch.channels_last), hnn.GroupNorm(4, 8))


@pytest.mark.gpu
def test_forward_mode_tracing_and_function_transforms_are_refused():
    x, gn = torch.randn(2, 8, 4, 4, device=DEV).contiguous(memory_format=torch.channels_last), hnn.GroupNorm(4, 8).to(DEV)
    refused_transforms(x, gn)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: gn(t), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: gn(t).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: gn(t))(x[None])
    assert torch.isfinite(gn(x)).all()                          # and the operator still works afterwards


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "leakyrelu", "relu6"])
@pytest.mark.parametrize("residual", [False, True])
def test_zero_weights_beside_a_rectified_residual(residual, act):
    """pre = r exactly, 0 for half of the elements: the slope of the activation at 0, in both forms of the kernels."""
    for shape, dtype in (((2, 32, 9, 11, 8), torch.float32), ((3, 72, 90, 70, 8), torch.bfloat16)):
        x, dy, r, gn = make(shape, dtype, 18, residual=residual)
        with torch.no_grad():
            gn.weight.zero_()
            gn.bias.zero_()
        if residual:
            r = r.relu()
        check(x, dy, r, gn, act, run(x, dy, r, gn, act))


@pytest.mark.gpu
@pytest.mark.parametrize("shape, dtype", [((2, 64, 512, 512, 32), torch.bfloat16), ((64, 64, 64, 64, 8), torch.float32)])
def test_zero_weights_take_the_time_of_any_others(shape, dtype):
    """The same passes over the same bytes; half as much again is allowed for the clock."""
    x, dy, r, gn = make(shape, dtype, 19, residual=True)
    cl = lambda t: t.to(DEV).contiguous(memory_format=torch.channels_last)      # noqa: E731
    x, dy, r = cl(x).requires_grad_(), cl(dy), cl(r.relu()).requires_grad_()
    outs = []
    for zero in (False, True):
        norm = hnn.GroupNorm(shape[4], shape[1]).to(DEV)
        with torch.no_grad():
            norm.weight.copy_(0 * gn.weight if zero else gn.weight)
            norm.bias.copy_(0 * gn.bias if zero else gn.bias)
        outs.append((ops.gn_act(x, norm, residual=r), norm))
    best = [float("inf")] * 2
    for _ in range(25):
        for i, (y, norm) in enumerate(outs):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            torch.autograd.grad(y, [x, r, norm.weight, norm.bias], dy, retain_graph=True)
            end.record()
            end.synchronize()
            best[i] = min(best[i], start.elapsed_time(end))
    assert best[1] < 1.5 * best[0], best


# ------------------------------------------------------------------------------ every pixel counts once
def trips_per_workgroup(shape, dtype, vec):
    """What the launch plan of the streaming passes gives a workgroup: trips of 4 vectors per thread, 256 threads."""
    n, c, h, w, _ = shape
    v = (8 if dtype == torch.bfloat16 else 4) if vec else 1
    cq = -(-c // v)
    cqb = min(cq, 256)
    slots, zs = 256 // cqb, -(-cq // cqb)
    trips, per = -(-h * w // (4 * slots)), n * zs
    best, plan = 0.0, None
    for k in range(6, 0, -1):
        chunks = max(1, min(256 * k // per, trips))
        each = -(-trips // chunks)
        chunks = -(-trips // each)
        even = trips * per / (each * (-(-per * chunks // 256) * 256))
        if even > best * 1.02:
            best, plan = even, each
    return plan, h * w % (4 * slots)


def whole_numbers(shape, dtype, seed, act, residual, kink):
    """Inputs whose sums are whole numbers below 2^24 in every fp32 accumulator: x of mean exactly 0 in every channel, in random
    pixel order, dy and the residual small.  A pixel left out or counted twice shows.  kink: biases that put one value of x
    within 1e-8 of it."""
    n, c, h, w, groups = shape
    g = torch.Generator(device=DEV).manual_seed(seed)
    hw, rand = h * w, lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device=DEV, dtype=torch.int8).to(dtype)     # noqa: E731
    half = rand(-6, 7, n, hw // 2, c)
    order = torch.randperm(hw, generator=g, device=DEV)
    x = torch.cat([half, -half, half.new_zeros(n, hw % 2, c)], 1)[:, order].view(n, h, w, c).permute(0, 3, 1, 2)
    dy = rand(-3, 4, n, h, w, c).permute(0, 3, 1, 2)
    r = rand(-4, 5, n, h, w, c).permute(0, 3, 1, 2) if residual else None
    gn = hnn.GroupNorm(groups, c).to(DEV)
    with torch.no_grad():
        gn.weight.copy_(1 + 0.3 * torch.randn(c, generator=g, device=DEV))
        gn.bias.copy_(0.3 * torch.randn(c, generator=g, device=DEV))
        if kink:
            var = x[0].double().square().reshape(groups, -1).mean(1)
            gn.bias.copy_(-2 * (var + gn.eps).rsqrt().repeat_interleave(c // groups) * gn.weight)
    return x, dy, r, gn


def check_whole_numbers(shape, dtype, act, residual, kink=False, seed=20):
    x, dy, r, gn = whole_numbers(shape, dtype, seed, act, residual, kink)
    n, c, h, w, groups = shape
    xd, rd = x.detach().requires_grad_(), None if r is None else r.detach().requires_grad_()
    y = ops.gn_act(xd, gn, residual=rd, act=ACTS[act], slope=0.25)
    got = torch.autograd.grad(y, [xd, gn.weight, gn.bias] + ([] if r is None else [rd]), dy)

    # in 64 bits on the GPU: [n][pixels][groups][channels of a group]
    def split(t):
        return t.detach().permute(0, 2, 3, 1).reshape(n, h * w, groups, -1).double()
    ga, be = (t.detach().double().view(groups, -1) for t in (gn.weight, gn.bias))
    xs, m = split(x), h * w * (c // groups)
    assert xs.sum((1, 3)).abs().max() == 0
    rstd = (xs.square().sum((1, 3), keepdim=True) / m + gn.eps).rsqrt()
    pre = xs * rstd * ga + be
    size = (xs * rstd * ga).abs() + be.abs()
    if r is not None:
        pre, size = pre + split(r), size + split(r).abs()
    slope = {"none": torch.ones_like(pre), "relu": (pre > 0).double(), "leakyrelu": torch.where(pre > 0, 1.0, 0.25).double()}[act]
    gs = split(dy) * slope
    s1, s2 = gs.sum(1), (gs * xs).sum(1)                               # exact
    p1, p2 = (s1 * ga).sum(2) / m, (s2 * ga).sum(2) / m
    p1, p2 = p1.view(n, 1, groups, 1), p2.view(n, 1, groups, 1) * rstd
    dx = rstd * (ga * gs - p1 - xs * rstd * p2)
    size_dx = rstd * ((ga * gs).abs() + p1.abs() + (xs * rstd * p2).abs())
    half = HALF[dtype]

    def close(a, want, tol, what):
        off = (split(a) if a.dim() == 4 else a.detach().double().view(groups, -1)) - want
        assert (off.abs() <= tol).all(), "%s: off by %.3g" % (what, off.abs().max().item())
    # one rounding each of A, B (mean exactly 0: B is the bias), the product with the sum and the residual's sum: 4 of 2^-24
    close(y, pre * torch.where(pre > 0, 1.0, {"none": 1.0, "relu": 0.0, "leakyrelu": 0.25}[act]), half * pre.abs() + 6 * E24 * size, "y")
    # A, the two constants of a group (one rounding each after exact sums), two sums
    close(got[0], dx, half * dx.abs() + 6 * E24 * size_dx, "dx")
    # whole numbers times rstd (64 bits), rounded once
    want = (s2 * rstd[:, 0]).sum(0)
    close(got[1], want, E24 * want.abs() * 1.01 + 1e-12 * (s2.abs() * rstd[:, 0]).sum(0), "dgamma")
    close(got[2], s1.sum(0), E24 * s1.sum(0).abs(), "dbeta")
    if r is not None:
        close(got[3], gs, torch.zeros(()), "dres") if act != "none" else close(got[3], split(dy), torch.zeros(()), "dres")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES + [(2, 1024, 3, 3, 1), (1, 4088, 2, 2, 8), (3, 72, 90, 70, 8), (64, 64, 32, 32, 8), (5, 60, 41, 47, 20)])
def test_every_pixel_counts_once(shape, dtype):
    for act, residual in (("none", False), ("relu", True)):
        check_whole_numbers(shape, dtype, act, residual)


LONG = [  # shape, dtype, vectors, trips per workgroup
    ((6, 64, 181, 361, 32), torch.bfloat16, True, 2),
    ((1, 64, 523, 1031, 32), torch.bfloat16, True, 17),
    ((2, 512, 113, 181, 32), torch.bfloat16, True, 2),
    ((1, 256, 409, 479, 8), torch.bfloat16, True, 4),
    ((3, 40, 331, 499, 5), torch.bfloat16, True, 2),
    ((1, 64, 421, 691, 8), torch.float32, True, 3),
    ((2, 96, 173, 397, 32), torch.float32, True, 7),
    ((1, 60, 277, 307, 20), torch.bfloat16, False, 7),
    ((2, 3, 557, 1021, 3), torch.float32, False, 7),
    ((4, 300, 53, 61, 300), torch.bfloat16, False, 13),
]


def test_long_shapes_take_several_trips_and_leave_a_remainder():
    for shape, dtype, vec, trips in LONG:
        got, rest = trips_per_workgroup(shape, dtype, vec)
        assert got == trips and rest, (shape, got, rest)


@pytest.mark.gpu
@pytest.mark.parametrize("act, residual, kink", [("none", False, False), ("relu", False, True), ("relu", True, False), ("leakyrelu", True, True)])
@pytest.mark.parametrize("shape, dtype, vec, trips", LONG)
def test_every_pixel_counts_once_over_several_trips(shape, dtype, vec, trips, act, residual, kink):
    check_whole_numbers(shape, dtype, act, residual, kink)


@pytest.mark.gpu
@pytest.mark.parametrize("act, low, high", [("relu", 0.0, None), ("relu6", 0.0, 6.0), ("hswish", -3.0, None)])
@pytest.mark.parametrize("shape, dtype", [((2, 32, 9, 11, 8), torch.float32), ((3, 72, 90, 70, 8), torch.bfloat16), ((2, 5, 6, 7, 5), torch.float32)])
def test_infinite_gradients_where_the_slope_is_zero_count_for_nothing(shape, dtype, act, low, high):
    """As the gradient of a square root behind a ReLU is: infinite exactly where nothing passes."""
    x, dy, r, gn = make(shape, dtype, 21, residual=True)
    r = (4 * r.float()).to(dtype)
    n, c, h, w, groups = shape
    xs = x.double().reshape(n, groups, -1)
    xhat = ((xs - xs.mean(2, keepdim=True)) * (xs.var(2, unbiased=False, keepdim=True) + gn.eps).rsqrt()).view(n, c, h, w)
    pre = xhat * gn.weight.detach().double().view(c, 1, 1) + gn.bias.detach().double().view(c, 1, 1) + r.double()
    closed = (pre < low - 1e-3) | (pre > high + 1e-3) if high is not None else pre < low - 1e-3
    bad = dy.clone()
    bad[closed] = float("inf")
    bad[closed & (r > 1)] = float("nan")
    want = run(x, torch.where(closed, torch.zeros_like(dy), dy), r, gn, act)
    got = run(x, bad, r, gn, act)
    assert closed.any() and all(torch.equal(got[k], want[k]) for k in want)


@pytest.mark.gpu
def test_activation_checkpointing_and_errors_of_saved_tensor_hooks():
    """Checkpointing without reentry ends its recomputation by an exception out of the hook that packs the last saved tensor."""
    from torch.utils.checkpoint import checkpoint
    x, dy, r, gn = make((2, 16, 9, 5, 4), torch.bfloat16, 22, residual=True)
    gn, cl = gn.to(DEV), lambda t: t.to(DEV).contiguous(memory_format=torch.channels_last)      # noqa: E731
    second = hnn.GroupNorm(2, 16).to(DEV)
    xd, rd, dyd = cl(x).requires_grad_(), cl(r).requires_grad_(), cl(dy)

    def last(a, b):
        return ops.gn_act(a, gn, residual=b)

    def inside(a, b):
        return ops.gn_act(ops.gn_act(a, gn, residual=b, act=ACTS["silu"]), second).float() * 2
    for f, norms in ((last, [gn]), (inside, [gn, second])):
        wrt = [xd, rd] + [p for m in norms for p in m.parameters()]
        want = torch.autograd.grad(f(xd, rd), wrt, dyd.to(f(xd, rd).dtype))
        for early_stop in (True, False):
            with torch.utils.checkpoint.set_checkpoint_early_stop(early_stop):
                y = checkpoint(f, xd, rd, use_reentrant=False)
                assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, wrt, dyd.to(y.dtype)), want))

    def fails(t):
        raise KeyError("the hook's own")
    with torch.autograd.graph.saved_tensors_hooks(fails, lambda t: t), pytest.raises(KeyError, match="the hook's own"):
        ops.gn_act(xd, gn)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, fails):
        y = ops.gn_act(xd, gn)
    with pytest.raises(KeyError, match="the hook's own"):
        y.sum().backward()
    with pytest.raises(_lib.UResNetHipError, match="limits"):      # errors of the entry points as before
        ops.gn_act(torch.zeros(1, 16392, 1, 1, device=DEV), hnn.GroupNorm(1, 16392).to(DEV))
