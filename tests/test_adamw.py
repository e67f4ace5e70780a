"""train.AdamW (32- and 8-bit moments) and train.clip_grad_norm_ against the formulas in 64 bits.

Tolerances.  A step in fp32 rounds each of its operations once: m and v carry at most 4 roundings of 2^-24 (6 with the clipping
factor), the update at most 12 of itself, the parameter 2 of itself.  The norm is summed in 64 bits and rounded once (2^-24;
one more where it is multiplied).  8-bit codes are compared as codes: an element whose value lies within the fp32 error of a
border between two codes may take the other one, so codes may differ by one step in at most FLIPS of the elements (the
relative error of the value, 8 * 2^-24, over the distance between borders, 2^-4, is 8e-6)."""
import math

import pytest
import torch

from uresnet_amd import _lib, ops, train

DEV = "cuda:0"
E24 = 2.0 ** -24
FLIPS = 1e-4
CODES = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
SIZES = [(1,), (3,), (255,), (256,), (257,), (64, 3, 7, 7), (2048,), (2049,), (33, 65), (4099,), (128, 64, 3, 3), (5, 0)]


def tensors(seed, sizes=SIZES, scale=0.05):
    g = torch.Generator().manual_seed(seed)
    return [scale * torch.randn(s, generator=g) for s in sizes]


def params_on_gpu(values, grads):
    out = []
    for v, g in zip(values, grads):
        p = torch.nn.Parameter(v.to(DEV))
        if g is not None:
            p.grad = g.to(DEV)
        out.append(p)
    return out


def dither(places, step):
    mask = 0xFFFFFFFF
    h = (places * 0x9E3779B9 + step * 0xA3D8F1B5) & mask
    h = ((h ^ (h >> 16)) * 0x45D9F3B5) & mask
    h = ((h ^ (h >> 15)) * 0x2C92774D) & mask
    return (h ^ (h >> 16)) & 0xFFFFF


def quantise(t, places=None, step=None):
    """Codes (as values) and scales of a flat tensor in 64 bits; the last block may be short."""
    n = t.numel()
    blocks = torch.cat([t, t.new_zeros(-n % 256)]).view(-1, 256)
    finite = torch.where(blocks.isfinite(), blocks.abs(), blocks.new_zeros(()))
    scale = finite.amax(1).clamp_min(2.0 ** -100) / 448
    y = (blocks / scale.unsqueeze(1)).view(-1)[:n]
    a = y.abs().nan_to_num(0.0, 0.0).clamp_max(448)
    lo = (torch.bucketize(a, CODES, right=True) - 1).clamp(0, 125)
    part = (a - CODES[lo]) / (CODES[lo + 1] - CODES[lo])
    if step is None:
        up = torch.where(lo % 2 == 0, part > 0.5, part >= 0.5)
    else:
        up = part + dither(places, step).double() / 2.0 ** 20 >= 1
    q = CODES[lo + up.long()] * y.sign()
    return torch.where(y.isfinite(), q, torch.full_like(q, float("nan"))), scale


def dequantise(q, scale):
    return q.double() * scale.double().repeat_interleave(256)[:q.numel()]


def reference_step(p, g, m, v, t, lr, b1, b2, eps, wd, factor):
    p, g, m, v = p.double(), g.double() * factor, m.double(), v.double()
    m = m + (g - m) * (1 - b1)
    v = v * b2 + (1 - b2) * g * g
    step = lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return p * (1 - lr * wd) - step, m, v, step.abs()


def within(got, want, tol, what):
    got = got.detach().double().cpu().reshape(want.shape)
    off = (got - want).abs()
    assert (off <= tol).all(), "%s: off by %.3g" % (what, off.max().item())


def factor_of(grads, limit, scale=1.0):
    norm = math.sqrt(sum(g.double().square().sum().item() for g in grads)) * abs(scale)
    return norm, scale * (1.0 if limit is None else min(1.0, limit / (norm + 1e-6)))


# ------------------------------------------------------------------------------ refusals and checkpoints (CPU)
def test_refusals_without_a_gpu():
    p = torch.nn.Parameter(torch.zeros(4))
    for kw, err in ((dict(state_bits=16), ValueError), (dict(max_grad_norm=0.0), ValueError), (dict(lr=-1.0), ValueError),
                    (dict(betas=(0.9, 1.0)), ValueError), (dict(eps=-1e-8), ValueError), (dict(weight_decay=-0.1), ValueError),
                    (dict(lr=torch.tensor(0.1)), TypeError)):
        with pytest.raises(err):
            train.AdamW([p], **kw)
    opt = train.AdamW([p])
    assert opt.step() is None                                  # no gradients: nothing to do
    p.grad = torch.ones(4)
    with pytest.raises(_lib.UResNetHipError, match="GPU"):
        opt.step()
    with pytest.raises(_lib.UResNetHipError, match="GPU"):
        train.clip_grad_norm_([p], 1.0)
    with pytest.raises(NotImplementedError):
        train.clip_grad_norm_([p], 1.0, norm_type=1)
    with pytest.raises(ValueError):
        train.clip_grad_norm_([p], -1.0)
    assert train.clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0).item() == 0.0
    with pytest.raises(_lib.UResNetHipError, match="contiguous fp32"):
        train.AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))]).state_buffers()


def test_parameters_listed_twice_or_sharing_memory_are_refused():
    import warnings
    p, q = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(3))
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with pytest.raises(ValueError, match="twice"):
            train.AdamW([p, q, p])
        opt = train.AdamW([q])
        with pytest.raises(ValueError, match="twice"):
            opt.add_param_group(dict(params=[p, p]))
    assert len(opt.param_groups) == 1
    flat = torch.zeros(10)
    a, b, c = (torch.nn.Parameter(flat[i:i + 5]) for i in (0, 5, 4))
    train.AdamW([a, b]).state_buffers()                        # neighbours
    with pytest.raises(_lib.UResNetHipError, match="share memory"):
        train.AdamW([a, c]).state_buffers()


def test_entry_points_refuse_before_any_launch():
    import ctypes as C
    n = C.c_longlong()

    def table(grads=(16,), sizes=(5,), size=1 << 20, count=None):
        arr = [(C.c_longlong * len(v))(*v) for v in (grads, sizes)]
        _lib.call("ur_param_table", None, arr[0], arr[1], None, len(grads) if count is None else count, 16, size, None, 0.0, 0.0, 0.0,
                  C.byref(n), None)
    for kw in (dict(grads=(0,)), dict(sizes=(0,)), dict(sizes=(-1,)), dict(size=8), dict(count=0), dict(sizes=(1 << 41,)),
               dict(grads=(16,) * 5, sizes=(1 << 40,) * 5)):
        with pytest.raises(_lib.UResNetHipError, match="param_table"):
            table(**kw)
    assert _lib.query("ur_grad_sqnorm_max_parts") == _lib.query("ur_param_table_max_rows") == 1024
    with pytest.raises(_lib.UResNetHipError, match="more than"):
        table(grads=(16,) * 1025, sizes=(1,) * 1025)
    def adamw(bits=32, m=16, scale=16, chunks=1, nparts=0, parts=None):
        _lib.call("ur_adamw_multi", 16, 1, chunks, bits, m, 16, scale, scale, 1e-3, 0.9, 0.999, 1e-8, 0.0, parts, nparts, 1.0, 1.0, None, None)
    for kw in (dict(bits=16), dict(m=None), dict(m=24), dict(bits=8, scale=None), dict(chunks=0), dict(nparts=3)):
        with pytest.raises(_lib.UResNetHipError, match="adamw_multi"):
            adamw(**kw)
    k = C.c_int()
    with pytest.raises(_lib.UResNetHipError, match="grad_sqnorm"):
        _lib.call("ur_grad_sqnorm", 16, 1, 0, 16, C.byref(k), None)
    with pytest.raises(_lib.UResNetHipError, match="grad_clip"):
        _lib.call("ur_grad_clip", 16, 1, 1, 16, 0, 1.0, None, None)


def test_state_dict_moves_to_torch_and_back():
    vals = tensors(1, SIZES[:6])
    tp = [torch.nn.Parameter(v.clone()) for v in vals]
    topt = torch.optim.AdamW([{"params": tp[:3]}, {"params": tp[3:], "weight_decay": 0.0}], lr=1e-3, weight_decay=0.02)
    for p in tp[1:]:
        p.grad = torch.ones_like(p)
    topt.step(), topt.step()
    op = [torch.nn.Parameter(v.clone()) for v in vals]
    opt = train.AdamW([{"params": op[:3]}, {"params": op[3:]}])
    opt.load_state_dict(topt.state_dict())
    assert opt.param_groups[0]["lr"] == 1e-3 and opt.param_groups[1]["weight_decay"] == 0.0
    assert op[0] not in opt.state and int(opt.state[op[1]]["step"]) == 2
    for a, b in zip(op[1:], tp[1:]):
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(opt.state[a][k], topt.state[b][k])
    back = torch.optim.AdamW([{"params": tp[:3]}, {"params": tp[3:]}])
    back.load_state_dict(opt.state_dict())
    assert back.param_groups[0]["weight_decay"] == 0.02 and float(back.state[tp[1]]["step"]) == 2.0
    back.step()                                                # torch keeps stepping with it
    for bad in ({"amsgrad": True}, {"maximize": True}, {"decoupled_weight_decay": False}):
        sd = topt.state_dict()
        sd["param_groups"][0].update(bad)
        with pytest.raises(NotImplementedError):
            opt.load_state_dict(sd)
    with pytest.raises(ValueError, match="8-bit"):
        train.AdamW([{"params": op[:3]}, {"params": op[3:]}], state_bits=8).load_state_dict(topt.state_dict())
    with pytest.raises(ValueError, match="groups"):
        train.AdamW(op).load_state_dict(topt.state_dict())


def test_eight_bit_checkpoints_round_trip_through_a_file(tmp_path):
    vals = tensors(2, SIZES[:6])
    ps = [torch.nn.Parameter(v) for v in vals]
    opt = train.AdamW(ps, state_bits=8)
    state = {}
    for i, v in enumerate(vals):
        q, s = quantise(v.double().flatten())
        r, u = quantise(v.double().flatten().abs(), torch.arange(v.numel()), 3)
        state[i] = {"step": torch.tensor(7.0), "exp_avg": q.float().to(torch.float8_e4m3fn).view(v.shape), "exp_avg_scale": s.float(),
                    "exp_avg_sq_root": r.float().to(torch.float8_e4m3fn).view(v.shape), "exp_avg_sq_root_scale": u.float()}
    opt.load_state_dict({"state": state, "param_groups": opt.state_dict()["param_groups"]})
    path = str(tmp_path / "opt.pth")
    torch.save(opt.state_dict(), path)
    sd = torch.load(path, weights_only=True)
    other = train.AdamW(ps, state_bits=8)
    other.load_state_dict(sd)
    for i, p in enumerate(ps):
        assert int(other.state[p]["step"]) == 7
        for k in state[i]:
            if k != "step":
                assert torch.equal(other.state[p][k].float(), state[i][k].float()), k
    with pytest.raises(ValueError, match="32-bit"):
        train.AdamW(ps).load_state_dict(sd)
    assert sorted(other.state_buffers()) == ["exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale"]
    import copy
    clone = copy.deepcopy(other)
    assert clone.state_dict()["state"][3]["step"] == 7.0
    # a parameter that joins the group later leaves the others' moments as they were
    new = torch.nn.Parameter(torch.zeros(300))
    other.param_groups[0]["params"].append(new)
    other.state_buffers()
    assert torch.equal(other.state[ps[5]]["exp_avg"].float(), state[5]["exp_avg"].float()) and int(other.state[ps[5]]["step"]) == 7


def made_up_state(ps, bits, step=7.0):
    state = {}
    for i, p in enumerate(ps):
        n, g = p.numel(), torch.Generator().manual_seed(i)
        m, v = torch.randn(n, generator=g), torch.rand(n, generator=g)
        if bits == 32:
            state[i] = {"exp_avg": m.view(p.shape), "exp_avg_sq": v.view(p.shape)}
        else:
            (q, s), (r, u) = quantise(m.double()), quantise(v.double(), torch.arange(n), 3)
            state[i] = {"exp_avg": q.to(torch.float8_e4m3fn).view(p.shape), "exp_avg_scale": s.float(),
                        "exp_avg_sq_root": r.to(torch.float8_e4m3fn).view(p.shape), "exp_avg_sq_root_scale": u.float()}
        state[i]["step"] = torch.tensor(step)
    return state


@pytest.mark.parametrize("bits", [32, 8])
def test_loading_keeps_every_group_key_and_runs_the_hooks(bits):
    """A scheduler continues from a loaded state (its initial_lr travels in the groups); registered hooks run, those before the
    load may change what is loaded, those after it see the loaded moments."""
    ps = [torch.nn.Parameter(v) for v in tensors(40, SIZES[:5])]
    opt = train.AdamW(ps, lr=0.5, state_bits=bits)
    torch.optim.lr_scheduler.StepLR(opt, 3)
    opt.param_groups[0]["note"] = "kept"
    sd = {**opt.state_dict(), "state": made_up_state(ps, bits)}
    other = train.AdamW(ps, state_bits=bits)
    seen = []

    def before(o, d):
        seen.append("before")
        d["param_groups"][0]["eps"] = 1e-6
        return {**d}

    def after(o):
        seen.append(o.state[ps[3]]["exp_avg"].float().clone())
    other.register_load_state_dict_pre_hook(before)
    other.register_load_state_dict_post_hook(after)
    other.load_state_dict(sd)
    group = other.param_groups[0]
    assert group["note"] == "kept" and group["lr"] == 0.5 and group["eps"] == 1e-6 and group["state_bits"] == bits
    sched = torch.optim.lr_scheduler.StepLR(other, 3, last_epoch=2)
    assert sched.get_last_lr()[0] == pytest.approx(0.05)
    assert seen[0] == "before" and torch.equal(seen[1], sd["state"][3]["exp_avg"].float()) and len(seen) == 2
    for i, p in enumerate(ps):
        for k, v in other.state[p].items():
            assert torch.equal(v.float(), sd["state"][i][k].float()), k
    other.load_state_dict(sd)                                  # nothing of the first load is left behind
    assert len(seen) == 4


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_does_not_fit_leaves_the_optimiser_as_it_was(bits):
    ps = [torch.nn.Parameter(v) for v in tensors(41, SIZES[:5])]
    opt = train.AdamW(ps, lr=0.25, state_bits=bits)
    opt.load_state_dict({**opt.state_dict(), "state": made_up_state(ps, bits)})
    want = {k: v.float().clone() for k, v in opt.state_buffers().items()}
    for key in ("exp_avg", "exp_avg_sq") if bits == 32 else ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale"):
        bad = {**opt.state_dict(), "state": made_up_state(ps, bits, 9.0)}
        bad["param_groups"][0]["lr"] = 1.0
        bad["state"][4][key] = torch.cat([bad["state"][4][key].flatten().float()] * 2)
        with pytest.raises(ValueError, match=key):
            opt.load_state_dict(bad)
        state, group = opt.state, opt.param_groups[0]
        assert group["lr"] == 0.25 and all(int(state[p]["step"]) == 7 for p in ps)
        assert all(torch.equal(v.float(), want[k]) for k, v in opt.state_buffers().items())
        assert state[ps[4]]["exp_avg"].untyped_storage().data_ptr() == opt.state_buffers()["exp_avg"].untyped_storage().data_ptr()

    def fails(o):
        raise OSError("a hook that fails")
    handle = opt.register_load_state_dict_post_hook(fails)
    with pytest.raises(OSError):
        opt.load_state_dict({**opt.state_dict(), "state": made_up_state(ps, bits, 9.0)})
    handle.remove()
    assert int(opt.state[ps[0]]["step"]) == 7 and opt.step() is None
    assert all(torch.equal(v.float(), want[k]) for k, v in opt.state_buffers().items())


def test_eight_bit_moments_need_a_first_beta_that_lets_them_fall():
    """A falling m leaves every code that nearest rounding could keep it on only if 9/8 * b1 < 17/16."""
    values = (1 + torch.arange(8) / 8).double()
    for b1, moves in ((17 / 18 - 1e-6, True), (0.9, True), (0.95, False)):
        rounded = (values * b1 * 16).float().to(torch.float8_e4m3fn).double() / 16
        assert bool((rounded < values).all()) is moves
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="17/18"):
        train.AdamW([p], betas=(0.95, 0.999), state_bits=8)
    train.AdamW([p], betas=(0.95, 0.999))
    opt = train.AdamW([p], betas=(17 / 18, 0.999), state_bits=8)
    sd = opt.state_dict()
    sd["param_groups"][0]["betas"] = (0.99, 0.999)
    with pytest.raises(ValueError, match="17/18"):
        opt.load_state_dict(sd)
    assert opt.param_groups[0]["betas"][0] == 17 / 18
    opt.param_groups[0]["betas"] = (0.95, 0.999)               # as a scheduler that cycles the momentum sets it
    with pytest.raises(_lib.UResNetHipError, match="17/18"):
        opt.step()
    with pytest.raises(_lib.UResNetHipError, match="17/18"):
        _lib.call("ur_adamw_multi", 16, 1, 1, 8, 16, 16, 16, 16, 1e-3, 0.95, 0.999, 1e-8, 0.0, None, 0, 1.0, 1.0, None, None)


@pytest.mark.parametrize("bits", [32, 8])
def test_what_a_caller_puts_into_the_state_counts(bits):
    """Entries emptied or replaced between steps, tensors replaced inside an entry, entries of the caller's own."""
    ps = [torch.nn.Parameter(v) for v in tensors(42, SIZES[:5])]
    opt = train.AdamW(ps, state_bits=bits)
    opt.load_state_dict({**opt.state_dict(), "state": made_up_state(ps, bits)})
    want = {i: {k: v.float().clone() for k, v in opt.state[p].items()} for i, p in enumerate(ps)}
    opt.state[ps[0]] = {}
    opt.state[ps[2]]["exp_avg"] = torch.full(ps[2].shape, 2.0)
    opt.state[ps[3]] = {**opt.state[ps[3]], "step": torch.tensor(3.0), "mine": "kept"}
    opt.state[ps[4]]["exp_avg"].zero_()                        # in place, as ever
    sd = opt.state_dict()["state"]
    assert sd[0] == {} and [float(sd[i]["step"]) for i in (1, 2, 3, 4)] == [7, 7, 3, 7]
    opt.step()                                                 # no gradients: only what the optimiser holds is looked at
    flat, at = opt.state_buffers()["exp_avg"].float(), 0
    for i, p in enumerate(ps):
        n = p.numel()
        expected = {0: torch.zeros(n), 2: torch.full((n,), 2.0), 4: torch.zeros(n)}.get(i, want[i]["exp_avg"].flatten())
        assert torch.equal(flat[at:at + n], expected), i
        at += -(-n // 256) * 256
    assert not opt.state[ps[0]] and opt.state[ps[3]]["mine"] == "kept" and int(opt.state[ps[3]]["step"]) == 3
    pool = opt._pools[0]
    opt.step()
    assert opt._pools[0] is pool and 0 in pool.waiting         # nothing changed since: nothing is built again
    del opt.state[ps[1]]
    opt.step()
    assert not opt.state_buffers()["exp_avg"].float()[256:256 + 3].any() and sorted(opt._pools[0].waiting) == [0, 1]


def test_dither_is_uniform_over_places_and_steps():
    """Mean and correlation of 2^16 draws against their standard errors (4 of them)."""
    n = 1 << 16
    for step in (1, 2, 1000):
        u = dither(torch.arange(n), step).double() / 2 ** 20
        assert abs(u.mean().item() - 0.5) < 4 * math.sqrt(1 / 12 / n)
        assert abs(((u[1:] - 0.5) * (u[:-1] - 0.5)).mean().item()) < 4 / 12 / math.sqrt(n)
        w = dither(torch.arange(n), step + 1).double() / 2 ** 20
        assert abs(((u - 0.5) * (w - 0.5)).mean().item()) < 4 / 12 / math.sqrt(n)
        assert torch.histc(u, 64).sub(n / 64).abs().max() < 5 * math.sqrt(n / 64)


# ------------------------------------------------------------------------------ steps (GPU)
@pytest.mark.gpu
@pytest.mark.parametrize("limit", [None, 0.5, 1e6])
@pytest.mark.parametrize("bits", [32, 8])
def test_three_steps_against_the_formula(bits, limit):
    lr, b1, b2, eps, wd = 1e-2, 0.9, 0.99, 1e-8, 0.1
    vals = tensors(3)
    ps = params_on_gpu(vals, [None] * len(vals))
    opt = train.AdamW(ps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=bits, max_grad_norm=limit)
    first = [0]
    for v in vals:
        first.append(first[-1] + -(-v.numel() // 256) * 256)
    for t in range(1, 4):
        grads = tensors(10 + t, scale=0.3)
        if t == 2:
            grads[4] = grads[4] * 0                            # a tensor without any gradient signal
        for p, g in zip(ps, grads):
            p.grad = g.to(DEV)
        before = [(p.detach().cpu().clone(), {k: v.cpu().clone() for k, v in opt.state[p].items()} if p in opt.state else None) for p in ps]
        opt.step()
        torch.cuda.synchronize()
        norm, factor = factor_of(grads, limit)
        if limit is not None:
            assert abs(opt.grad_norm.item() - norm) <= 2 * E24 * norm
        else:
            assert opt.grad_norm is None
        for i, (p, g, (p0, st)) in enumerate(zip(ps, grads, before)):
            assert torch.equal(p.grad.cpu(), g)                # the step leaves the gradients
            n = g.numel()
            if n == 0:
                continue
            flat = g.flatten()
            if st is None:
                m = v = torch.zeros(n, dtype=torch.float64)
            elif bits == 32:
                m, v = st["exp_avg"].flatten(), st["exp_avg_sq"].flatten()
            else:
                m = dequantise(st["exp_avg"].flatten(), st["exp_avg_scale"])
                v = dequantise(st["exp_avg_sq_root"].flatten(), st["exp_avg_sq_root_scale"]).square()
            want, m1, v1, upd = reference_step(p0.flatten(), flat, m, v, t, lr, b1, b2, eps, wd, factor)
            size_m = m.double().abs() + 0.1 * flat.double().abs() * abs(factor)
            # m by cancellation: relative to its terms, which the update inherits
            upd = upd * (1 + size_m / m1.abs().clamp_min(1e-300)).nan_to_num(1.0, 1.0)
            within(p.detach().flatten(), want, 2 * E24 * want.abs() + 2 * E24 * p0.flatten().double().abs() + 16 * E24 * upd + 1e-30, "p")
            new = {k: x.cpu() for k, x in opt.state[p].items()}
            assert int(new["step"]) == t
            if bits == 32:
                within(new["exp_avg"], m1.view(g.shape), 8 * E24 * size_m.view(g.shape) + 1e-40, "exp_avg")
                within(new["exp_avg_sq"], v1.view(g.shape), 8 * E24 * v1.view(g.shape) + 1e-40, "exp_avg_sq")
                continue
            places = torch.arange(n) + first[i]
            for key, (q, s) in (("exp_avg", quantise(m1)), ("exp_avg_sq_root", quantise(v1.sqrt(), places, t))):
                within(new[key + "_scale"], s, 16 * E24 * s, key + "_scale")
                got = new[key].flatten().double()
                differ = got != q
                assert differ.sum() <= max(1, FLIPS * n), (key, int(differ.sum()))
                assert ((got - q).abs() <= 0.126 * q.abs().clamp_min(2.0 ** -6)).all()
    for k, buf in opt.state_buffers().items():                 # what lies between the tensors stays zero
        if not k.endswith("scale"):
            used = torch.zeros(buf.numel(), dtype=torch.bool)
            for at, v in zip(first, vals):
                used[at:at + v.numel()] = True
            assert not buf.float().cpu()[~used].any(), k


@pytest.mark.gpu
def test_codes_of_the_device_are_those_of_torch():
    """Every e4m3 code decodes to its value (lr 0, b1 = b2 = 0 would lose it: b close to 1 keeps m), and nearest rounding on
    the device is that of torch's cast for values on, between and halfway between codes."""
    codes = torch.cat([CODES, -CODES[1:]])
    mid = (CODES[1:] + CODES[:-1]) / 2
    vals = torch.cat([codes, mid, -mid, torch.tensor([448.0])]).float()
    n = vals.numel()
    pad = -n % 255
    vals = torch.cat([vals, vals.new_zeros(pad)]).view(-1, 255)
    vals = torch.cat([vals, torch.full((vals.shape[0], 1), 448.0)], 1).flatten()        # every block has the scale 1
    p = torch.nn.Parameter(torch.zeros(vals.numel(), device=DEV))
    opt = train.AdamW([p], lr=0.0, betas=(0.0, 0.0), state_bits=8)                     # m = g, r = |g|
    p.grad = vals.to(DEV)
    opt.step()
    st = opt.state[p]
    assert (st["exp_avg_scale"] == 1).all()
    assert torch.equal(st["exp_avg"].cpu().float(), vals.to(torch.float8_e4m3fn).float())
    on_code = torch.isin(vals.abs().double(), CODES)
    # sqrt(g * g) is g within a rounding, so a code goes to itself or, just below, up to it with all but 2^-20 probability
    r = st["exp_avg_sq_root"].cpu().float()
    assert (r[on_code] == vals.abs()[on_code]).float().mean() > 0.999


@pytest.mark.gpu
def test_the_rounding_of_the_root_is_right_in_expectation():
    """64 steps with b2 = 0 and the same gradients: the mean of the codes' values approaches the value.  A code step is at most
    1/8 of a value: the standard error of the mean is below 1/16/8 of it, averaged over 4096 elements below 1.3e-4."""
    g = torch.rand(4096, generator=torch.Generator().manual_seed(4)) * 400 + 40
    g[::256] = 448.0
    p = torch.nn.Parameter(torch.zeros(4096, device=DEV))
    opt = train.AdamW([p], lr=0.0, betas=(0.0, 0.0), state_bits=8)
    p.grad = g.to(DEV)
    total = torch.zeros(4096, dtype=torch.float64)
    for _ in range(64):
        opt.step()
        total += dequantise(opt.state[p]["exp_avg_sq_root"].cpu(), opt.state[p]["exp_avg_sq_root_scale"].cpu())
    assert abs((total / 64 / g.double()).mean().item() - 1) < 5 * 1.3e-4


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_non_finite_gradients_and_extreme_sizes(bits):
    """NaN and infinity stay with their elements; blocks of zeros, of tiny and of huge values keep their scale finite."""
    n = 256 * 5
    g = torch.randn(n, generator=torch.Generator().manual_seed(5))
    g[3], g[700], g[701] = float("nan"), float("inf"), -float("inf")
    g[256:512] = 0
    g[768:1024] *= 1e-35
    g[1024:] *= 1e15
    p = torch.nn.Parameter(torch.ones(n, device=DEV))
    opt = train.AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits)
    p.grad = g.to(DEV)
    for _ in range(2):
        opt.step()
    bad = ~g.isfinite()
    out = p.detach().cpu()
    assert not out[bad].isfinite().all() and out[~bad].isfinite().all()
    assert (out[256:512] == 1).all()
    # the others move as if the bad ones were not there
    q = torch.nn.Parameter(torch.ones(n, device=DEV))
    ref = train.AdamW([q], lr=1e-3, weight_decay=0.0, state_bits=bits)
    q.grad = torch.where(bad, torch.zeros_like(g), g).to(DEV)
    for _ in range(2):
        ref.step()
    assert torch.equal(out[~bad], q.detach().cpu()[~bad])
    if bits == 8:
        assert all(v.isfinite().all() for k, v in opt.state_buffers().items() if k.endswith("scale"))


@pytest.mark.gpu
def test_clipping_with_a_nan_or_infinite_norm_follows_torch():
    for bad in (float("nan"), float("inf")):
        g = torch.ones(300)
        g[7] = bad
        p, q = torch.nn.Parameter(torch.zeros(300, device=DEV)), torch.nn.Parameter(torch.zeros(300))
        p.grad, q.grad = g.to(DEV), g.clone()
        norm = train.clip_grad_norm_([p], 1.0)
        want = torch.nn.utils.clip_grad_norm_([q], 1.0)
        assert torch.equal(norm.cpu(), want) or (norm.isnan() and want.isnan())
        assert torch.equal(p.grad.cpu().isnan(), q.grad.isnan()) and torch.equal(p.grad.cpu().nan_to_num(), q.grad.nan_to_num())
        p.grad = g.to(DEV)
        with pytest.raises(RuntimeError, match="finite"):
            train.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
        assert torch.equal(p.grad.cpu().nan_to_num(), g.nan_to_num())


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [SIZES, [(1,)], [(40001,)] * 3, [(7,)] * 200, [(1 << 22,), (5,)], [(5,)] * 2500])
@pytest.mark.parametrize("limit", [0.25, 1e9])
def test_clip_grad_norm(sizes, limit):
    grads = tensors(6, sizes, 1.0)
    ps = params_on_gpu([torch.zeros(s) for s in sizes], grads)
    norm, factor = factor_of(grads, limit)
    got = train.clip_grad_norm_(iter(ps), limit)
    assert got.shape == () and abs(got.item() - norm) <= 2 * E24 * norm
    for p, g in zip(ps, grads):
        if factor == 1.0:
            assert torch.equal(p.grad.cpu(), g)
        else:
            within(p.grad, g.double() * factor, 5 * E24 * g.double().abs() * factor, "grad")


@pytest.mark.gpu
def test_unaligned_views_channels_last_gradients_and_refused_layouts():
    buf = torch.randn(5000, generator=torch.Generator().manual_seed(7))
    flat_p, flat_g = torch.zeros(5000, device=DEV), buf.to(DEV)
    ps, at = [], 1
    for n in (1000, 37, 2049):                                 # at odd places of one buffer
        p = torch.nn.Parameter(flat_p[at:at + n])
        p.grad = flat_g[at:at + n]
        ps.append(p)
        at += n + 3
    cl = torch.nn.Parameter(torch.zeros(4, 8, 3, 3, device=DEV))
    cl.grad = torch.randn(4, 8, 3, 3, device=DEV).contiguous(memory_format=torch.channels_last)
    grads = [p.grad.cpu().clone() for p in ps + [cl]]
    norm, factor = factor_of(grads, 0.5)
    assert abs(train.clip_grad_norm_(ps + [cl], 0.5).item() - norm) <= 2 * E24 * norm
    for p, g in zip(ps + [cl], grads):
        within(p.grad, g.double() * factor, 5 * E24 * g.double().abs() * factor, "grad")
    outside = torch.ones(5000, dtype=torch.bool)
    for p in ps:
        outside[p.grad.storage_offset():p.grad.storage_offset() + p.numel()] = False
    assert torch.equal(flat_g.cpu()[outside], buf[outside])
    for bits in (32, 8):
        opt = train.AdamW(ps + [cl], lr=1e-2, weight_decay=0.0, state_bits=bits)
        before = flat_p.clone()
        cl_before = cl.detach().clone()
        opt.step()
        for p, old in zip(ps, [before[p.storage_offset():p.storage_offset() + p.numel()] for p in ps]):
            want, _, _, upd = reference_step(old.cpu(), p.grad.cpu(), torch.zeros(p.numel()), torch.zeros(p.numel()), 1, 1e-2, 0.9, 0.999, 1e-8, 0.0, 1.0)
            within(p, want, 4 * E24 * want.abs() + 32 * E24 * upd, "p")
        want, _, _, upd = reference_step(cl_before.cpu(), cl.grad.cpu(), torch.zeros(()), torch.zeros(()), 1, 1e-2, 0.9, 0.999, 1e-8, 0.0, 1.0)
        within(cl, want, 4 * E24 * want.abs() + 32 * E24 * upd, "channels-last gradient")
        assert torch.equal(flat_p[outside.to(DEV)], before[outside.to(DEV)])
    bad = torch.nn.Parameter(torch.zeros(4, 4, device=DEV))
    bad.grad = torch.ones(4, device=DEV).expand(4, 4)
    with pytest.raises(_lib.UResNetHipError, match="dense"):
        train.clip_grad_norm_([bad], 1.0)
    with pytest.raises(ValueError, match="twice"):
        train.clip_grad_norm_([cl, cl], 1.0)
    overlapping = [torch.nn.Parameter(torch.zeros(6, device=DEV)) for _ in range(2)]
    overlapping[0].grad, overlapping[1].grad = flat_g[:6], flat_g[5:11]
    with pytest.raises(ValueError, match="overlap"):
        train.clip_grad_norm_(overlapping, 1.0)
    turned = torch.nn.Parameter(torch.zeros(30, 7, device=DEV))
    turned.grad = torch.randn(7, 30, device=DEV).t()           # dense in another order
    g = turned.grad.cpu()
    norm, factor = factor_of([g], 0.5)
    assert abs(train.clip_grad_norm_([turned], 0.5).item() - norm) <= 2 * E24 * norm
    within(turned.grad, g.double() * factor, 5 * E24 * g.double().abs() * factor, "transposed gradient")
    bad.grad = torch.zeros(4, 4, device=DEV).to_sparse()
    for f in (lambda: train.clip_grad_norm_([bad], 1.0), lambda: train.AdamW([bad]).step()):
        with pytest.raises(_lib.UResNetHipError, match="dense"):
            f()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_groups_late_parameters_and_many_tensors(bits):
    """More tensors than one table launch takes, groups of their own constants under one norm, parameters without gradients,
    counts per parameter."""
    count, cut = 1500, 1300
    vals = tensors(8, [(17 + i % 400,) for i in range(count)])
    grads = tensors(9, [(17 + i % 400,) for i in range(count)], 0.5)
    ps = params_on_gpu(vals, [None if i % 3 == 1 else g for i, g in enumerate(grads)])
    opt = train.AdamW([{"params": ps[:cut], "lr": 1e-2, "state_bits": bits}, {"params": ps[cut:], "lr": 1e-3, "weight_decay": 0.0}],
                      weight_decay=0.1, max_grad_norm=0.75)
    opt.grad_scale = 0.5
    opt.step()
    live = [g for i, g in enumerate(grads) if i % 3 != 1]
    norm, factor = factor_of(live, 0.75, 0.5)
    assert abs(opt.grad_norm.item() - norm) <= 3 * E24 * norm
    for i, (p, v, g) in enumerate(zip(ps, vals, grads)):
        if i % 3 == 1:
            assert torch.equal(p.detach().cpu(), v) and p not in opt.state
            continue
        lr, wd = (1e-2, 0.1) if i < cut else (1e-3, 0.0)
        zero = torch.zeros(v.shape)
        want, _, _, upd = reference_step(v, g, zero, zero, 1, lr, 0.9, 0.999, 1e-8, wd, factor)
        within(p, want, 4 * E24 * want.abs() + 32 * E24 * upd, "p")
    ps[1].grad = grads[1].to(DEV)                              # joins at the second step with a count of its own
    opt.max_grad_norm, opt.grad_scale = None, 1.0
    opt.step()
    assert int(opt.state[ps[1]]["step"]) == 1 and int(opt.state[ps[0]]["step"]) == 2
    zero = torch.zeros(vals[1].shape)
    want, _, _, upd = reference_step(vals[1], grads[1], zero, zero, 1, 1e-2, 0.9, 0.999, 1e-8, 0.1, 1.0)
    within(ps[1], want, 4 * E24 * want.abs() + 32 * E24 * upd, "late p")


@pytest.mark.gpu
def test_matches_torch_over_twenty_steps():
    vals = tensors(11, SIZES[:-1])
    ours, ref = params_on_gpu(vals, [None] * len(vals)), [torch.nn.Parameter(v.double()) for v in vals]
    a = train.AdamW(ours, lr=1e-3, weight_decay=0.05)
    b = torch.optim.AdamW(ref, lr=1e-3, weight_decay=0.05)
    for t in range(20):
        for p, q, g in zip(ours, ref, tensors(100 + t, SIZES[:-1], 0.1)):
            p.grad, q.grad = g.to(DEV), g.double()
        a.step(), b.step()
    for p, q in zip(ours, ref):
        # twenty updates of at most a few lr, each with 32 roundings at most
        within(p, q.detach(), 20 * (3 * E24 * q.detach().abs() + 32 * E24 * 4e-3), "p")


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_replayed_graphs_make_the_eager_steps_bit_for_bit(bits):
    vals, grads = tensors(12, SIZES[:-1]), [tensors(20 + t, SIZES[:-1], 0.3) for t in range(6)]

    def build():
        ps = params_on_gpu(vals, [torch.zeros_like(v) for v in vals])
        return ps, train.AdamW(ps, lr=1e-2, state_bits=bits, max_grad_norm=0.5)

    def feed(ps, gs):
        for p, g in zip(ps, gs):
            p.grad.copy_(g.to(DEV))
    eager, opt_e = build()
    norms = []
    for gs in grads:
        feed(eager, gs)
        opt_e.step()
        norms.append(opt_e.grad_norm.item())
    ps, opt = build()
    with pytest.raises(RuntimeError, match="eager step"):
        g0 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g0, capture_error_mode="thread_local"):
            opt.step()
    torch.cuda.synchronize()
    feed(ps, grads[0])
    opt.step()
    captured = []
    for _ in range(2):                                         # two graphs of one optimiser, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            opt.step()
        captured.append((graph, opt.grad_norm))
    for t in range(1, 6):
        feed(ps, grads[t])
        if t == 3:
            opt.step()                                         # an eager step between the replays
            assert opt.grad_norm.item() == norms[t]
        else:
            captured[t % 2][0].replay()
            assert captured[t % 2][1].item() == norms[t]
    torch.cuda.synchronize()
    for p, q in zip(ps, eager):
        assert torch.equal(p, q)
    for k, buf in opt.state_buffers().items():
        assert torch.equal(buf.float(), opt_e.state_buffers()[k].float()), k
    assert int(opt.state[ps[0]]["step"]) == 6


@pytest.mark.gpu
def test_resumed_training_is_the_same_training():
    for bits in (32, 8):
        vals = tensors(13, SIZES[:-1])
        a = params_on_gpu(vals, [None] * len(vals))
        opt = train.AdamW(a, lr=1e-2, state_bits=bits)

        def steps(ps, o, lo, hi):
            for t in range(lo, hi):
                for p, g in zip(ps, tensors(30 + t, SIZES[:-1], 0.3)):
                    p.grad = g.to(DEV)
                o.step()
        steps(a, opt, 0, 2)
        sd = {k: v for k, v in opt.state_dict().items()}
        import io
        f = io.BytesIO()
        torch.save(sd, f)
        f.seek(0)
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        opt2 = train.AdamW(b, state_bits=bits)
        opt2.load_state_dict(torch.load(f, map_location="cpu", weights_only=True))
        steps(a, opt, 2, 4)
        steps(b, opt2, 2, 4)
        assert all(torch.equal(p, q) for p, q in zip(a, b)), bits


@pytest.mark.gpu
def test_a_closure_and_weight_images():
    p = torch.nn.Parameter(torch.ones(10, device=DEV))
    opt = train.AdamW([p], lr=0.1, weight_decay=0.0)
    epoch = ops._weights_epoch

    def closure():
        opt.zero_grad()
        loss = (p * p).sum()
        loss.backward()
        return loss
    assert opt.step(closure).item() == 10.0
    assert ops._weights_epoch == epoch + 1 and torch.allclose(p, torch.full_like(p, 0.9))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_from_before_the_step_is_refused_after_it(bits):
    """The step rewrites what the graph saved: as with any in-place change, autograd has to see it."""
    from uresnet_amd import nn as hnn
    gn = hnn.GroupNorm(4, 8).to(DEV)
    other = torch.nn.Parameter(torch.ones(5, device=DEV))                  # without a gradient: not written
    opt = train.AdamW(list(gn.parameters()) + [other], lr=0.5, state_bits=bits)
    x = torch.randn(2, 8, 4, 4, device=DEV).contiguous(memory_format=torch.channels_last).requires_grad_()
    y = ops.gn_act(x, gn)
    (y ** 2).sum().backward(retain_graph=True)
    versions = [t._version for t in (gn.weight, gn.bias, other)]
    opt.step()
    assert [t._version for t in (gn.weight, gn.bias, other)] == [versions[0] + 1, versions[1] + 1, versions[2]]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (y ** 2).sum().backward()
    opt.zero_grad()
    (ops.gn_act(x, gn) ** 2).sum().backward()                              # a new graph is what such a loop needs
    opt.step()
    with torch.inference_mode():
        p = torch.nn.Parameter(torch.ones(3, device=DEV))                  # has no version
        p.grad = torch.ones(3, device=DEV)
        train.AdamW([p], lr=0.1, state_bits=bits).step()
        assert (p < 1).all()


@pytest.mark.gpu
def test_clipped_gradients_count_as_written():
    p = torch.nn.Parameter(torch.zeros(7, device=DEV))
    p.grad = torch.full((7,), 3.0, device=DEV)
    w = torch.ones(7, device=DEV, requires_grad=True)
    y = (p.grad * w).sum()                                                 # saves the gradient
    train.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
def test_a_root_above_zero_keeps_a_code_above_zero():
    """b2 = 0: the root is |g|.  Twelve decades inside every block: what is far below the lowest code (2^-9 of the scale) gets
    that code, only exact zeros get 0."""
    gen = torch.Generator().manual_seed(50)
    g = 10 ** (-12 * torch.rand(16, 256, generator=gen)) * torch.randn(16, 256, generator=gen).sign()
    g[:, 7], g[:, 0] = 0.0, 1.0
    p = torch.nn.Parameter(torch.zeros(g.numel(), device=DEV))
    opt = train.AdamW([p], lr=0.0, betas=(0.0, 0.0), state_bits=8)
    p.grad = g.flatten().to(DEV)
    for _ in range(3):
        opt.step()
        codes = opt.state_buffers()["exp_avg_sq_root"].float().cpu().view(16, 256)
        assert (codes[g == 0] == 0).all() and (codes[g != 0] >= 2.0 ** -9).all()
        below = (g != 0) & (g.abs() * 448 < 2.0 ** -9)
        assert below.sum() > 1000 and (codes[below] == 2.0 ** -9).all()


@pytest.mark.gpu
def test_eight_bit_steps_with_six_decades_inside_a_block_stay_bounded():
    """(1 - b1) / sqrt(1 - b2) = 3.2 lr bounds a step in 32 bits; a code more or less among the lowest ones is a factor of two
    for m and for the root: four times that."""
    gen = torch.Generator(device=DEV).manual_seed(51)
    n = 256 * 64
    size = 10 ** (-6 * torch.rand(n, generator=gen, device=DEV))
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = train.AdamW([p], lr=1.0, weight_decay=0.0, state_bits=8)
    largest = torch.zeros((), device=DEV)
    for _ in range(300):
        p.grad = size * torch.randn(n, generator=gen, device=DEV)
        before = p.detach().clone()
        opt.step()
        largest = torch.maximum(largest, (p.detach() - before).abs().max())
    assert largest.item() < 4 * 3.2


@pytest.mark.gpu
def test_weights_without_a_gradient_come_to_rest_in_eight_bits():
    """Half of every block stops getting gradients.  Its first moment falls by at least one code per step while the scale does
    not fall (a tenth is more than half a step between normal codes, and lower ones are rounded down): the 127 codes are
    passed in at most 127 steps, then the weights stay where they are."""
    gen = torch.Generator(device=DEV).manual_seed(52)
    n, lr = 256 * 16, 1e-2
    live = (torch.arange(n, device=DEV) % 2).float()
    g = torch.randn(n, generator=gen, device=DEV)
    g[1::256] = 4.0                                            # the largest of its block, and constant: the scale only grows
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = train.AdamW([p], lr=lr, betas=(0.9, 0.95), weight_decay=0.0, state_bits=8)
    for t in range(20 + 127):
        p.grad = (g if t < 20 else g * live).clamp(-4, 4)
        opt.step()
    dead = live == 0
    assert not opt.state_buffers()["exp_avg"].float()[dead].any() and opt.state_buffers()["exp_avg"].float()[~dead].any()
    rest = p.detach().clone()
    for _ in range(800):                                       # the roots fall to their lowest code
        opt.step()
    assert torch.equal(p.detach()[dead], rest[dead]) and (opt.state_buffers()["exp_avg_sq_root"].float()[dead] == 2.0 ** -9).all()


@pytest.mark.gpu
def test_eight_bit_moments_over_some_hundred_steps():
    """Against the recurrences in 64 bits.  The root's rounding adds a variance of f (1 - f) s^2 per step, f the fraction of the
    code step s by which it moves: to first order |change| s.  The change is (1 - b2) / 2 |g^2 / v - 1|, 0.97 (1 - b2) / 2 on
    average for Gaussian gradients, s is 0.090 on average (1/8 of the power of two below), and what is there decays by b2 per
    step: 0.97 * 0.090 / 4 = 0.0218 remains, 14.8 % rms.  m's nearest rounding adds s^2 / 12 per step, kept for 1 / (1 - b1^2):
    5.5 % rms, together 15.8 % for the update.  A third more is allowed for the higher orders."""
    gen = torch.Generator(device=DEV).manual_seed(53)
    n, steps = 256 * 256, 400
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = train.AdamW([p], lr=1.0, weight_decay=0.0, state_bits=8)
    m, v = torch.zeros(2, n, dtype=torch.float64, device=DEV)
    for t in range(1, steps + 1):
        g = 1e-3 * torch.randn(n, generator=gen, device=DEV)
        m, v = 0.9 * m + 0.1 * g.double(), 0.999 * v + 0.001 * g.double() ** 2
        before = p.detach().clone()
        p.grad = g
        opt.step()
    want = m / (1 - 0.9 ** steps) / ((v / (1 - 0.999 ** steps)).sqrt() + 1e-8)
    off = (before - p.detach()).double() - want
    assert (off.square().mean() / want.square().mean()).sqrt().item() < 0.158 * 4 / 3
    st = opt.state_buffers()
    root = dequantise(st["exp_avg_sq_root"].float().cpu(), st["exp_avg_sq_root_scale"].cpu()) / v.sqrt().cpu() - 1
    assert root.square().mean().sqrt().item() < 0.148 * 4 / 3
    # The rounding keeps r on average and so adds its variance to v = r^2: 0.97 * 0.090 * (1 - b2) / 2 of v per step, which decays
    # by 1 - b2 of itself: 0.0437 = 2 * 0.148^2 above.  The same third more on a root, its square here.
    assert 0 < ((root + 1) ** 2).mean().item() - 1 < 2 * (0.148 * 4 / 3) ** 2


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_nan_norm_leaves_the_state_between_the_tensors_zero(bits):
    sizes = [(300,), (5,), (2049,)]
    ps = params_on_gpu([torch.ones(s) for s in sizes], tensors(54, sizes))
    ps[1].grad[2] = float("nan")
    opt = train.AdamW(ps, state_bits=bits, max_grad_norm=1.0)
    for _ in range(2):
        opt.step()
    assert opt.grad_norm.isnan() and all(p.isnan().all() for p in ps)
    for k, buf in opt.state_buffers().items():
        if not k.endswith("scale"):
            buf = buf.float().cpu()
            for lo, hi in ((300, 512), (512 + 5, 768), (768 + 2049, buf.numel())):
                assert (buf[lo:hi] == 0).all(), (k, lo)


@pytest.mark.gpu
def test_a_norm_beyond_fp32_is_not_finite():
    """Finite gradients whose norm is no fp32 number: infinity, as in torch (and gradients scaled to zero), or an error."""
    p = torch.nn.Parameter(torch.zeros(3, device=DEV))
    p.grad = torch.full((3,), 3e38, device=DEV)
    with pytest.raises(RuntimeError, match="not finite"):
        train.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert (p.grad == 3e38).all()
    assert train.clip_grad_norm_([p], 1.0).isinf() and (p.grad == 0).all()
    p.grad = torch.full((3,), 1.9e38, device=DEV)              # 3.3e38: still one
    norm = train.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert abs(norm.item() - 1.9e38 * 3 ** 0.5) <= 4 * E24 * norm.item()


@pytest.mark.gpu
def test_parameters_that_come_to_share_memory_are_refused():
    """Tied by hand after the first step: both would be written by one launch."""
    a, b, c = (torch.nn.Parameter(torch.ones(40, device=DEV)) for _ in range(3))
    opt = train.AdamW([a, b, c], lr=0.1)
    for p in (a, b, c):
        p.grad = torch.ones(40, device=DEV)
    opt.step()
    whole = torch.ones(60, device=DEV)
    for first, second in ((whole[:40], whole[:40]), (whole[20:], whole[:40])):
        a.data, c.data = first, second
        with pytest.raises(_lib.UResNetHipError, match="share memory"):
            opt.step()
        assert (whole == 1).all() and int(opt.state[a]["step"]) == 1
    c.grad = None                                              # not written: no race
    opt.step()
    assert (whole[20:] < 1).all() and (whole[:20] == 1).all()
    a.data, c.data, c.grad = whole[:30], whole[30:], torch.ones(30, device=DEV)
    with pytest.raises(_lib.UResNetHipError, match="size"):
        opt.step()


@pytest.mark.gpu
def test_running_out_of_memory_raises_as_in_torch():
    """What a program catches to go on with smaller batches; afterwards the calls work."""
    from uresnet_amd import nn as hnn
    gn = hnn.GroupNorm(4, 64).to(DEV)
    x = torch.randn(8, 64, 256, 256, device=DEV).contiguous(memory_format=torch.channels_last)          # 134 MB
    p = torch.nn.Parameter(torch.zeros(4096, 4096, device=DEV))
    p.grad = torch.ones(4096, 8192, device=DEV)[:, ::2]                                                # has to be copied: 67 MB
    opt = train.AdamW([p], lr=0.1, weight_decay=0.0)
    opt.state_buffers()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    try:
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (8 << 20)) / total)
        for call in (lambda: gn(x), opt.step):
            with pytest.raises(torch.OutOfMemoryError):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    version = p._version
    assert torch.isfinite(gn(x)).all()
    opt.step()
    assert (p < 0).all() and p._version == version + 1 and int(opt.state[p]["step"]) == 1
