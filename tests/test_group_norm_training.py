"""The networks with GroupNorm (nn.to_group_norm) trained by AdamW with clipping: the path a user takes with few images per
GPU.  Logits and gradients against the CPU oracle with its BatchNorm2d replaced the same way, at the tolerances of the
BatchNorm networks' tests; a captured step against the eager one, bit for bit."""
import pytest
import torch

from conftest import rel_l2

from uresnet_amd import nn as hnn, ops, train

DEV = "cuda:0"
pytestmark = pytest.mark.gpu


def oracle_group_norm(module, num_groups):
    for name, child in list(module.named_children()):
        if isinstance(child, torch.nn.BatchNorm2d):
            c = child.num_features
            groups = max(g for g in range(1, min(num_groups, c) + 1) if c % g == 0)
            gn = torch.nn.GroupNorm(groups, c, eps=child.eps)
            gn.weight, gn.bias = child.weight, child.bias
            setattr(module, name, gn)
        else:
            oracle_group_norm(child, num_groups)
    return module


def inputs(n=2, h=32, w=64):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(n, 3, h, w, generator=g)
    y = torch.randint(0, 19, (n, h, w), generator=g)
    y[torch.rand(y.shape, generator=g) < 0.1] = 255
    return x, y


def pair(oracle, cls, dtype, seed=0):
    from uresnet_amd.modules import U_ResNet as M
    torch.manual_seed(seed)
    ref = getattr(oracle, cls)(19, 3, 8)
    model = getattr(M, cls)(19, 3, 8).set_compute_dtype(dtype)
    model.load_state_dict(ref.state_dict())
    return oracle_group_norm(ref, 8).train(), hnn.to_group_norm(model, 8).to(DEV).train()


@pytest.mark.parametrize("cls", ["UResNetNewEUCB", "UResNet", "UResNetNoEUCB"])
def test_fp32_network_matches_the_oracle(oracle, cls):
    ref, model = pair(oracle, cls, torch.float32)
    x, y = inputs()
    out = model(x.to(DEV))
    loss = train.compute_loss(out, y.to(DEV))
    loss.backward()
    ro = ref(x)
    rl = oracle.compute_loss(ro, y)
    rl.backward()
    assert rel_l2(ops.to_nchw_raw(out.detach(), torch.float32).cpu(), ro.detach()) < 2e-4
    assert abs(loss.item() - rl.item()) < 1e-4
    grads = dict(ref.named_parameters())
    for k, p in model.named_parameters():
        want = grads[k].grad
        # gradients that cancel analytically (a bias before a group norm with one channel per group) have no relative error
        if want.norm() > 1e-5:
            assert rel_l2(p.grad.cpu(), want) < 5e-3, k
    model.eval(), ref.eval()
    with torch.no_grad():
        assert rel_l2(ops.to_nchw_raw(model(x.to(DEV)), torch.float32).cpu(), ref(x)) < 2e-4


@pytest.mark.parametrize("module, cls, oracle_cls, args, kwargs, shape", [
    ("U_ResNet", "UNet", "UNet", (19, 3, 8), {}, (2, 3, 32, 64)),
    ("U_ResNet", "UResNetNoResBlock", "UResNetNoResBlock", (19, 3, 8), {}, (2, 3, 32, 64)),
    ("U_ResNet_CIFAR", "UResNet4_No_SU", "UResNet4_No_SU", (10, 3), {"scale": 3}, (2, 3, 32, 32)),
    ("U_ResNet_CIFAR", "UResNet3_No_EUCB", "UResNet3_No_EUCB", (10, 3), {"scale": 3}, (2, 3, 32, 32)),
    ("U_ResNet_CIFAR", "UResNet3_No_UBlock", "UResNet3_No_UBlock", (10, 3), {"scale": 3}, (2, 3, 32, 32)),
    ("U_ResNet_CIFAR", "E_ResNet", "E_ResNet", (), {}, (2, 3, 32, 32)),
    ("U_ResNet_MiniImageNet", "U_ResNet", "MiniU_ResNet", (100, 3), {}, (2, 3, 224, 224))])       # the size the class is made for
def test_other_networks_match_the_oracle(oracle, module, cls, oracle_cls, args, kwargs, shape):
    """Logits and gradient norms, at the tolerances of the same classes with BatchNorm."""
    import uresnet_amd
    torch.manual_seed(0)
    ref = getattr(oracle, oracle_cls)(*args, **kwargs)
    model = getattr(getattr(uresnet_amd.modules, module), cls)(*args, **kwargs).set_compute_dtype(torch.float32)
    model.load_state_dict(ref.state_dict())
    oracle_group_norm(ref, 8).train()
    hnn.to_group_norm(model, 8).to(DEV).train()
    g = torch.Generator().manual_seed(2)
    x = torch.randn(shape, generator=g)
    out, ro = model(x.to(DEV)), ref(x)
    got = out if out.dim() == 2 else ops.to_nchw_raw(out, torch.float32)
    dy = torch.randn(ro.shape, generator=g)
    ro.backward(dy)
    out.backward(dy.to(DEV))
    assert rel_l2(got.detach().float().cpu(), ro.detach()) < 2e-4
    want = dict(ref.named_parameters())
    assert {k for k, p in model.named_parameters() if p.grad is None} == {k for k, p in want.items() if p.grad is None}
    norms = [(p.grad.double().norm().item(), want[k].grad.double().norm().item()) for k, p in model.named_parameters() if p.grad is not None]
    floor = 1e-5 * max(n for _, n in norms)
    errs = sorted(abs(a - b) / b for a, b in norms if b > floor)
    assert errs[len(errs) // 2] < 1e-4 and errs[-1] < 3e-2, (errs[len(errs) // 2], errs[-1])


def test_bf16_network_tracks_fp32(oracle):
    _, a = pair(oracle, "UResNetNewEUCB", torch.float32)
    _, b = pair(oracle, "UResNetNewEUCB", torch.bfloat16)
    x, _ = inputs()
    with torch.no_grad():
        assert rel_l2(b(x.to(DEV)).float().cpu(), a(x.to(DEV)).cpu()) < 6e-2


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_steps_are_the_eager_ones(oracle, bits):
    """Five steps of the network with its matrices in `bits`-bit states, norms and biases in 32, one norm over both groups."""
    def build():
        _, model = pair(oracle, "UResNetNewEUCB", torch.bfloat16)
        wide = [p for p in model.parameters() if p.dim() > 1]
        thin = [p for p in model.parameters() if p.dim() <= 1]
        return model, train.AdamW([{"params": wide, "state_bits": bits}, {"params": thin, "weight_decay": 0.0}], lr=1e-3,
                                  max_grad_norm=1.0)
    x, y = (t.to(DEV) for t in inputs())
    model, opt = build()
    eager = []
    for k in range(5):
        loss, _ = train.seg_train_step(model, opt, x + 0.01 * k, y)
        eager.append((loss.item(), opt.grad_norm.item()))
    assert all(torch.isfinite(torch.tensor(v)).all() for v in eager) and len({v[0] for v in eager}) == 5
    other, opt2 = build()
    del loss
    step = train.GraphedStep(train.seg_train_step, other, opt2, x, y, warmup=1)      # its warm-up step is the first eager one
    for k in range(1, 5):
        loss, _ = step(x + 0.01 * k, y)
        assert (loss.item(), opt2.grad_norm.item()) == eager[k], k
    torch.cuda.synchronize()
    for (n, p), q in zip(model.named_parameters(), other.parameters()):
        assert torch.equal(p, q), n


def test_classification_network_with_every_activation_fused():
    """The EUCB* stage with a GroupNorm and each of act_layer's activations: the fused pass against the two modules."""
    from uresnet_amd.modules._blocks import DoubleConv, EUCB2, act_layer
    g = torch.Generator().manual_seed(3)
    for name in ("relu", "relu6", "leakyrelu", "gelu", "hswish", "prelu"):
        torch.manual_seed(5)
        blk = hnn.to_group_norm(EUCB2(16, 8, activation=name), 4).to(DEV)
        x = torch.randn(2, 16, 6, 7, generator=g).to(DEV)
        fused = blk(x)
        handle = blk.up_dwc1[1].register_forward_hook(lambda m, i, o: None)          # layer by layer
        plain = blk(x)
        handle.remove()
        assert rel_l2(fused.detach().cpu(), plain.detach().cpu()) < 1e-5, name
    assert act_layer("gelu") is not None and DoubleConv is not None


def test_clipping_beside_the_other_optimisers(oracle):
    """clip_grad_norm_ between backward and Adam's step: the same parameters as torch's clipping gives."""
    grads = None
    results = []
    for clip in (train.clip_grad_norm_, torch.nn.utils.clip_grad_norm_):
        _, model = pair(oracle, "UResNetNewEUCB", torch.float32)
        opt = train.Adam(model.parameters(), lr=1e-3)
        x, y = (t.to(DEV) for t in inputs())
        train.compute_loss(model(x), y).backward()
        if grads is None:
            grads = [p.grad.clone() for p in model.parameters()]
        else:
            for p, g in zip(model.parameters(), grads):
                p.grad.copy_(g)
        norm = clip(model.parameters(), 0.5)
        clipped = [p.grad.clone() for p in model.parameters()]
        opt.step()
        results.append((norm.item(), clipped))
    # torch sums squares in fp32 per tensor: relative error below sqrt(elements) * 2^-24
    assert abs(results[0][0] - results[1][0]) < 1e-4 * results[1][0] and results[0][0] > 0.5
    for a, b in zip(results[0][1], results[1][1]):
        assert torch.allclose(a, b, rtol=2e-4, atol=0)


SCRIPT = r'''
import os, sys, torch
import torch.distributed as dist
sys.path.insert(0, os.environ["UR_ROOT"])
import uresnet_amd
from uresnet_amd import nn as hnn, train
from uresnet_amd.modules.U_ResNet import UResNetNewEUCB

torch.cuda.set_device(0)
dev = torch.device("cuda", 0)
dist.init_process_group("nccl", init_method="tcp://127.0.0.1:29543", rank=0, world_size=1, device_id=dev)
g = torch.Generator().manual_seed(7)
x = torch.randn(2, 3, 64, 96, generator=g).to(dev)
y = torch.randint(0, 19, (2, 64, 96), generator=g).to(dev)
for bits in (32, 8):
    runs = []
    for wrapped in (False, True):
        torch.manual_seed(0)
        m = hnn.to_group_norm(UResNetNewEUCB(19, 3, 8).set_compute_dtype(torch.float32), 8).to(dev).train()
        opt = train.AdamW(m.parameters(), lr=1e-3, state_bits=bits, max_grad_norm=1.0)
        ddp = uresnet_amd.ddp.DataParallel(m, bucket_mb=0.05) if wrapped else None
        seen = []
        for _ in range(3):
            if ddp is None:
                loss, _ = train.seg_train_step(m, opt, x, y)
            else:
                loss, _ = train.seg_train_step(m, opt, x, y, count_hook=ddp.count_hook, grad_hook=ddp.finish)
            seen += [loss.item(), opt.grad_norm.item()]
        runs.append(seen)
        if wrapped:
            assert {p.grad.data_ptr() % 16 for p in m.parameters() if p.grad is not None} == {0}
    # the loss is divided by an all-reduced count: equal up to rounding, which the steps then carry on
    assert all(abs(a - b) <= 1e-3 * abs(a) for a, b in zip(*runs)), runs
dist.destroy_process_group()
print("DDP_OK")
'''


def test_one_rank_data_parallel_step_with_group_norm_and_adamw():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, UR_ROOT=root, HSA_ENABLE_IPC_MODE_LEGACY="0")
    r = subprocess.run([sys.executable, "-c", SCRIPT], env=env, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "DDP_OK" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
