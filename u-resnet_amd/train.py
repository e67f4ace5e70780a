"""Loss, mask and optimiser-step counterparts of the reference's training loops, on HIP kernels.

  compute_loss      Segmentation/Cityscapes/train_UResNetAblitionStudy.py:62-68
  AdamW, clipping   no counterpart (the reference trains with Adam and without clipping)
  Adam / SGD        optim.Adam(lr=1e-4) (same file :203), optim.SGD(lr=0.01) (Classification/CNN-CIFAR10.py:130)
  train steps       train_UResNetAblitionStudy.py:115-122, CNN-CIFAR10.py:145-149, Ice-Seg/TrainingCode.py:107-115
  masks             preds.argmax(1) (train_UResNetAblitionStudy.py:73), sigmoid(outputs) > 0.5 (TrainingCode.py:132)
  metrics           calculate_metrics / validate (train_UResNetAblitionStudy.py:70-100, 128-164)
  checkpoints       the dict written at train_UResNetAblitionStudy.py:244-252 (save_checkpoint / load_checkpoint)
"""
import array
import itertools
import operator

import torch

from . import _lib, ops


def compute_loss(outputs, targets, count_hook=None):
    """CrossEntropyLoss(ignore_index=255)(outputs, targets.long()): mean NLL over the valid pixels."""
    if isinstance(outputs, list):
        outputs = outputs[0]
    if targets.dtype != torch.int64:
        targets = targets.long()
    return ops.cross_entropy(outputs, targets, ignore_index=255, count_hook=count_hook)


def cross_entropy_loss(outputs, targets):
    """nn.CrossEntropyLoss() on [B, classes] logits (CNN-CIFAR10.py:129)."""
    return ops.cross_entropy(outputs, targets, ignore_index=-100)


def bce_with_logits_loss(outputs, masks):
    """nn.BCEWithLogitsLoss() (Ice-Seg/TrainingCode.py:97)."""
    return ops.bce_with_logits(outputs, masks)


def argmax_mask(outputs):
    return ops.argmax_channels(outputs)


def sigmoid_mask(outputs):
    return ops.sigmoid_mask(outputs)


_METRIC_KEYS = ('precision', 'recall', 'accuracy', 'f1', 'iou')


def _metrics_dict(acc):
    v = acc.cpu().tolist()                       # the only host synchronisation
    n = v[5] if v[5] > 0 else 1.0
    m = {k: v[i] / n for i, k in enumerate(_METRIC_KEYS)}
    m['dice'] = m['f1']                          # the reference reports the F1 score again as `dice`
    return m, v[6] / n


def calculate_metrics(preds, targets, num_classes):
    """train_UResNetAblitionStudy.py:70-100: macro precision / recall / F1 / IoU and accuracy of argmax(preds) on the
    pixels whose target is not 255 -- from a confusion matrix built on the GPU instead of sklearn on flattened copies."""
    if isinstance(preds, list):
        preds = preds[0]
    cm = ops.confusion_matrix(preds, targets, num_classes, ignore_index=255)
    acc = torch.zeros(7, dtype=torch.float64, device=cm.device)
    ops.seg_metrics_accumulate(cm, acc)
    return _metrics_dict(acc)[0]


def validate(model, data_loader, device, num_classes):
    """train_UResNetAblitionStudy.py:128-164: eval-mode forward, mean loss and mean per-batch metrics.  Loss and metrics
    accumulate on the device; the host reads them once after the last batch."""
    model.eval()
    acc = None
    with torch.no_grad():
        for images, targets in data_loader:
            images, targets = images.to(device), targets.to(device)
            outputs = model(images)
            loss = compute_loss(outputs, targets)
            if isinstance(outputs, list):
                outputs = outputs[0]
            if acc is None:
                acc = torch.zeros(7, dtype=torch.float64, device=outputs.device)
                cm = torch.zeros((num_classes, num_classes), dtype=torch.int64, device=outputs.device)
            cm.zero_()
            ops.confusion_matrix(outputs, targets, num_classes, ignore_index=255, out=cm)
            ops.seg_metrics_accumulate(cm, acc, loss.detach().float().reshape(1))
    if acc is None:
        raise ZeroDivisionError("validate: empty data loader")
    metrics, mean_loss = _metrics_dict(acc)
    return mean_loss, metrics


def save_checkpoint(path, model, optimizer, epoch, val_loss, metrics):
    """The reference's best-model file (train_UResNetAblitionStudy.py:244-252): same keys, `module.`-free parameter
    names, CPU tensors, torch.optim-compatible optimiser state."""
    inner = getattr(model, 'module', model)
    torch.save({'epoch': epoch,
                'model_state_dict': {k: v.detach().cpu() for k, v in inner.state_dict().items()},
                'optimizer_state_dict': optimizer.state_dict(),
                'val_loss': val_loss,
                'metrics': metrics}, path)


def load_checkpoint(path, model, optimizer=None, map_location='cpu'):
    """Load a checkpoint written by the reference's loop or by save_checkpoint (or a bare state_dict).  The file is read
    with weights_only=True (tensors and plain containers only, nothing in it is executed); a `module.` prefix left by
    nn.DataParallel is stripped.  Returns the checkpoint dict without the two state dicts."""
    ckpt = torch.load(path, map_location=map_location, weights_only=True)
    state = ckpt.get('model_state_dict', ckpt) if isinstance(ckpt, dict) else ckpt
    state = {(k[7:] if k.startswith('module.') else k): v for k, v in state.items()}
    getattr(model, 'module', model).load_state_dict(state, strict=True)
    if optimizer is not None and isinstance(ckpt, dict) and 'optimizer_state_dict' in ckpt:
        optimizer.load_state_dict(ckpt['optimizer_state_dict'])
    return {k: v for k, v in ckpt.items() if k not in ('model_state_dict', 'optimizer_state_dict')} if 'model_state_dict' in ckpt else {}


class _MultiTensorOptimizer(torch.optim.Optimizer):
    """One kernel launch per step over every parameter that has a gradient (fp32 master weights)."""
    _slots = ()

    def __init__(self, params, defaults):
        super().__init__(params, defaults)
        self._table_key = None
        self._table = None
        self._pin = None
        self._ring = None
        self._ring_next = 0
        self.grad_scale = 1.0

    def _gather(self, group):
        ps = [p for p in group['params'] if p.grad is not None]
        for p in ps:
            if p.dtype != torch.float32 or not p.is_cuda or not p.is_contiguous():
                raise _lib.UResNetHipError("optimizer: parameters must be contiguous fp32 GPU tensors")
            if p.grad.dtype != torch.float32:
                raise _lib.UResNetHipError("optimizer: gradients must be fp32")
            if not p.grad.is_contiguous():
                p.grad = p.grad.contiguous()
        return ps

    def _pointer_table(self, rows, sizes, device):
        key = tuple(v for r in rows for v in r)
        if key != self._table_key:
            flat, sz = torch.tensor(key, dtype=torch.int64), torch.tensor(sizes, dtype=torch.int64)
            fits = self._pin is not None and self._pin[0].numel() == len(key) and self._pin[1].numel() == len(sizes)
            if torch.cuda.is_current_stream_capturing():
                # Under HIP graph capture the upload must be an asynchronous copy from pinned memory (it becomes a graph
                # node that re-reads the staging buffer at every replay); the buffer was allocated by an eager step.
                if not fits:
                    raise RuntimeError("optimizer: run at least one eager step with the same parameters before capturing")
                self._pin[0].copy_(flat)
                self._pin[1].copy_(sz)
                self._table = (self._pin[0].to(device, non_blocking=True), self._pin[1].to(device, non_blocking=True), max(sizes))
            else:
                # Eager: gradient tensors are new allocations every step, so the table changes every step.  A blocking
                # upload would drain the GPU once per step (the host waits for the whole backward pass, then the next
                # forward starts from an empty queue).  Instead: asynchronous copies from a ring of pinned staging
                # buffers; a slot is rewritten only after the event behind its last copy has completed (four steps
                # later, so the wait never blocks in practice).
                if not fits:
                    self._pin = (torch.empty(len(key), dtype=torch.int64).pin_memory(),
                                 torch.empty(len(sizes), dtype=torch.int64).pin_memory())
                    self._ring = [(torch.empty(len(key), dtype=torch.int64).pin_memory(),
                                   torch.empty(len(sizes), dtype=torch.int64).pin_memory(), torch.cuda.Event())
                                  for _ in range(4)]
                    self._ring_next = 0
                pf, ps_, ev = self._ring[self._ring_next]
                self._ring_next = (self._ring_next + 1) % len(self._ring)
                ev.synchronize()
                pf.copy_(flat)
                ps_.copy_(sz)
                self._table = (pf.to(device, non_blocking=True), ps_.to(device, non_blocking=True), max(sizes))
                ev.record(torch.cuda.current_stream(device))
            self._table_key = key
        return self._table


class Adam(_MultiTensorOptimizer):
    """torch.optim.Adam semantics (no amsgrad): exp_avg / exp_avg_sq state, bias correction, eps outside sqrt.

    Every parameter's step count lives in device memory (one int32 slot of a per-group pool; `state[p]['step']` is a
    0-dim view of it) and is advanced by the kernel, so a step carries no host-side value: a captured HIP graph
    replays it correctly, and parameters whose state began later are corrected with their own count, as
    torch.optim.Adam does.  state_dict() / load_state_dict() use torch.optim.Adam's layout (`step` as a float32 CPU
    scalar tensor), so optimiser states move between the two in either direction."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._step_pools = {}          # (group index, device) -> int32 pool of step counters
        self._pool_index = {}          # (group index, device) -> {parameter: slot}

    def _step_slot(self, gi, p):
        """0-dim int32 device view: the step counter of parameter p of group gi.  One pool per (group, device); a pool
        grows by copy when the group has gained parameters, so counters handed out earlier keep their values (their
        old views stay valid for the kernel table, which is rebuilt from `state[p]['step']` at every step)."""
        key = (gi, p.device)
        pool = self._step_pools.get(key)
        index = self._pool_index.setdefault(key, {})
        if p not in index:
            index[p] = len(index)
        need = index[p] + 1
        if pool is None or pool.numel() < need:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("Adam: run at least one eager step before capturing")
            size = max(need, len(self.param_groups[gi]['params']))
            grown = torch.zeros(size, dtype=torch.int32, device=p.device)
            if pool is not None:
                grown[:pool.numel()].copy_(pool)
                for q, i in index.items():                  # counters already handed out move with their values
                    st = self.state.get(q)
                    if st and 'step' in st and i < pool.numel():
                        st['step'] = grown[i]
            pool = self._step_pools[key] = grown
        return pool[index[p]]

    def state_dict(self):
        sd = super().state_dict()
        # one device read per pool instead of one per parameter
        host = {key: pool.cpu() for key, pool in self._step_pools.items()}
        slot = {q: (key, i) for key, index in self._pool_index.items() for q, i in index.items()}
        order = [q for group in self.param_groups for q in group['params']]      # torch numbers the parameters this way

        def step_of(k, v):
            q = order[k]
            if q in slot and slot[q][0] in host:
                return float(host[slot[q][0]][slot[q][1]])
            return float(v['step'])
        sd['state'] = {k: ({**v, 'step': torch.tensor(step_of(k, v))} if 'step' in v else v) for k, v in sd['state'].items()}
        for g in sd['param_groups']:                 # torch.optim.Adam's remaining group keys, at their defaults
            for k, v in (('amsgrad', False), ('maximize', False), ('foreach', None), ('capturable', False),
                         ('differentiable', False), ('fused', None), ('decoupled_weight_decay', False)):
                g.setdefault(k, v)
        return sd

    def load_state_dict(self, state_dict):
        for g in state_dict['param_groups']:
            if g.get('amsgrad') or g.get('maximize'):
                raise NotImplementedError("Adam: amsgrad / maximize states cannot be loaded")
        keep = set(self.defaults) | {'params'}
        slim = {'state': state_dict['state'],
                'param_groups': [{k: v for k, v in g.items() if k in keep} for g in state_dict['param_groups']]}
        super().load_state_dict(slim)
        self._step_pools, self._pool_index = {}, {}
        for gi, group in enumerate(self.param_groups):
            for p in group['params']:
                st = self.state.get(p)
                if st and 'step' in st:
                    count = int(round(float(st['step'])))
                    st['step'] = self._step_slot(gi, p)
                    st['step'].fill_(count)
        self._table_key = None

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        for gi, group in enumerate(self.param_groups):
            ps = self._gather(group)
            if not ps:
                continue
            rows, sizes = [], []
            for p in ps:                                  # states first: a new counter may move the whole pool
                st = self.state[p]
                if not st:
                    st['step'] = self._step_slot(gi, p)
                    st['exp_avg'] = torch.zeros_like(p)
                    st['exp_avg_sq'] = torch.zeros_like(p)
            for p in ps:
                st = self.state[p]
                rows.append((p.data_ptr(), p.grad.data_ptr(), st['exp_avg'].data_ptr(), st['exp_avg_sq'].data_ptr(),
                             st['step'].data_ptr()))
                sizes.append(p.numel())
            table, sz, mx = self._pointer_table(rows, sizes, ps[0].device)
            b1, b2 = group['betas']
            _lib.call("ur_adam_multi_dev", table.data_ptr(), sz.data_ptr(), len(ps), mx, group['lr'], b1, b2, group['eps'],
                      group['weight_decay'], self.grad_scale, ops._stream())
        ops.bump_weights_epoch()
        return loss


class SGD(_MultiTensorOptimizer):
    """torch.optim.SGD semantics without momentum (the reference uses plain SGD)."""

    def __init__(self, params, lr=1e-3, momentum=0, weight_decay=0.0):
        if momentum != 0:
            raise NotImplementedError("SGD momentum is not implemented (the reference trains with momentum=0)")
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay))

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        for group in self.param_groups:
            ps = self._gather(group)
            if not ps:
                continue
            rows = [(p.data_ptr(), p.grad.data_ptr()) for p in ps]
            sizes = [p.numel() for p in ps]
            table, sz, mx = self._pointer_table(rows, sizes, ps[0].device)
            _lib.call("ur_sgd_multi", table.data_ptr(), sz.data_ptr(), len(ps), mx, group['lr'], group['weight_decay'],
                      self.grad_scale, ops._stream())
        ops.bump_weights_epoch()
        return loss


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ for fp32 gradients on one GPU: scales them in place by min(1, max_norm / (norm + 1e-6))
    and returns their norm before that as a 0-dim device tensor.  No host synchronisation (except with error_if_nonfinite,
    which raises before anything is scaled), no staging buffers: it can be captured in a graph.  A norm within the limit
    leaves the gradients untouched.  Only the 2-norm; gradients that overlap are refused."""
    if norm_type != 2:
        raise NotImplementedError("clip_grad_norm_: only norm_type=2 is implemented (got %r)" % (norm_type,))
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("clip_grad_norm_: max_norm must not be negative (got %r)" % (max_norm,))
    norm = _lib.host().clip_grads([parameters] if torch.is_tensor(parameters) else list(parameters), max_norm, bool(error_if_nonfinite))
    return torch.tensor(0.0) if norm is None else norm


class _MomentPool:
    """The moments of one parameter group in flat buffers: every parameter starts at a multiple of 256 elements (what lies
    between stays zero), step counts in one int32 array.  state[p] holds views."""
    BLOCK = 256

    def __init__(self, group, state):
        self.params, self.bits, self.device = list(group['params']), group['state_bits'], group['params'][0].device
        sizes = [p.numel() for p in self.params]
        places = sorted((p.data_ptr(), p.data_ptr() + 4 * n) for p, n in zip(self.params, sizes) if n)
        if any(a[1] > b[0] for a, b in zip(places, places[1:])):
            raise _lib.UResNetHipError("AdamW: two parameters of a group share memory")
        self.blocks, at = [], 0
        for p, n in zip(self.params, sizes):
            if p.dtype != torch.float32 or not p.is_contiguous() or p.device != self.device:
                raise _lib.UResNetHipError("AdamW: the parameters of a group must be contiguous fp32 tensors on one device")
            self.blocks.append(at)
            at += -(-n // self.BLOCK)
        self.sizes = array.array('q', sizes).tobytes()
        self.blocks_there = torch.tensor(self.blocks, dtype=torch.int64, device=self.device)
        self.steps = torch.zeros(len(self.params), dtype=torch.int32, device=self.device)
        many = at * self.BLOCK
        if self.bits == 32:
            self.buffers = {k: torch.zeros(many, device=self.device) for k in ('exp_avg', 'exp_avg_sq')}
        else:
            self.buffers = {}
            for k in ('exp_avg', 'exp_avg_sq_root'):
                self.buffers[k] = torch.zeros(many, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn)
                self.buffers[k + '_scale'] = torch.zeros(at, device=self.device)
        moments = [buf.data_ptr() for buf in self.buffers.values()]
        if self.bits == 8:                                     # codes before scales
            moments = moments[0::2] + moments[1::2]
        self.places = (self.blocks_there.data_ptr(), self.steps.data_ptr(), self.bits, *(moments + [0, 0])[:4])
        self.waiting = []                                      # parameters without a state: no gradient yet
        for i, p in enumerate(self.params):                    # what the others bring along
            old = state.get(p)
            if not old:
                self.waiting.append(i)
            else:
                new = self.views(i)
                for k, v in new.items():
                    v.copy_(torch.as_tensor(old[k]).reshape(v.shape))
                state[p] = {**old, **new}

    def holds(self, group):
        ps = group['params']
        return (len(ps) == len(self.params) and all(map(operator.is_, ps, self.params)) and group['state_bits'] == self.bits
                and ps[0].device == self.device)

    def views(self, i):
        b, p = self.blocks[i], self.params[i]
        n = p.numel()
        out = {'step': self.steps[i]}
        for k, buf in self.buffers.items():
            if k.endswith('_scale'):
                out[k] = buf[b:b + -(-n // self.BLOCK)]
            else:
                out[k] = buf[b * self.BLOCK:b * self.BLOCK + n].view(p.shape)
        return out


class _Loaded:
    """A parameter's loaded state on its way through torch.optim.Optimizer.load_state_dict, which would cast 8-bit codes."""

    def __init__(self, entry):
        self.entry = entry


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW semantics (decoupled weight decay, no amsgrad) over all tensors of a group in one launch.  A group's moments
    are allocated together, also those of parameters that never get a gradient.

    state_bits (also per group): 32, or 8 -- both moments as e4m3 codes with one fp32 scale per 256 elements, 2 bytes per
    element instead of 8.  The second moment is held by its root and rounded in proportion (a rounding keeps the root's
    expectation); the same step gives the same bits.  Norm and bias parameters are best left at 32 in a group of their own.
    What 8 bits cost (betas 0.9, 0.999): with noisy gradients of one size the root scatters by 16 % rms around the 32-bit one
    after some hundred steps (its square lies 5 % above on average) and the update by 17 %.  m does not follow a change below
    half a code (3 to 6 %) per step: under an exactly steady gradient it can stop 38 % short of it.  Elements whose gradients are
    below some 1e-5 of their block's largest get smaller updates: their m rounds to 0, their root to the lowest code.
    betas[0] is at most 17/18: above, a first moment could not fall.
    max_grad_norm: clip by the global norm of all groups' gradients, as clip_grad_norm_ would before the step, but without
    writing the gradients; `grad_norm` is the norm before clipping (a 0-dim device tensor; None without clipping).
    grad_scale multiplies every gradient first, as in the other optimisers here.

    Step counts live on the device and nothing is staged on the host: after one eager step a step can be captured in a graph
    and replayed (learning rate and the other constants are then those of the capture).  state_dict() has torch.optim.AdamW's
    layout with 32-bit moments and loads into it; 8-bit moments load into 8-bit groups only.  Checkpoints hold `exp_avg` and
    `exp_avg_sq_root` as float8_e4m3fn beside their `_scale`s.  An infinite or NaN gradient makes its own element NaN only
    (with max_grad_norm all of them, as its norm is the factor's)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_grad_norm=None):
        self._pools = {}                       # group index -> _MomentPool
        self._held = [], []                    # the entries of `state` and what is in them, as the last step left them
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))
        if max_grad_norm is not None and not float(max_grad_norm) > 0:
            raise ValueError("AdamW: max_grad_norm must be positive (got %r)" % (max_grad_norm,))
        self.max_grad_norm = max_grad_norm
        self.grad_scale = 1.0
        self.grad_norm = None

    def add_param_group(self, group):
        g = {**self.defaults, **group}
        if g['state_bits'] not in (32, 8):
            raise ValueError("AdamW: state_bits is 32 or 8 (got %r)" % (g['state_bits'],))
        if torch.is_tensor(g['lr']):
            raise TypeError("AdamW: lr is a number, not a tensor")
        if not (g['lr'] >= 0 and g['eps'] >= 0 and g['weight_decay'] >= 0 and all(0 <= b < 1 for b in g['betas'])):
            raise ValueError("AdamW: lr, eps and weight_decay must not be negative, betas lie in [0, 1)")
        self._check_beta(g['state_bits'], g['betas'])
        super().add_param_group(group)
        if len(set(self.param_groups[-1]['params'])) < len(self.param_groups[-1]['params']):
            self.param_groups.pop()
            raise ValueError("AdamW: a parameter is listed twice")

    @staticmethod
    def _check_beta(bits, betas):
        if bits == 8 and betas[0] > 17 / 18:                   # a falling first moment would stay on its code
            raise ValueError("AdamW: 8-bit moments need betas[0] <= 17/18 (got %r)" % (betas[0],))

    def __setstate__(self, state):             # copied or unpickled: the pools are built again from `state`
        super().__setstate__(state)
        for p, entry in self.state.items():
            if isinstance(entry, _Loaded):
                self.state[p] = entry.entry
        self._pools = {}
        self._held = [], []
        for k, v in (('max_grad_norm', None), ('grad_scale', 1.0), ('grad_norm', None)):
            self.__dict__.setdefault(k, v)

    def __getstate__(self):
        return {**super().__getstate__(), 'max_grad_norm': self.max_grad_norm, 'grad_scale': self.grad_scale}

    def _pool(self, gi, group):
        pool = self._pools.get(gi)
        if pool is None or not pool.holds(group):
            dev = group['params'][0].device
            if dev.type == 'cuda' and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: run at least one eager step before capturing")
            pool = self._pools[gi] = _MomentPool(group, self.state)
            self._held = self._contents()
        return pool

    def _contents(self):
        entries = list(self.state.values())
        return entries, list(itertools.chain.from_iterable(map(dict.values, entries)))

    def _look_at_state(self):
        """What was cleared or replaced in `state` since the last step counts: the pools are then built again from it."""
        if not _lib.host().holds(self.state, *self._held):
            self._pools = {}

    def state_buffers(self, group=0):
        """The moments of a parameter group as flat tensors, parameters in order, each at a multiple of 256 elements (32 bits:
        exp_avg, exp_avg_sq; 8 bits: exp_avg, exp_avg_sq_root and a scale per 256 elements).  The optimiser's own buffers."""
        self._look_at_state()
        return dict(self._pool(group, self.param_groups[group]).buffers)

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._look_at_state()
        pools = [(group, self._pool(gi, group)) for gi, group in enumerate(self.param_groups) if group['params']]
        launched, self.grad_norm = _lib.host().adamw_step(
            [(pool.params, pool.sizes, *pool.places, float(group['lr']), *group['betas'], group['eps'], group['weight_decay'])
             for group, pool in pools], self.max_grad_norm, self.grad_scale)
        new = [(pool, i) for _, pool in pools for i in pool.waiting if pool.params[i].grad is not None]
        for pool, i in new:
            pool.waiting.remove(i)
            self.state[pool.params[i]] = pool.views(i)
        if new:
            self._held = self._contents()
        if launched:
            ops.bump_weights_epoch()
        return loss

    def state_dict(self):
        self._look_at_state()
        sd = super().state_dict()
        host = {gi: pool.steps.cpu() for gi, pool in self._pools.items()}          # one device read per group
        order = [(gi, i) for gi, group in enumerate(self.param_groups) for i in range(len(group['params']))]

        def step_of(k, v):
            gi, i = order[k]
            return float(host[gi][i]) if gi in host and self._pools[gi].holds(self.param_groups[gi]) else float(v['step'])
        sd['state'] = {k: {**v, 'step': torch.tensor(step_of(k, v))} if v else v for k, v in sd['state'].items()}
        for g in sd['param_groups']:                 # torch.optim.AdamW's remaining group keys, at their defaults
            for k, v in (('amsgrad', False), ('maximize', False), ('foreach', None), ('capturable', False),
                         ('differentiable', False), ('fused', None), ('decoupled_weight_decay', True)):
                g.setdefault(k, v)
        return sd

    def _checked(self, state_dict):
        """What load_state_dict takes over, looked through as a whole: this group's state_bits, the other keys as saved."""
        groups, saved = self.param_groups, state_dict['param_groups']
        if [len(g['params']) for g in groups] != [len(g['params']) for g in saved]:
            raise ValueError("AdamW: the loaded state has other parameter groups")
        state, taken = {}, []
        for group, old in zip(groups, saved):
            if old.get('amsgrad') or old.get('maximize') or old.get('decoupled_weight_decay') is False:
                raise NotImplementedError("AdamW: amsgrad, maximize and coupled weight decay states cannot be loaded")
            bits = old.get('state_bits', group['state_bits'])
            names = ('exp_avg', 'exp_avg_sq') if bits == 32 else ('exp_avg', 'exp_avg_scale', 'exp_avg_sq_root', 'exp_avg_sq_root_scale')
            for p, k in zip(group['params'], old['params']):
                entry = state_dict['state'].get(k)
                if not entry:
                    continue
                if not {*names, 'step'} <= set(entry) or bits != group['state_bits']:
                    raise ValueError("AdamW: the loaded moments are not %d-bit ones" % group['state_bits'])
                for n in names:
                    if entry[n].numel() != (-(-p.numel() // _MomentPool.BLOCK) if n.endswith('_scale') else p.numel()):
                        raise ValueError("AdamW: a loaded %s of shape %s for a parameter of shape %s" % (n, tuple(entry[n].shape), tuple(p.shape)))
                state[k] = _Loaded({**{n: entry[n] for n in names}, 'step': torch.as_tensor(entry['step']).round().to(torch.int32)})
            taken.append({**{k: v for k, v in group.items() if k != 'params'}, **old, 'state_bits': group['state_bits']})
            taken[-1]['lr'] = float(taken[-1]['lr'])
            self._check_beta(group['state_bits'], taken[-1]['betas'])
        return {**state_dict, 'state': state, 'param_groups': taken}

    def load_state_dict(self, state_dict):
        """Takes over the moments and every key of the groups but state_bits (a scheduler's `initial_lr` among them).  A state
        that does not fit is refused and leaves the optimiser as it was."""
        before = self.state, self.param_groups, self._pools, self._held
        last = self.register_load_state_dict_pre_hook(AdamW._checked)        # sees what the other hooks made of it
        try:
            super().load_state_dict(state_dict)
            for gi, group in enumerate(self.param_groups):
                if group['params']:
                    self._pool(gi, group)
        except BaseException:
            self.state, self.param_groups, self._pools, self._held = before
            raise
        finally:
            last.remove()


class GraphedStep:
    """One training step captured as a HIP graph and replayed: for small inputs the step is bound by the few hundred
    host-side launches, not by the GPU (CIFAR-shaped batch: 9 ms eager).  `step_fn(model, optimizer, *inputs)` is one of
    the *_train_step functions; inputs are copied into static buffers before each replay, the returned loss / outputs
    are static tensors that the next replay overwrites.  Works with this module's SGD, Adam and AdamW (whose step counts live
    on the device); shapes are fixed at construction; BatchNorm running statistics and counters advance on the device as in
    eager mode."""

    def __init__(self, step_fn, model, optimizer, *example_inputs, warmup=3):
        import gc
        gc.collect()                                # dead models drop out of the shared weight-image table now, not mid-capture
        self._static = [t.clone() for t in example_inputs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(warmup):                 # allocator pools, weight images and pointer tables reach steady state
                step_fn(model, optimizer, *self._static)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        optimizer.zero_grad(set_to_none=True)
        with torch.cuda.graph(self.graph, capture_error_mode="thread_local"):
            self._out = step_fn(model, optimizer, *self._static)
        self.warmup_steps = warmup

    def __call__(self, *inputs):
        for dst, src in zip(self._static, inputs):
            dst.copy_(src, non_blocking=True)
        self.graph.replay()
        # the replayed update rewrote the parameters through raw pointers: weight images cached by eager forwards
        # (an evaluation pass between training epochs) are stale now, and nothing else tells the caches so
        ops.bump_weights_epoch()
        return self._out


def seg_train_step(model, optimizer, images, targets, count_hook=None, grad_hook=None):
    """forward -> CE(ignore 255) -> zero_grad -> backward -> step; returns (loss, outputs) without syncing."""
    outputs = model(images)
    loss = compute_loss(outputs, targets, count_hook)
    optimizer.zero_grad()
    loss.backward()
    if grad_hook is not None:
        grad_hook()
    optimizer.step()
    return loss.detach(), outputs.detach()


def cls_train_step(model, optimizer, data, target, grad_hook=None):
    optimizer.zero_grad()
    output = model(data)
    loss = cross_entropy_loss(output, target)
    loss.backward()
    if grad_hook is not None:
        grad_hook()
    optimizer.step()
    return loss.detach(), output.detach()


def ice_train_step(model, optimizer, images, masks, grad_hook=None):
    optimizer.zero_grad()
    outputs = model(images)
    loss = bce_with_logits_loss(outputs, masks)
    loss.backward()
    if grad_hook is not None:
        grad_hook()
    optimizer.step()
    return loss.detach(), outputs.detach()
