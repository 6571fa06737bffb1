"""AdamW over many tensors in one launch, with the moments in 32 or in 8 bits.

    opt = AdamW(model.parameters(), lr=5e-4, weight_decay=1e-2, state_bits=8)
    loss.backward(); opt.step(); opt.zero_grad()

`AdamW` is a torch.optim.Optimizer: parameter groups, learning-rate schedulers, state_dict / load_state_dict work as usual.  It
stands beside the flat-arena Adam of trainer.Trainer (coupled weight decay, one arena) for parameters that live in tensors of
their own, and decays the weights apart from the gradient:

    m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

State per parameter, `state[p]`:
  "step"                                            number of steps taken (written back by state_dict())
  state_bits=32: "exp_avg", "exp_avg_sq"            fp32, shaped and laid out as the parameter
  state_bits=8:  "exp_avg", "exp_avg_sq_root"       float8_e4m3fn codes of m and sqrt(v), shaped and laid out as the parameter
                 "exp_avg_scale", "exp_avg_sq_root_scale"    fp32 powers of two, one for each 256 elements in memory order
8 bits take 2 1/32 bytes per parameter in place of 8.  Codes are rounded up or down at random (from `seed`, the step and the
element's position alone: the same run gives the same bits); the update itself uses the moments before they are rounded.

Parameters are fp32 or bf16.  bf16 parameters are rounded to the nearest value after each update, so that changes below half a
bf16 step (2^-9 of the value) are lost: keep fp32 parameters where such changes matter.
"""
from __future__ import annotations

import ctypes
import operator

import torch

from . import ops
from ._lib import BF16, F32, call, size_query

_data_ptr = torch.Tensor.data_ptr


class _Plan:
    """The device tables of one launch: parameters of one group, device and type that have a gradient."""

    def __init__(self, device, code):
        self.device, self.code = device, code
        self.params, self.bases = [], []
        self.captured = False                           # a captured launch may write the grad fields at any time


class AdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits is 32 or 8, got {state_bits}")
        self.state_bits, self.seed = int(state_bits), int(seed) & 0xFFFFFFFF
        self._reset()
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def _reset(self):
        self._plans = None                              # [[_Plan, ...] per group], None: to be built
        self._lr = []                                   # per group: [value on the devices, {device: double tensor}]
        self._kept = []                                 # what captured launches still read
        self._copies, self._copies_captured = [], False

    def __getstate__(self):
        self._write_back_steps()
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._reset()

    # -- argument checks ------------------------------------------------------------------------
    def _check_group(self, group):
        b1, b2 = group["betas"]
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas lie in [0, 1), got {group['betas']}")
        lr = group["lr"]
        if isinstance(lr, torch.Tensor) and lr.numel() != 1:
            raise ValueError("a learning rate tensor has one element")
        if not isinstance(lr, torch.Tensor) and not 0.0 <= lr < float("inf"):
            raise ValueError(f"invalid learning rate {lr}")
        if not 0.0 <= group["eps"] < float("inf"):
            raise ValueError(f"invalid eps {group['eps']}")
        if not 0.0 <= group["weight_decay"] < float("inf"):
            raise ValueError(f"invalid weight decay {group['weight_decay']}")
        for p in group["params"]:
            if p.dtype not in (torch.float32, torch.bfloat16):
                raise TypeError(f"AdamW updates float32 or bfloat16 parameters, got {p.dtype}")
            if not _dense(p):
                raise ValueError(f"AdamW updates parameters whose memory has no gaps or overlaps, got shape {tuple(p.shape)} strides {p.stride()}")

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            self._check_group(self.param_groups[-1])
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise
        self._drop_plans()

    # -- state ----------------------------------------------------------------------------------
    def _state_of(self, p):
        st = self.state[p]
        if not st:
            st["step"] = torch.zeros(())
            if self.state_bits == 32:
                st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
                st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
            else:
                blocks = -(-p.numel() // size_query("erf_adamw_scale_block"))
                for k in ("exp_avg", "exp_avg_sq_root"):
                    st[k] = torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn)
                    st[k + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        names = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("exp_avg", "exp_avg_sq_root")
        want = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
        for k in names:
            t = st.get(k)
            if t is None or t.dtype != want or t.device != p.device or t.numel() != p.numel() or not (
                    t.stride() == p.stride() or (t.is_contiguous() and p.is_contiguous())):
                raise ValueError(f"state '{k}' of a parameter of shape {tuple(p.shape)}: expected a {want} tensor laid out as the parameter")
            if self.state_bits == 8:
                s = st.get(k + "_scale")
                if s is None or s.dtype != torch.float32 or s.device != p.device or not s.is_contiguous() or \
                        s.numel() != -(-p.numel() // size_query("erf_adamw_scale_block")):
                    raise ValueError(f"state '{k}_scale' of a parameter of shape {tuple(p.shape)}: expected one fp32 value per 256 elements")
        return st

    def _write_back_steps(self):
        for plans in self._plans or ():
            for plan in plans:
                counts = plan.steps.cpu()
                for p, first in zip(plan.params, plan.first_chunk):
                    self.state[p]["step"] = counts[first].float()

    def _drop_plans(self):
        """Forget the device tables: the next step builds them anew from `state` and the parameters."""
        if self._plans is not None:
            self._write_back_steps()
            self._kept += [plan for plans in self._plans for plan in plans if plan.captured]
        self._plans = None

    def refresh(self):
        """To be called after entries of `state` were replaced by hand between two steps."""
        self._drop_plans()

    def state_dict(self):
        self._write_back_steps()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        # torch's loader casts every state tensor to the parameter's type: the values are put in place again as they were saved
        self._write_back_steps()
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            for k, v in saved.get(i, {}).items():
                if k == "step":
                    self.state[p][k] = torch.as_tensor(float(v))
                elif isinstance(v, torch.Tensor):
                    here = torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device=p.device) if _dense(v) else \
                        torch.empty(v.shape, dtype=v.dtype, device=p.device)
                    _raw(here).copy_(_raw(v))
                    self.state[p][k] = here
        for group in self.param_groups:
            self._check_group(group)
        if self._plans is not None:
            self._kept += [plan for plans in self._plans for plan in plans if plan.captured]
        self._plans = None                              # the loaded step counts stand

    # -- device tables --------------------------------------------------------------------------
    def _build(self):
        live = [p for g in self.param_groups for p in g["params"] if p.grad is not None and p.numel()]
        for p in live:
            ops.require_gpu(p, "AdamW")
        if live and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the first step with these parameters builds device tables and cannot be captured: "
                               "run one step before the capture")
        self._drop_plans()
        chunk, block = size_query("erf_adamw_chunk_elements"), size_query("erf_adamw_scale_block")
        plans, base = [], 0
        for group in self.param_groups:
            mine = {}
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    key = (p.device, F32 if p.dtype == torch.float32 else BF16)
                    plan = mine.setdefault(key, _Plan(*key))
                    plan.params.append(p)
                    plan.bases.append(base)
                base += -(-p.numel() // block) * block
            plans.append(list(mine.values()))
        _no_overlap([p for ps in plans for plan in ps for p in plan.params])
        for ps in plans:
            for plan in ps:
                rows, where, steps, plan.first_chunk, at = [], [], [], [], 0
                for t, (p, b) in enumerate(zip(plan.params, plan.bases)):
                    st = self._state_of(p)
                    second = st["exp_avg_sq"] if self.state_bits == 32 else st["exp_avg_sq_root"]
                    scales = (st["exp_avg_scale"].data_ptr(), st["exp_avg_sq_root_scale"].data_ptr()) if self.state_bits == 8 else (0, 0)
                    rows.append([p.data_ptr(), 0, st["exp_avg"].data_ptr(), second.data_ptr(), *scales, p.numel(), b])
                    n = -(-p.numel() // chunk)
                    plan.first_chunk.append(at)
                    at += n
                    where.append(torch.stack([torch.full((n,), t, dtype=torch.int32), torch.arange(n, dtype=torch.int32)], 1))
                    steps.append(torch.full((n,), int(st["step"]), dtype=torch.int32))
                plan.table = torch.tensor(rows, dtype=torch.int64).to(plan.device)
                plan.chunks = torch.cat(where).to(plan.device)
                plan.steps = torch.cat(steps).to(plan.device)
                # the states that the table points at live as long as it does
                plan.holds = [t for p in plan.params for t in self.state[p].values()] + [p.data for p in plan.params]
        self._plans = plans
        self._params = [p for ps in plans for plan in ps for p in plan.params]
        self._ptrs = tuple(map(_data_ptr, self._params))

    def _bind_grads(self, grads):
        """Check new gradients and note the addresses for the tables."""
        copies, used = [], []
        for p, g in zip(self._params, grads):
            if g.is_sparse or g.dtype != p.dtype or g.device != p.device or g.shape != p.shape:
                raise ValueError(f"AdamW: a gradient of a parameter {p.dtype} {tuple(p.shape)} has to be a dense tensor of the same type, "
                                 f"shape and device, got {g.dtype} {tuple(g.shape)}")
            if g.stride() != p.stride() and not (g.is_contiguous() and p.is_contiguous()):
                own = torch.empty_like(p)               # other strides than the parameter's: a copy in its order, renewed every step
                copies.append((own, g))
                g = own
            used.append(g)
        if self._copies_captured:
            self._kept.append(self._copies)
        self._copies, self._copies_captured = copies, False
        at = 0
        for ps in self._plans:
            for plan in ps:
                n = len(plan.params)
                plan.grads = (ctypes.c_void_p * n)(*map(_data_ptr, used[at:at + n]))
                plan.fresh = True
                at += n
        self._grads, self._grad_ptrs = grads, tuple(map(_data_ptr, grads))

    def refresh_lr(self):
        """Bring the learning rates to the device.  step() does so by itself; a program that replays a captured step calls this
        after it has changed `param_groups[i]["lr"]` and before the replay.  A learning rate that is a device tensor is read by
        the step itself, captured or not."""
        for i, group in enumerate(self.param_groups):
            if len(self._lr) <= i:
                self._lr.append([None, {}])
            lr, (value, where) = group["lr"], self._lr[i]
            for plan in self._plans[i] if self._plans else ():
                if plan.device not in where:
                    where[plan.device] = torch.empty(1, dtype=torch.float64, device=plan.device)
                    value = None
            if isinstance(lr, torch.Tensor) and not lr.is_cuda:
                lr = float(lr)
            if isinstance(lr, torch.Tensor):
                for t in where.values():
                    t.copy_(lr.reshape(1))
                self._lr[i][0] = None
            elif lr != value:
                for t in where.values():
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: the learning rate changed since the last step; call refresh_lr() before the capture "
                                           "(a captured step reads it from device memory)")
                    t.fill_(float(lr))
                self._lr[i][0] = lr

    def note_replay(self):
        """To be called after the replay of a captured step: weights packed from the parameters are packed anew when next used."""
        ops.bump_param_epoch()

    # -- the step -------------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        grads = [p.grad for g in self.param_groups for p in g["params"]]
        if self._plans is None or not self._same(grads):
            self._build()
            self._bind_grads([p.grad for p in self._params])
            self._all_grads, self._without = grads, [g is None for g in grads]
        if not self._params:
            return loss
        capturing = torch.cuda.is_current_stream_capturing()
        if self._copies:
            self._copies_captured = self._copies_captured or capturing
            for own, g in self._copies:
                own.copy_(g)
        self.refresh_lr()
        for group, where, plans in zip(self.param_groups, self._lr, self._plans):
            for plan in plans:
                if plan.device.index == torch._C._cuda_getDevice():
                    self._launch(group, where[1][plan.device], plan, capturing)
                else:
                    with torch.cuda.device(plan.device):
                        self._launch(group, where[1][plan.device], plan, capturing)
        torch.autograd.graph.increment_version(self._params)
        ops.bump_param_epoch()                          # the parameters changed through raw pointers
        return loss

    def _same(self, grads):
        """Whether the tables describe these gradients, and the parameters are where they were; new gradients of the same
        parameters are bound on the way."""
        if len(grads) != len(self._all_grads):
            return False
        if all(map(operator.is_, grads, self._all_grads)):
            if tuple(map(_data_ptr, self._params)) != self._ptrs:
                return False
            if tuple(map(_data_ptr, self._grads)) != self._grad_ptrs:
                self._bind_grads(self._grads)
            return True
        if [g is None for g in grads] != self._without or tuple(map(_data_ptr, self._params)) != self._ptrs:
            return False
        self._bind_grads([p.grad for p in self._params])
        self._all_grads = grads
        return True

    def _launch(self, group, lr, plan, capturing):
        stream = ops._stream()
        if plan.fresh or plan.captured or capturing:
            call("erf_adamw_set_grads", plan.table.data_ptr(), plan.grads, len(plan.params), stream)
            plan.fresh = False
            plan.captured = plan.captured or capturing
        b1, b2 = group["betas"]
        call("erf_adamw_step", plan.table.data_ptr(), plan.chunks.data_ptr(), plan.steps.data_ptr(), plan.chunks.shape[0], lr.data_ptr(),
             b1, b2, group["eps"], group["weight_decay"], plan.code, self.state_bits, self.seed, stream)


def _dense(t):
    """Whether the elements fill a stretch of memory without gaps or overlaps, in any order of the axes."""
    need = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride != need:
            return False
        need *= size
    return True


def _raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _no_overlap(params):
    spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size(), p.device.index) for p in params)
    for a, b in zip(spans, spans[1:]):
        if a[2] == b[2] and b[0] < a[1]:
            raise ValueError("AdamW: two parameters share memory; give the optimizer one of them")
