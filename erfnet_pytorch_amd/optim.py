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

import numpy as np
import torch
from torch.optim import optimizer as _torch_optimizer

from . import ops
from ._lib import BF16, F32, call, size_query
from .train_ops import _host


_CODES = {torch.float32: F32, torch.bfloat16: BF16}


class _Plan:
    """The device tables of one launch: parameters of one group, device and type.  A parameter comes in with its first gradient and
    stays; where it has none its address is NULL and the launch leaves it alone, so its step count is in one place for all launches."""

    def __init__(self, group, device, code):
        self.group, self.device, self.code = group, device, code
        self.params, self.which = [], []                # which: places among all parameters in tables
        self.captured = False                           # a captured launch may write the grad fields at any time
        self.stale = True                               # the table lacks the gradients' present addresses


class AdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits is 32 or 8, got {state_bits}")
        self.state_bits, self.seed = int(state_bits), int(seed) & 0xFFFFFFFF
        self._reset()
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def _reset(self):
        self._plans = None                              # [[_Plan, ...] per group], None: to be built
        self._active = []                               # those with a gradient in them
        self._lr = []                                   # per group: [value on the devices, {device: double tensor}]
        self._kept = []                                 # what captured launches still read
        self._copies, self._copies_captured = {}, False
        self._moved = False                             # gradients moved, and the copies' places do not follow yet
        self._watch = _host.ParamWatch()

    def __getstate__(self):
        self._write_back_steps()
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed}

    def __setstate__(self, state):
        # unpickling and copying start without tables; torch's load_state_dict comes here too, with an optimizer whose tables captured
        # launches may read: load_state_dict below puts those aside
        super().__setstate__(state)
        if "_watch" not in self.__dict__:
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
        self._check_params(group["params"])

    @staticmethod
    def _settings(group):
        """The group's numbers as a launch takes them; they may have been changed by hand."""
        b1, b2, eps = float(group["betas"][0]), float(group["betas"][1]), float(group["eps"])
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0):
            raise ValueError(f"betas lie in [0, 1) and eps is not negative, got {group['betas']} and {group['eps']}")
        return b1, b2, eps, float(group["weight_decay"])

    @staticmethod
    def _check_params(params):
        for p in params:
            if p.dtype not in (torch.float32, torch.bfloat16):
                raise TypeError(f"AdamW updates float32 or bfloat16 parameters, got {p.dtype}")
            if p.is_neg():
                raise ValueError("AdamW updates parameters in memory of their own, got a view that holds their negative")
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
        return st

    def _write_back_steps(self):
        """The device's counts into `state`, except where the count there was changed by hand (or the state taken away) since the last time."""
        for plans in self._plans or ():
            for plan in plans:
                counts = plan.steps.cpu()
                for i, (p, first) in enumerate(zip(plan.params, plan.first_chunk)):
                    st = self.state.get(p, {})
                    if "step" in st and float(st["step"]) == plan.counts[i]:
                        st["step"] = counts[int(first)].float()
                        plan.counts[i] = float(st["step"])

    def _drop_plans(self):
        """Forget the device tables: the next step builds them anew from `state` and the parameters."""
        if self._plans is not None:
            self._write_back_steps()
            self._kept += [plan for plans in self._plans for plan in plans if plan.captured]
        self._plans = None

    def refresh(self):
        """To be called after entries of `state` were replaced or removed by hand between two steps.  Counts too: state_dict() brings
        those in `state` up to date, and a count that differs from what it wrote is taken over."""
        self._drop_plans()

    def state_dict(self):
        self._write_back_steps()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        for group in state_dict["param_groups"]:        # before anything is taken over
            lacking = [k for k in self.defaults if k not in group]
            if lacking:
                raise ValueError(f"AdamW: a saved group lacks {', '.join(lacking)}")
            for k, plain in (("amsgrad", False), ("maximize", False), ("decoupled_weight_decay", True)):
                if group.get(k, plain) != plain and (k != "decoupled_weight_decay" or group["weight_decay"]):
                    raise ValueError(f"AdamW: a saved group has {k}={group[k]}, which this optimizer does not compute")
            self._check_group({**group, "params": []})
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
        if self._plans is not None:
            self._kept += [plan for plans in self._plans for plan in plans if plan.captured]
        self._plans = None                              # the loaded step counts stand

    # -- device tables --------------------------------------------------------------------------
    def _build(self, groups):
        live = [p for g in groups for p in g if p.grad is not None and p.numel()]
        self._check_params(live)                        # they may have changed, or been put into a group by hand
        for p in live:
            ops.require_gpu(p, "AdamW")
        if live and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the first step with these parameters builds device tables and cannot be captured: "
                               "run one step before the capture")
        known = [plan for plans in self._plans or () for plan in plans] + [k for k in self._kept if isinstance(k, _Plan)] if live else []
        known = {id(p): (p.device, plan.code) for plan in known for p in plan.params}
        self._drop_plans()

        def again(p):                                   # without a gradient now, but as it was in a table before
            return p.grad is None and known.get(id(p)) == (p.device, _CODES.get(p.dtype)) and p.numel() and _dense(p)
        _host.adamw_no_overlap(live)
        more = {id(p): p for g in groups for p in g if again(p)} if known else {}
        try:
            _host.adamw_no_overlap(live + list(more.values()) if more else [])
        except ValueError:                              # with one that has a gradient
            more = {}
        held = more.keys() | {id(p) for p in live}
        block = size_query("erf_adamw_scale_block")
        plans, base, place, at, places = [], 0, 0, 0, []
        for number, group in enumerate(groups):
            rows = {}                                   # per device and type: id -> (parameter, random base, place)
            for p in group:
                if id(p) in held:
                    if id(p) in more:
                        places.append(at)
                    rows.setdefault((p.device, _CODES[p.dtype]), {})[id(p)] = (p, base, place)
                    place += 1
                base += -(-p.numel() // block) * block
                at += 1
            plans.append([plan for key, mine in rows.items() for plan in self._tables(number, *key, mine)])
        self._watch.bind(groups, places)
        self._plans, self._active = plans, None
        self._kept = [k for k in self._kept if not any(k is plan for ps in plans for plan in ps)]

    def _tables(self, number, device, code, mine):
        """Plans for these parameters.  Captured ones that describe some of them as they are now are taken up again, with the counts of
        `state`: a captured launch and the next step then move the same counts.  The rest come into one new plan."""
        names = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("exp_avg", "exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale")
        chunk = size_query("erf_adamw_chunk_elements")

        def describe(of):                               # [(parameter, random base, place)]
            states = [self._state_of(p) for p, _, _ in of]
            try:
                states, counts = [[st[k] for k in names] for st in states], [float(st["step"]) for st in states]
            except KeyError as e:
                raise ValueError(f"AdamW: a parameter's state lacks {e} (state_bits={self.state_bits})") from None
            rows, holds = _host.adamw_table([p for p, _, _ in of], states, [base for _, base, _ in of])
            return rows, holds, counts, np.array(counts).astype(np.int32)
        plans, rest = [], dict(mine)
        for plan in reversed([k for k in self._kept if isinstance(k, _Plan)]):
            if (plan.group, plan.device, plan.code) != (number, device, code) or any(id(p) not in rest for p in plan.params):
                continue
            of = [rest[id(p)] for p in plan.params]
            rows, _, counts, steps = describe(of)
            if not torch.equal(rows, plan.rows):
                continue
            plan.steps.copy_(torch.from_numpy(steps[plan.owner]))
            plan.counts = counts                        # as they stand in `state`
            plan.which, plan.stale = [place for _, _, place in of], True
            plans.append(plan)
            for p in plan.params:
                del rest[id(p)]
        if rest:
            plan = _Plan(number, device, code)
            plan.params, plan.which = [p for p, _, _ in rest.values()], [place for _, _, place in rest.values()]
            plan.rows, plan.holds, plan.counts, steps = describe(list(rest.values()))
            per = -(-plan.rows[:, 6].numpy() // chunk)  # chunks of each tensor
            plan.first_chunk = np.cumsum(per) - per
            plan.owner = np.repeat(np.arange(len(per)), per)
            where = np.stack([plan.owner, np.arange(len(plan.owner)) - plan.first_chunk[plan.owner]], 1).astype(np.int32)
            plan.table = plan.rows.to(device)
            plan.chunks = torch.from_numpy(where).to(device)
            plan.steps = torch.from_numpy(steps[plan.owner]).to(device)
            plans.append(plan)
        return plans

    def _copy_places(self):
        """Gradients with other strides than their parameter's are copied into its order every step; where the copies lie."""
        if self._copies_captured:
            self._kept.append(self._copies)
        self._copies_captured = False
        copied = self._watch.copied()
        params = [p for _, p in sorted((i, p) for ps in self._plans for plan in ps for i, p in zip(plan.which, plan.params))] if copied else []
        self._copies = {i: (torch.empty_like(params[i]).detach(), params[i]) for i in copied}
        for ps in self._plans:
            for plan in ps:
                plan.copies = [self._copies[i][0].data_ptr() if i in self._copies else 0 for i in plan.which] if copied else [0] * len(plan.which)

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
    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        settings = [self._settings(g) for g in self.param_groups]              # a refused step updates no group
        groups = [g["params"] for g in self.param_groups]
        seen = 2 if self._plans is None else self._watch.look(groups)
        if seen == 2:
            with torch.no_grad():
                self._build(groups)
            try:
                self._watch.look(groups)
            except BaseException:
                self._drop_plans()
                raise
        if seen:
            self._moved = True                          # until the copies have their places, and each table its addresses
            for plans in self._plans:
                for plan in plans:
                    plan.stale = True
            if self._active is None or self._watch.changed:
                present = self._watch.present()
                self._active = [plan for plans in self._plans for plan in plans if any(present[i] for i in plan.which)]
        if self._moved:
            with torch.no_grad():
                self._copy_places()
            self._moved = False
        if not self._active:
            return loss
        capturing = torch.cuda.is_current_stream_capturing()
        if self._copies:
            self._copies_captured = self._copies_captured or capturing
            with torch.no_grad():
                for own, p in self._copies.values():
                    own.copy_(p.grad)
        self.refresh_lr()
        here = torch._C._cuda_getDevice()
        for plan in self._active:
            numbers, lr = settings[plan.group], self._lr[plan.group][1][plan.device]
            if plan.device.index == here:
                self._launch(numbers, lr, plan, capturing)
            else:
                with torch.cuda.device(plan.device):
                    self._launch(numbers, lr, plan, capturing)
        self._watch.bump()
        ops.bump_param_epoch()                          # the parameters changed through raw pointers
        return loss

    def step(self, closure=None):
        """One update of every parameter that has a gradient."""
        if self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _torch_optimizer._global_optimizer_pre_hooks or \
                _torch_optimizer._global_optimizer_post_hooks:
            return _hooked_step(self, closure)
        return self._step(closure)

    step.hooked = True                                  # torch's wrapper (hooks and a profiler range, 8 us) is used where a hook asks for it

    def _launch(self, numbers, lr, plan, capturing):
        stream = ops._stream()
        table = plan.table.data_ptr()
        if plan.stale or plan.captured or capturing:
            plan.captured = plan.captured or capturing
            self._watch.set_grads(table, plan.which, plan.copies, stream)
            if not capturing:                           # a captured launch writes its addresses when it is replayed
                plan.stale = False
        call("erf_adamw_step", table, plan.chunks.data_ptr(), plan.steps.data_ptr(), plan.chunks.shape[0], lr.data_ptr(),
             *numbers, plan.code, self.state_bits, self.seed, stream)


_hooked_step = torch.optim.Optimizer.profile_hook_step(AdamW._step)


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
