"""Operators of training and answering beside the convolution engine's: log probabilities of labels with entropy and top
alternatives, group normalisation with an activation on channels-last maps.

Each is a plain function on tensors (one call through the C ABI on the current stream of the tensor's device, outputs from
torch's allocator) and a registered op of the namespace `erfnet_mi355`, with a fake kernel for shapes and types and no CPU
kernel, like those of torch_ops.py.  The differentiable entry points are loss.class_log_probs and norm.group_norm_act.
"""
from __future__ import annotations

import contextlib

import torch

from ._lib import BF16, F32, call, size_query
from .torch_ops import LIB, NS

OPS = []                      # names, in registration order (tests walk this list)

_no_guard = contextlib.nullcontext()


def _register(schema: str, impl, fake):
    name = schema.split("(", 1)[0]
    LIB.define(schema)
    LIB.impl(name, impl, "CUDA")
    torch.library.register_fake(f"{NS}::{name}", fake, lib=LIB)
    OPS.append(name)


def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def on_device_of(t: torch.Tensor):
    """Launches inside go to the current stream of t's device, whichever device is current outside."""
    return _no_guard if t.device.index == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def dtype_code(t: torch.Tensor, who: str) -> int:
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"{who}: float32 or bfloat16 tensors, got {t.dtype}")


def _p(t):
    return 0 if t is None else t.data_ptr()


def _same_device(who, t, **others):
    for name, o in others.items():
        if o is not None and o.device != t.device:
            raise ValueError(f"{who}: {name} is on {o.device}, the input on {t.device}")


# ------------------------------------------------------------------------------------------------ label log probabilities
TOP_MAX = 32


def class_layout(z: torch.Tensor):
    """(tensor, N, C, L, stride of N, stride of C, shape without the class axis, rows) of logits [N, C, ...]: `rows` where the
    classes of a position lie side by side ([N, C], or a channels-last map), else planes of L positions.  Other layouts are
    copied into planes."""
    n, c = z.shape[:2]
    rest = z.shape[2:]
    length = rest.numel()
    if length == 1:
        z = z if c == 1 or z.stride(1) == 1 else z.contiguous()
        return z, n, c, 1, z.stride(0) if n > 1 else c, 1, (n, *rest), True
    if c > 1 and z.stride(1) == 1 and z.movedim(1, -1).is_contiguous():
        return z, n * length, c, 1, c, 1, (n, *rest), True
    dense = 1                                               # the map's own axes, innermost last, without gaps
    for size, stride in zip(reversed(rest), reversed(z.stride()[2:])):
        dense = dense * size if size == 1 or stride == dense else 0
    if not dense or not (c == 1 or z.stride(1) >= max(length, 2)):
        z = z.contiguous()
    return z, n, c, length, z.stride(0) if n > 1 else c * length, max(z.stride(1) if c > 1 else 0, length, 2), (n, *rest), False


def _like_layout(z, rows):
    """A dense tensor for the gradient: classes side by side for rows (channels-last for maps), else planes."""
    if rows and z.dim() > 2:
        return z.new_empty((z.shape[0], *z.shape[2:], z.shape[1])).movedim(-1, 1)
    return z.new_empty(z.shape)


def _top_shape(shape, k, rows):
    """Memory shape of the alternatives, and the axis order that puts k where the class axis was."""
    if rows:
        return (*shape, k), (0, len(shape), *range(1, len(shape)))
    return (shape[0], k, *shape[1:]), None


def _check_target(who, target, shape, z):
    if target is None:
        return None
    if target.dtype != torch.int64:
        raise TypeError(f"{who}: targets are int64 class indices, got {target.dtype}")
    if target.shape != shape:
        raise ValueError(f"{who}: expected targets of shape {tuple(shape)}, got {tuple(target.shape)}")
    if target.device != z.device:
        raise ValueError(f"{who}: target is on {target.device}, the input on {z.device}")
    return target.contiguous()


def class_log_probs_fwd(logits, target, top_k=0, ignore_index=-100, with_stats=True):
    """(log_prob, entropy, stats, top_log_probs, top_indices) of logits [N, C, ...]; loss.class_log_probs describes them.  stats
    [2, ...]: the row maximum and log sum e^{z - max}, for the backward pass (None without `with_stats`).  Without a target
    log_prob is empty."""
    who = "class_log_probs"
    code = dtype_code(logits, who)
    if logits.dim() < 2 or logits.shape[1] < 1:
        raise ValueError(f"{who}: logits have shape [N, C, ...] with at least one class, got {tuple(logits.shape)}")
    if not 0 <= top_k <= min(TOP_MAX, logits.shape[1]):
        raise ValueError(f"{who}: top_k lies between 0 and min({TOP_MAX}, classes), got {top_k} for {logits.shape[1]} classes")
    z, n, c, length, sn, sc, shape, rows = class_layout(logits)
    target = _check_target(who, target, shape, z)
    new = z.new_empty
    log_prob = new(shape if target is not None else (0,), dtype=torch.float32)
    entropy = new(shape, dtype=torch.float32)
    stats = new((2, *shape), dtype=torch.float32) if with_stats else None
    top_shape, order = _top_shape(shape, top_k, rows)
    top, index = new(top_shape, dtype=torch.float32), new(top_shape, dtype=torch.int64)
    if entropy.numel():
        with on_device_of(z):
            nbytes = size_query("erf_class_log_probs_workspace_bytes", code, n, c, length, sc, top_k)
            ws = new(nbytes, dtype=torch.uint8) if nbytes else None
            call("erf_class_log_probs_fwd", z.data_ptr(), code, n, c, length, sn, sc, _p(target), ignore_index,
                 log_prob.data_ptr() if target is not None else 0, entropy.data_ptr(), _p(stats), top_k, top.data_ptr() if top_k else 0,
                 index.data_ptr() if top_k else 0, _p(ws), _stream())
    if order is not None and top_k:
        top, index = top.permute(order), index.permute(order)
    elif not top_k:
        top, index = top.view(shape[0], 0, *shape[1:]), index.view(shape[0], 0, *shape[1:])
    return log_prob, entropy, stats, top, index


def class_log_probs_bwd(logits, target, stats, entropy, top_indices, g_log_prob, g_entropy, g_top, ignore_index=-100):
    """d logits, laid out as the logits."""
    z, n, c, length, sn, sc, shape, rows = class_layout(logits)
    code = dtype_code(z, "class_log_probs")
    target = _check_target("class_log_probs", target, shape, z)
    dz = _like_layout(z, rows)
    if not dz.numel():
        return dz
    if rows:
        dn, dc = c, 1
    else:
        dn, dc = c * length, max(length, 2)              
    k = top_indices.shape[1] if g_top is not None else 0

    def flat(t, like_top=False):
        if t is None:
            return None
        if like_top and rows and t.dim() > 2:
            t = t.movedim(1, -1)
        return t.float().contiguous() if t.dtype != torch.int64 else t.contiguous()
    g_log_prob, g_entropy = flat(g_log_prob), flat(g_entropy)
    g_top, top_indices = (flat(g_top, True), flat(top_indices, True)) if k else (None, None)
    with on_device_of(z):
        call("erf_class_log_probs_bwd", z.data_ptr(), code, n, c, length, sn, sc, _p(target), ignore_index, stats.data_ptr(), entropy.data_ptr(),
             _p(g_log_prob), _p(g_entropy), k, _p(top_indices), _p(g_top), dz.data_ptr(), dn, dc, _stream())
    return dz


def _lp_fwd_fake(logits, target, top_k, ignore_index):
    shape = (logits.shape[0], *logits.shape[2:])
    new = logits.new_empty
    top = (shape[0], top_k, *shape[1:])
    outs = [new(top, dtype=torch.float32), new(top, dtype=torch.int64)]
    if top_k and len(shape) > 1 and class_layout(logits)[-1]:
        outs = [new((*shape, top_k), dtype=o.dtype).movedim(-1, 1) for o in outs]
    return (new(shape if target is not None else (0,), dtype=torch.float32), new(shape, dtype=torch.float32), new((2, *shape), dtype=torch.float32), *outs)


_register("class_log_probs_fwd(Tensor logits, Tensor? target, int top_k, int ignore_index) -> (Tensor, Tensor, Tensor, Tensor, Tensor)",
          lambda logits, target, top_k, ignore_index: class_log_probs_fwd(logits, target, top_k, ignore_index), _lp_fwd_fake)


def _lp_bwd_fake(logits, target, stats, entropy, top_indices, g_log_prob, g_entropy, g_top, ignore_index):
    z, *_, rows = class_layout(logits)
    return _like_layout(z, rows)


_register("class_log_probs_bwd(Tensor logits, Tensor? target, Tensor stats, Tensor entropy, Tensor top_indices, Tensor? g_log_prob, "
          "Tensor? g_entropy, Tensor? g_top, int ignore_index) -> Tensor", class_log_probs_bwd, _lp_bwd_fake)


# ------------------------------------------------------------------------------------------------ group norm + activation
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2}


def channels_last(x: torch.Tensor) -> torch.Tensor:
    """Logical [N, C, ...] as a contiguous [N, ..., C]; zero-copy where the memory is channels-last."""
    last = x.movedim(1, -1)
    if last.is_contiguous():
        return last
    if x.dim() == 4 and x.is_contiguous() and x.numel():
        n, c, h, w = x.shape
        out = x.new_empty((n, h, w, c))
        code = dtype_code(x, "group_norm_act")
        with on_device_of(x):
            call("erf_nchw_to_nhwc", x.data_ptr(), code, out.data_ptr(), code, n, c, h, w, _stream())
        return out
    return last.contiguous()


def _gn_check(x, weight, bias, groups, activation):
    who = "group_norm_act"
    code = dtype_code(x, who)
    if x.dim() < 2 or not x.is_contiguous():
        raise ValueError(f"{who}: a contiguous channels-last tensor [N, ..., C], got shape {tuple(x.shape)} strides {x.stride()}")
    c = x.shape[-1]
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"{who}: {c} channels do not split into {groups} groups")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{who}: activation is one of {sorted(ACTIVATIONS)}, got {activation!r}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (c,):
            raise ValueError(f"{who}: {name} has shape [{c}], got {tuple(t.shape)}")
    _same_device(who, x, weight=weight, bias=bias)
    return code, x.shape[0], x.numel() // max(1, x.shape[0] * c), c


def _f32(t):
    return t if t is None or (t.dtype == torch.float32 and t.is_contiguous()) else t.float().contiguous()


def _gn_workspace(x, code, n, hw, c, groups):
    return torch.empty(size_query("erf_group_norm_workspace_bytes", code, n, hw, c, groups), dtype=torch.uint8, device=x.device)


def group_norm_act_fwd(x, weight, bias, groups, eps, activation):
    """(y, mean [N, groups], rstd [N, groups]) of a contiguous channels-last x [N, ..., C]; norm.group_norm_act describes them."""
    code, n, hw, c = _gn_check(x, weight, bias, groups, activation)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"group_norm_act: invalid eps {eps}")
    weight, bias = _f32(weight), _f32(bias)
    y = torch.empty_like(x)
    mean, rstd = x.new_empty((n, groups), dtype=torch.float32), x.new_empty((n, groups), dtype=torch.float32)
    if x.numel():
        with on_device_of(x):
            ws = _gn_workspace(x, code, n, hw, c, groups)
            call("erf_group_norm_fwd", x.data_ptr(), y.data_ptr(), code, n, hw, c, groups, _p(weight), _p(bias), eps, ACTIVATIONS[activation],
                 mean.data_ptr(), rstd.data_ptr(), ws.data_ptr(), _stream())
    return y, mean, rstd


def group_norm_act_bwd(dy, x, weight, bias, mean, rstd, groups, activation):
    """(dx, dweight [C], dbias [C]) from a contiguous channels-last dy; the parameter gradients are fp32 whatever the types."""
    code, n, hw, c = _gn_check(x, weight, bias, groups, activation)
    if dy.shape != x.shape or dy.dtype != x.dtype or not dy.is_contiguous():
        raise ValueError(f"group_norm_act: dy is a contiguous {x.dtype} tensor of shape {tuple(x.shape)}, got {dy.dtype} {tuple(dy.shape)} strides {dy.stride()}")
    if mean.shape != (n, groups) or rstd.shape != (n, groups) or mean.dtype != torch.float32 or rstd.dtype != torch.float32:
        raise ValueError(f"group_norm_act: mean and rstd are fp32 [{n}, {groups}]")
    _same_device("group_norm_act", x, dy=dy, mean=mean, rstd=rstd)
    weight, bias, mean, rstd = _f32(weight), _f32(bias), _f32(mean), _f32(rstd)
    dx = torch.empty_like(x)
    if not x.numel():
        return dx, x.new_zeros(c, dtype=torch.float32), x.new_zeros(c, dtype=torch.float32)
    dweight, dbias = x.new_empty(c, dtype=torch.float32), x.new_empty(c, dtype=torch.float32)
    with on_device_of(x):
        ws = _gn_workspace(x, code, n, hw, c, groups)
        call("erf_group_norm_bwd", x.data_ptr(), dy.data_ptr(), dx.data_ptr(), code, n, hw, c, groups, _p(weight), _p(bias), ACTIVATIONS[activation],
             mean.data_ptr(), rstd.data_ptr(), dweight.data_ptr(), dbias.data_ptr(), ws.data_ptr(), _stream())
    return dx, dweight, dbias


def _gn_fwd_fake(x, weight, bias, groups, eps, activation):
    stat = (x.shape[0], groups)
    return torch.empty_like(x), x.new_empty(stat, dtype=torch.float32), x.new_empty(stat, dtype=torch.float32)


_register("group_norm_act_fwd(Tensor x, Tensor? weight, Tensor? bias, int groups, float eps, str activation) -> (Tensor, Tensor, Tensor)",
          group_norm_act_fwd, _gn_fwd_fake)


def _gn_bwd_fake(dy, x, weight, bias, mean, rstd, groups, activation):
    return torch.empty_like(x), x.new_empty(x.shape[-1], dtype=torch.float32), x.new_empty(x.shape[-1], dtype=torch.float32)


_register("group_norm_act_bwd(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor mean, Tensor rstd, int groups, str activation) -> "
          "(Tensor, Tensor, Tensor)", group_norm_act_bwd, _gn_bwd_fake)
