"""Operators of training and answering beside the convolution engine's: log probabilities of labels with entropy and top
alternatives, group normalisation with an activation on channels-last maps.

Each is a function of the C++ host extension _host (csrc/host_ops.cpp: argument checks, output allocation, one call through the C ABI
on the current stream of the tensors' device) and a registered op of the namespace `erfnet_mi355` with fake and device kernels and
no CPU kernel, like those of torch_ops.py.  The differentiable entry points are loss.class_log_probs and norm.group_norm_act.

    class_log_probs_fwd(logits [N, C, ...], target, top_k, ignore_index) -> log_prob, entropy, stats, top_log_probs, top_indices
        stats [2, N, ...]: the maximum and log sum e^{z - max} of every position, for the backward pass; log_prob is empty
        without a target
    class_log_probs_bwd(logits, target, stats, entropy, top_indices, g_log_prob, g_entropy, g_top, ignore_index) -> dlogits
    group_norm_act_fwd(x [N, ..., C], weight, bias, groups, eps, activation) -> y, stats [2, N, groups] (mean, 1 / sqrt(var + eps))
    group_norm_act_bwd(dy, x, weight, bias, stats, groups, activation) -> dx, dweight, dbias (fp32)
"""
from __future__ import annotations

import torch

from . import _lib  # noqa: F401  (says how to build when the library is missing)
from .torch_ops import LIB, NS

try:
    from . import _host
except ImportError as e:
    raise ImportError("erfnet_pytorch_amd/_host.so is missing or does not load: build it with `python -c 'import __graft_entry__ as g; "
                      "g.build()'` or `make -C erfnet_pytorch_amd/csrc`. There is no fallback path.") from e

OPS = []                      # names, in registration order (tests walk this list)

class_log_probs_fwd = _host.class_log_probs_fwd
class_log_probs_bwd = _host.class_log_probs_bwd
class_layout = _host.class_layout
group_norm_act_fwd = _host.group_norm_act_fwd
group_norm_act_bwd = _host.group_norm_act_bwd


def _symbolic(*tensors) -> bool:
    return any(isinstance(n, torch.SymInt) for t in tensors if t is not None for n in (*t.shape, *t.stride()))


def _refuse(unless, message):
    if not unless:
        raise ValueError(message)


# The shapes of the outputs where sizes are symbols (traced with dynamic shapes): the C++ functions take numbers
def _group_norm_fwd_shapes(x, weight, bias, groups, eps, activation):
    _refuse(activation in ("none", "relu", "silu"), f"group_norm_act: activation is one of none, relu, silu, got {activation!r}")
    _refuse(x.dim() >= 2 and x.is_contiguous(), "group_norm_act: a contiguous channels-last tensor [N, ..., C]")
    _refuse(groups >= 1 and x.shape[-1] % groups == 0, f"group_norm_act: channels do not split into {groups} groups")
    for t in (weight, bias):
        _refuse(t is None or (t.dim() == 1 and t.shape[0] == x.shape[-1]), "group_norm_act: weight and bias have shape [C]")
    return x.new_empty(x.shape), x.new_empty((2, x.shape[0], groups), dtype=torch.float32)


def _group_norm_bwd_shapes(dy, x, weight, bias, stats, groups, activation):
    _group_norm_fwd_shapes(x, weight, bias, groups, 0.0, activation)
    _refuse(dy.shape == x.shape and dy.dtype == x.dtype and dy.is_contiguous(), "group_norm_act: dy is a contiguous tensor like x")
    c = (x.shape[-1],)
    return x.new_empty(x.shape), x.new_empty(c, dtype=torch.float32), x.new_empty(c, dtype=torch.float32)


def _like_logits(logits, k, dtype):
    """[N, k, ...] laid out as the logits' classes are: side by side, or as planes."""
    shape = (logits.shape[0], k, *logits.shape[2:])
    if logits.dim() > 2:
        side_by_side = logits.shape[1] > 1 and logits.stride(1) == 1 and logits.movedim(1, -1).is_contiguous()
        if side_by_side or all(n == 1 for n in logits.shape[2:]):
            return logits.new_empty((shape[0], *shape[2:], k), dtype=dtype).movedim(-1, 1)
    return logits.new_empty(shape, dtype=dtype)


def _class_log_probs_fwd_shapes(logits, target, top_k, ignore_index):
    _refuse(logits.dim() >= 2 and logits.shape[1] >= 1, "class_log_probs: logits have shape [N, C, ...] with at least one class")
    _refuse(0 <= top_k <= 32 and top_k <= logits.shape[1], f"class_log_probs: top_k lies between 0 and min(32, classes), got {top_k}")
    pos = (logits.shape[0], *logits.shape[2:])
    _refuse(target is None or (target.dtype == torch.int64 and target.shape == pos), "class_log_probs: int64 targets of shape [N, ...]")

    def f(*shape):
        return logits.new_empty(shape, dtype=torch.float32)
    return (f(0) if target is None else f(*pos)), f(*pos), f(2, *pos), _like_logits(logits, top_k, torch.float32), _like_logits(logits, top_k, torch.int64)


def _class_log_probs_bwd_shapes(logits, target, stats, entropy, top_indices, g_log_prob, g_entropy, g_top, ignore_index):
    _refuse(logits.dim() >= 2 and logits.shape[1] >= 1, "class_log_probs: logits have shape [N, C, ...] with at least one class")
    return _like_logits(logits, logits.shape[1], logits.dtype)


def _register(schema: str, impl, shapes):
    """The C++ function serves as the device kernel and as the fake kernel: on meta and fake tensors it launches nothing."""
    name = schema.split("(", 1)[0]

    def fake(*args):
        tensors = [t for t in args if isinstance(t, torch.Tensor)]
        if not _symbolic(*tensors):
            return impl(*args)
        if tensors[0].dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"{name}: float32 or bfloat16 tensors, got {tensors[0].dtype}")
        return shapes(*args)
    LIB.define(schema)
    LIB.impl(name, impl, "CUDA")
    torch.library.register_fake(f"{NS}::{name}", fake, lib=LIB)
    OPS.append(name)


_register("class_log_probs_fwd(Tensor logits, Tensor? target, int top_k, int ignore_index) -> (Tensor, Tensor, Tensor, Tensor, Tensor)",
          class_log_probs_fwd, _class_log_probs_fwd_shapes)
_register("class_log_probs_bwd(Tensor logits, Tensor? target, Tensor stats, Tensor entropy, Tensor top_indices, Tensor? g_log_prob, "
          "Tensor? g_entropy, Tensor? g_top, int ignore_index) -> Tensor", class_log_probs_bwd, _class_log_probs_bwd_shapes)
_register("group_norm_act_fwd(Tensor x, Tensor? weight, Tensor? bias, int groups, float eps, str activation) -> (Tensor, Tensor)",
          group_norm_act_fwd, _group_norm_fwd_shapes)
_register("group_norm_act_bwd(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, int groups, str activation) -> "
          "(Tensor, Tensor, Tensor)", group_norm_act_bwd, _group_norm_bwd_shapes)
