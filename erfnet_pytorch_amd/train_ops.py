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


def _register(schema: str, impl):
    """The same function serves as the device kernel and as the fake kernel: on meta and fake tensors it launches nothing."""
    name = schema.split("(", 1)[0]
    LIB.define(schema)
    LIB.impl(name, impl, "CUDA")
    torch.library.register_fake(f"{NS}::{name}", impl, lib=LIB)
    OPS.append(name)


_register("class_log_probs_fwd(Tensor logits, Tensor? target, int top_k, int ignore_index) -> (Tensor, Tensor, Tensor, Tensor, Tensor)",
          class_log_probs_fwd)
_register("class_log_probs_bwd(Tensor logits, Tensor? target, Tensor stats, Tensor entropy, Tensor top_indices, Tensor? g_log_prob, "
          "Tensor? g_entropy, Tensor? g_top, int ignore_index) -> Tensor", class_log_probs_bwd)
_register("group_norm_act_fwd(Tensor x, Tensor? weight, Tensor? bias, int groups, float eps, str activation) -> (Tensor, Tensor)",
          group_norm_act_fwd)
_register("group_norm_act_bwd(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, int groups, str activation) -> "
          "(Tensor, Tensor, Tensor)", group_norm_act_bwd)
