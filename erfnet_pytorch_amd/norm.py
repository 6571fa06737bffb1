"""Group normalisation with an activation on channels-last maps: statistics per image and group of channels, so neither the
number of images per GPU nor running averages matter (train/erfnet.py uses BatchNorm2d, which couples the images of a batch).

`GroupNormAct2d` stands where a BatchNorm2d + ReLU pair stands in the reference's blocks (train/erfnet.py:20-22,60-62): logical
[N,C,H,W] in and out, channels_last memory as everywhere in this package.
"""
from __future__ import annotations

import torch
from torch import nn

from .train_ops import _host

ACTIVATIONS = ("none", "relu", "silu")


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, activation="relu"):
    """act((x - mean) / sqrt(var + eps) * weight + bias), mean and variance over each image's positions and C / num_groups
    neighbouring channels.

    x [N, C, ...] fp32 or bf16, read where it lies if its memory is channels-last, else copied; the result has x's type and
    channels-last memory.  weight, bias [C] or None; statistics and parameter gradients are fp32.  activation: "none", "relu" or
    "silu".  Differentiable (once) in x, weight and bias."""
    return _host.group_norm_act(x, num_groups, weight, bias, eps, activation)


class GroupNormAct2d(nn.Module):
    """nn.GroupNorm (same constructor order, same state_dict keys) followed by an activation."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation="relu"):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups:
            raise ValueError(f"num_channels ({num_channels}) is a multiple of num_groups ({num_groups})")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation is one of {ACTIVATIONS}, got {activation!r}")
        self.num_groups, self.num_channels, self.eps, self.affine, self.activation = num_groups, num_channels, eps, affine, activation
        if affine:
            self.weight, self.bias = nn.Parameter(torch.ones(num_channels)), nn.Parameter(torch.zeros(num_channels))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, input):
        return group_norm_act(input, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self):
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.affine}, activation={self.activation!r}"
