"""Modules over `group_norm` and `dropout`.

Batch statistics are of little use at the 4 to 8 images per GPU that the
training configurations hold; a group norm's are a sample's own, and the same
in training and inference.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from .functional import _act_code, dropout, group_norm


class GroupNormAct(nn.Module):
    """Group norm + affine + activation, and dropout while training, of
    channels-last features in one operator.

    groups: the largest common divisor of 32 and the channels unless given.
    """

    def __init__(self, channels: int, act: str | None = None,
                 groups: int | None = None, eps: float = 1e-5,
                 dropout: float = 0.0):
        super().__init__()
        self.groups = math.gcd(32, channels) if groups is None else groups
        if channels < 1 or self.groups < 1 or channels % self.groups:
            raise ValueError(f"{channels} channels in {self.groups} groups")
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"dropout probability must lie in [0, 1], got "
                             f"{dropout}")
        _act_code(act)  # refuses what is none
        self.act, self.eps, self.dropout = act, eps, dropout
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels))

    def forward(self, x):
        return group_norm(x, self.groups, self.weight, self.bias, self.eps,
                          self.act, self.dropout if self.training else 0.0)

    def extra_repr(self):
        return (f"{self.weight.numel()}, groups={self.groups}, act={self.act}, "
                f"eps={self.eps}, dropout={self.dropout}")


class CounterDropout(nn.Module):
    """Activation, and dropout behind it while training, with a mask from a
    counter-based generator.

    The mask is never stored: the way back computes it again from the two
    numbers that a pass draws from torch's generator.
    """

    def __init__(self, p: float = 0.5, act: str | None = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
        _act_code(act)  # refuses what is none
        self.p, self.act = p, act

    def forward(self, x):
        return dropout(x, self.p if self.training else 0.0, act=self.act)

    def extra_repr(self):
        return f"p={self.p}, act={self.act}"
