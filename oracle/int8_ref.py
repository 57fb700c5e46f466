"""Restatement of the 8-bit projections in 64 bits.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).  The reference has no
kernel for them; the layer around them is models/llama.py:101-106, 176-178,
240-254.
"""
from __future__ import annotations

import math

import torch

LEAST_SCALE = 2.0 ** -126


def normed(x, weight, eps):
    """(rms_norm in float64, nothing rounded between)."""
    x = x.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()


def silu_mul(x):
    g, u = x.double().chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def scales_of(y):
    """A scale for each row of float64 y: NaN where the row is not finite."""
    top = y.abs().amax(-1)
    s = (top / 127).clamp_min(LEAST_SCALE)
    return torch.where(y.isfinite().all(-1), s, torch.full_like(s, math.nan))


def product(codes, weight):
    """Whole numbers: codes [T, K] times weight [N, K]."""
    return codes.double() @ weight.double().T


def linear(codes, token_scales, weight, channel_scales, bias=None, residual=None):
    y = product(codes, weight) * token_scales.double()[:, None] * channel_scales.double()
    if bias is not None:
        y = y + bias.double()
    if residual is not None:
        y = y + residual.double()
    return y


def gate_up_silu(codes, token_scales, weight, channel_scales):
    return silu_mul(linear(codes, token_scales, weight, channel_scales))
