"""Restatement of the head norms with rotation, and of the step tables.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).  Rotation: the
reference's csrc/pos_encoding_kernels.cu:8-76; tables: the host lists of
flashinfer_attention_wrapper.py:75-209.
"""
from __future__ import annotations

import torch


def norm_rope(x, weight, eps, positions, cos_sin, neox):
    """(result, size) of heads x [T, heads, d] in float64; tokens whose position is
    outside the table as they are.  size: what an fp32 result's error goes with."""
    t, rot = x.shape[0], cos_sin.shape[1]
    y = x.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    inside = (positions >= 0) & (positions < cos_sin.shape[0])
    table = cos_sin.double()[torch.where(inside, positions, 0)][:, None]
    cos, sin = table[..., :rot // 2], table[..., rot // 2:]
    i = torch.arange(rot // 2)
    p, q = (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)
    out, size = y.clone(), y.abs()
    a, b = y[..., p], y[..., q]
    out[..., p] = a * cos - b * sin
    out[..., q] = b * cos + a * sin
    size[..., p] = size[..., q] = a.abs() + b.abs()
    keep = ~inside.view(t, 1, 1)
    return torch.where(keep, x.double(), out), torch.where(keep, torch.zeros_like(size), size)


def build(table, seq, new, page, free, height, num_tokens):
    """A step's arrays, walked request by request (lists; table and height in place)."""
    got = {k: [] for k in ("kv_indices", "kv_last_page_len", "batch_indices", "positions",
                           "slot_mapping")}
    got["append_indptr"], got["kv_indptr"] = [0], [0]
    for b, (n, q) in enumerate(zip(seq, new)):
        for k in range(-(-n // page), -(-(n + q) // page)):
            height -= 1
            table[b][k] = free[height]
        pages = table[b][:-(-(n + q) // page)]
        got["kv_indices"] += pages
        got["kv_indptr"].append(len(got["kv_indices"]))
        got["kv_last_page_len"].append((n + q - 1) % page + 1)
        for p in range(n, n + q):
            got["batch_indices"].append(b)
            got["positions"].append(p)
            got["slot_mapping"].append(pages[p // page] * page + p % page)
        got["append_indptr"].append(len(got["positions"]))
    for k in ("batch_indices", "positions", "slot_mapping"):
        got[k] += [-1] * (num_tokens - len(got[k]))
    return got, height
