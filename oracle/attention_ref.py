"""Restatement of the paged-attention operators in 64 bits.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).

The reference runs attention through FlashInfer's paged wrappers
(paceserve/model_executor/attention/flashinfer_attention_wrapper.py:165-188,
245-275; FlashInfer is not vendored).  Restated here from the definition, on
the CPU in float64: masked keys and values do not enter a row, whatever they
hold.
"""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


# ------------------------------------------------------ quantised rows --
def e4m3_value(code: int) -> float:
    """The value of an e4m3 code: sign, 4 exponent bits (bias 7), 3 mantissa bits."""
    sign = -1.0 if code & 0x80 else 1.0
    e, m = code >> 3 & 15, code & 7
    if e == 15 and m == 7:
        return math.nan
    return sign * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))


E4M3_VALUES = torch.tensor([e4m3_value(c) for c in range(256)], dtype=torch.float64)


def quantise_row(x: torch.Tensor):
    """(codes uint8, exponent byte) of one row of floats."""
    most = torch.finfo(x.dtype).max
    x = x.double()
    if bool(x.isnan().any()):
        return torch.zeros(x.shape, dtype=torch.uint8), 255
    finite = x[x.isfinite()].abs()
    top = float(finite.max()) if finite.numel() else 0.0
    e = 0 if bool(x.isinf().any()) else -126
    if top > 0:
        m, k = math.frexp(top)  # top = m * 2^k, 448 = 0.875 * 2^9
        e = max(k - 9 + (1 if m > 0.875 else 0), -126)
    y = (x * 2.0 ** -e).clamp(-E4M3_MAX, E4M3_MAX)
    # nearest of the 127 finite magnitudes; a tie goes to the even code
    grid = E4M3_VALUES[:127]
    hi = torch.searchsorted(grid, y.abs()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = y.abs() - grid[lo], grid[hi] - y.abs()
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    # what is finite in its type stays so
    code = torch.where(x.isfinite() & (grid[code] * 2.0 ** e > most), code - 1, code)
    return (code + 128 * torch.signbit(y).long()).to(torch.uint8), e + 127


def dequantise(codes: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    """float64 values of codes (uint8) with exponents (one fewer axis)."""
    v = E4M3_VALUES[codes.long()] * torch.exp2(exponents.double() - 127)[..., None]
    return torch.where((exponents == 255)[..., None], torch.full_like(v, math.nan), v)


def append_quantised(key, value, append_indptr, codes, exponents, kv_indices, kv_indptr,
                     kv_last_page_len):
    """In place on CPU tensors codes (uint8) and exponents."""
    page_size, heads, hd = codes.shape[2:]
    for b in range(len(append_indptr) - 1):
        t0, t1 = int(append_indptr[b]), int(append_indptr[b + 1])
        pages = kv_indices[int(kv_indptr[b]):int(kv_indptr[b + 1])].tolist()
        n = (len(pages) - 1) * page_size + int(kv_last_page_len[b])
        for t in range(t0, t1):
            pos = n - t1 + t
            for kind, x in enumerate((key, value)):
                for h in range(heads):
                    row = x.reshape(x.shape[0], heads, hd)[t, h]
                    c, e = quantise_row(row)
                    codes[pages[pos // page_size], kind, pos % page_size, h] = c
                    exponents[pages[pos // page_size], kind, pos % page_size, h] = e


# ------------------------------------------------------------- attention --
def gather_rows(cache, kv_indices, kv_indptr, kv_last_page_len, b):
    """(K, V) of request b in sequence order, [kv_len, kv_heads, hd]."""
    page_size = cache.shape[2]
    pages = kv_indices[int(kv_indptr[b]):int(kv_indptr[b + 1])].long()
    if pages.numel() == 0:
        empty = cache.new_zeros((0,) + tuple(cache.shape[3:]))
        return empty, empty
    n = (pages.numel() - 1) * page_size + int(kv_last_page_len[b])
    rows = cache[pages]  # [np, 2, ps, heads, hd]
    flat = rows.permute(1, 0, 2, 3, 4).reshape(2, -1, *cache.shape[3:])
    return flat[0, :n], flat[1, :n]


def visible(q_len, kv_len, window_left=-1, prefix=0, doc_starts=None, tree_mask=None):
    """[q_len, kv_len] truth values."""
    pos = torch.arange(kv_len - q_len, kv_len)[:, None]
    j = torch.arange(kv_len)[None]
    if tree_mask is not None:
        base = kv_len - q_len
        see = (j < base).expand(q_len, kv_len).clone()
        for i in range(q_len):
            for k in range(q_len):
                if int(tree_mask[i, k // 64]) >> (k % 64) & 1:
                    see[i, base + k] = True
        return see
    see = (j <= pos) | (j < prefix)
    if window_left >= 0:
        see &= j >= pos - window_left
    if doc_starts is not None:
        see &= j >= doc_starts[:, None].long()
    return see


def attention(query, cache, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, sm_scale,
              soft_cap=0.0, slopes=None, window_left=-1, prefix_lens=None, doc_starts=None,
              tree_mask=None):
    """(out float64 [tokens, heads, hd], lse float64 [tokens, heads]); cache any
    float type (a quantised one dequantised first)."""
    tokens, heads, hd = query.shape
    kv_heads = cache.shape[3]
    out = torch.zeros(tokens, heads, hd, dtype=torch.float64)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    for b in range(len(qo_indptr) - 1):
        t0, t1 = int(qo_indptr[b]), int(qo_indptr[b + 1])
        if t1 == t0:
            continue
        k, v = (x.double() for x in gather_rows(cache, kv_indices, kv_indptr, kv_last_page_len, b))
        n = k.shape[0]
        see = visible(t1 - t0, n, window_left, int(prefix_lens[b]) if prefix_lens is not None else 0,
                      None if doc_starts is None else doc_starts[t0:t1],
                      None if tree_mask is None else tree_mask[t0:t1])
        for h in range(heads):
            kh, vh = k[:, h * kv_heads // heads], v[:, h * kv_heads // heads]
            s = query[t0:t1, h].double() @ kh.T * sm_scale
            if soft_cap:
                s = soft_cap * torch.tanh(s / soft_cap)
            if slopes is not None:
                pos = torch.arange(n - (t1 - t0), n)[:, None]
                s = s - slopes[h].double() * (pos - torch.arange(n)[None]).abs()
            if bool(s.isfinite().all()) and bool(vh.isfinite().all()):
                s = s.masked_fill(~see, -math.inf)
                some = see.any(1)
                lse[t0:t1, h] = torch.logsumexp(s, 1)
                out[t0:t1, h][some] = torch.softmax(s[some], 1) @ vh
                continue
            for i in range(t1 - t0):  # what is masked must not enter a product either
                sel = see[i]
                if not bool(sel.any()):
                    continue
                lse[t0 + i, h] = torch.logsumexp(s[i, sel], 0)
                out[t0 + i, h] = torch.softmax(s[i, sel], 0) @ vh[sel]
    return out, lse
