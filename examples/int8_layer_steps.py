"""One decoder layer with 8-bit weights through an engine's steps, its page tables on the GPU.

    python -m examples.int8_layer_steps

The layer's four projections run on weights that were quantised once
(``quantise_weight``): the RMSNorm quantises the rows that enter them, a head's
norm, rotation and append to the cache are one pass, and the page tables and
slots come from the requests' lengths alone (``BlockTables``).  Two requests
share the steps: a prompt in two chunks, single tokens, and drafted tokens of
which some are not accepted.  The layer is PaceServe's with norms of queries and
keys added (paceserve/model_executor/models/llama.py:147-260).
"""
from __future__ import annotations

import torch

from paceserve_b200 import int8_ops, pos_encoding_ops, quantise_weight
from paceserve_b200.attention import PagedAttention
from paceserve_b200.block_tables import BlockTables

HIDDEN, HEADS, KV_HEADS, HEAD_DIM, INTER, PAGE, EPS = 1024, 16, 4, 64, 2048, 16, 1e-5


class Layer:
    """Weights, in 16 bits for the norms and in 8 for the projections, and the layer's cache."""

    def __init__(self, pages: int, device: str, g: torch.Generator):
        rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().to(device)  # noqa: E731
        norm = lambda n: (1 + torch.randn(n, generator=g) / 8).bfloat16().to(device)  # noqa: E731
        q, kv = HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM
        self.input_norm, self.post_norm = norm(HIDDEN), norm(HIDDEN)
        self.q_norm, self.k_norm = norm(HEAD_DIM), norm(HEAD_DIM)
        self.qkv = quantise_weight(rnd(q + 2 * kv, HIDDEN) / HIDDEN ** 0.5)
        self.out = quantise_weight(rnd(HIDDEN, q) / q ** 0.5)
        self.gate_up = quantise_weight(rnd(2 * INTER, HIDDEN) / HIDDEN ** 0.5)
        self.down = quantise_weight(rnd(HIDDEN, INTER) / INTER ** 0.5)
        self.cache = torch.zeros(pages, 2, PAGE, KV_HEADS, HEAD_DIM, dtype=torch.bfloat16, device=device)
        angle = torch.arange(2048, dtype=torch.float64)[:, None] \
            * 10000.0 ** (-torch.arange(0, HEAD_DIM, 2, dtype=torch.float64) / HEAD_DIM)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().to(device)
        # a bit is set in it if a kernel's bounded wait runs out, whose output is then undefined
        self.fault = torch.zeros(1, dtype=torch.int32, device=device)

    def check(self) -> None:
        """Raise if a call since the last one gave up; where the engine waits for the GPU anyway."""
        if int(self.fault):
            self.fault.zero_()
            raise RuntimeError("a kernel's wait ran out: the steps' outputs are undefined")


def _codes(rows: int, width: int, device):
    return (torch.empty(rows, width, dtype=torch.int8, device=device),
            torch.empty(rows, dtype=torch.float32, device=device))


def forward(layer: Layer, hidden: torch.Tensor, step, attention: PagedAttention, seen: dict | None = None):
    """The layer on `hidden` [tokens, HIDDEN], the residual stream, in place.  `seen` gets what each
    operator was given and made, for a check."""
    t, dev = hidden.shape[0], hidden.device
    note = (lambda **kw: seen.update({k: v.clone() for k, v in kw.items()})) if seen is not None else (lambda **kw: None)
    empty = lambda n: torch.empty(t, n, dtype=hidden.dtype, device=dev)  # noqa: E731

    codes, scales = _codes(t, HIDDEN, dev)
    note(hidden=hidden)
    int8_ops.rms_norm_quantise(codes, scales, hidden, layer.input_norm, EPS)
    q_size, kv_size = HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM
    qkv = empty(q_size + 2 * kv_size)
    int8_ops.linear(qkv, codes, scales, *layer.qkv, fault_flags=layer.fault)
    note(in_codes=codes, in_scales=scales, qkv=qkv)
    query, key, value = qkv.split([q_size, kv_size, kv_size], 1)
    pos_encoding_ops.qk_norm_rotary_append(step.positions, query, key, value, layer.q_norm, layer.k_norm, EPS,
                                           HEAD_DIM, layer.cos_sin, True, layer.cache, step.slot_mapping,
                                           fault_flags=layer.fault)
    attended = attention.forward(query.view(t, HEADS, HEAD_DIM), layer.cache).view(t, q_size)
    note(query=query, attended=attended)

    codes, scales = _codes(t, q_size, dev)
    int8_ops.quantise_rows(codes, scales, attended)
    int8_ops.linear_residual(hidden, codes, scales, *layer.out, fault_flags=layer.fault)
    note(out_codes=codes, out_scales=scales, middle=hidden)

    codes, scales = _codes(t, HIDDEN, dev)
    int8_ops.rms_norm_quantise(codes, scales, hidden, layer.post_norm, EPS)
    act = empty(INTER)
    int8_ops.gate_up_silu(act, codes, scales, *layer.gate_up, fault_flags=layer.fault)
    note(post_codes=codes, post_scales=scales, act=act)
    codes, scales = _codes(t, INTER, dev)
    int8_ops.quantise_rows(codes, scales, act)
    int8_ops.linear_residual(hidden, codes, scales, *layer.down, fault_flags=layer.fault)
    note(act_codes=codes, act_scales=scales, result=hidden)
    return hidden


def main(device: str = "cuda:0", pages: int = 64, seed: int = 0):
    """Runs the steps; returns the layer, the tables and what each step saw, for a check."""
    g = torch.Generator().manual_seed(seed)
    layer = Layer(pages, device, g)
    tables = BlockTables(2, 32, PAGE, pages, 256, device)
    attention = PagedAttention(HEADS, KV_HEADS, HEAD_DIM, PAGE, device)
    lens, done = [0, 0], []
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731

    def run(new):
        tokens = sum(new)
        step = tables.begin_step(ints(lens), ints(new))
        # the plan is the host's: it takes the tables back
        attention.begin_forward(step.append_indptr, step.kv_indptr, step.kv_indices, step.kv_last_page_len)
        hidden = torch.randn(tokens, HIDDEN, generator=g).bfloat16().to(device)
        seen = {"lens": list(lens), "new": list(new)}
        forward(layer, hidden, step, attention, seen)
        seen["tables"] = [x.clone() for x in step]
        seen["cache"] = layer.cache.clone()
        done.append(seen)
        for b, n in enumerate(new):
            lens[b] += n

    run([150, 0])               # a first prompt chunk
    run([61, 1])                # the rest beside another request's token
    run([1, 1])                 # single tokens
    run([7, 6])                 # drafted tokens, of which two and none are accepted
    kept = [lens[0] - 5, lens[1] - 6]
    tables.release(ints(lens), ints(kept))
    lens[:] = kept
    run([1, 1])
    tables.release(ints(lens), ints([0, lens[1]]))  # the first request is done
    lens[0] = 0
    run([33, 1])                # another takes its row
    tables.check()
    layer.check()
    attention.check()
    return layer, tables, done


if __name__ == "__main__":
    _, tables, steps = main()
    torch.cuda.synchronize()
    for s in steps:
        print(f"{sum(s['new']):4d} tokens  out {tuple(s['result'].shape)}  "
              f"mean |out| {s['result'].float().abs().mean().item():.4f}")
    print(f"free pages {tables.free_count.item()}")
