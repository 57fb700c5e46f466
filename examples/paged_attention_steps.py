"""The attention of one decoder layer through an engine's steps, over a quantised cache.

    python -m examples.paged_attention_steps

A prompt is appended and attended to in two chunks, one of them beside another
request's single token (a mixed step); single tokens follow; then a tree of
drafted tokens is verified in one step; and the request's keys and values are
read back in sequence order.  Every step runs the way PaceServe's attention
wrapper does: begin_forward once a step, then append and forward for each layer
(paceserve/model_executor/attention/flashinfer_attention_wrapper.py:75-275).
"""
from __future__ import annotations

import torch

from paceserve_b200 import kv_transfer_ops as kv
from paceserve_b200.attention import PagedAttention

HEADS, KV_HEADS, HEAD_DIM, PAGE = 32, 8, 128, 16


class Requests:
    """Page tables of a few requests over one pool of pages, as the block manager keeps them."""

    def __init__(self, pages: int):
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(0)).tolist()
        self.pages: dict[str, list[int]] = {}
        self.length: dict[str, int] = {}

    def grow(self, name: str, tokens: int) -> None:
        self.length[name] = self.length.get(name, 0) + tokens
        table = self.pages.setdefault(name, [])
        while len(table) * PAGE < self.length[name]:
            table.append(self.free.pop())

    def metadata(self, new_tokens: dict[str, int]):
        """(qo_indptr, kv_indptr, kv_indices, kv_last_page_len) of a step that adds these tokens."""
        for name, n in new_tokens.items():
            self.grow(name, n)
        names = list(new_tokens)
        ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
        return (ints([0] + [new_tokens[n] for n in names]).cumsum(0).int(),
                ints([0] + [len(self.pages[n]) for n in names]).cumsum(0).int(),
                ints([p for n in names for p in self.pages[n]]),
                ints([(self.length[n] - 1) % PAGE + 1 for n in names]))


def main(device: str = "cuda:0", pages: int = 256, seed: int = 0):
    """Runs the steps; returns what each computed, for a check."""
    g = torch.Generator().manual_seed(seed)
    requests = Requests(pages)
    shape = (pages, 2, PAGE, KV_HEADS, HEAD_DIM)
    codes = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    exponents = torch.zeros(shape[:-1], dtype=torch.uint8, device=device)
    attention = PagedAttention(HEADS, KV_HEADS, HEAD_DIM, PAGE, device)
    done = []

    def step(new_tokens: dict[str, int], tree_mask=None, **options):
        meta = requests.metadata(new_tokens)
        tokens = int(meta[0][-1])
        qkv = torch.randn(tokens, (HEADS + 2 * KV_HEADS) * HEAD_DIM, generator=g).bfloat16().to(device)
        query, key, value = qkv.split([HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM], 1)
        if tree_mask is None:
            attention.begin_forward(*meta)
        else:
            attention.begin_tree_forward(*meta, tree_mask)
        # for each layer:
        kv.append_quantised_paged_kv_cache(key, value, meta[0].to(device), codes, exponents,
                                           meta[2].to(device), meta[1].to(device), meta[3].to(device))
        out = attention.forward(query.view(tokens, HEADS, HEAD_DIM), codes, exponents=exponents,
                                **options)
        done.append({"meta": meta, "query": query.view(tokens, HEADS, HEAD_DIM), "out": out,
                     "tree_mask": tree_mask, "options": options,
                     "codes": codes.view(torch.uint8).clone(), "exponents": exponents.clone()})
        return out

    step({"a": 300}, logits_soft_cap=50.0)                      # a first prompt chunk
    step({"a": 211, "b": 1}, logits_soft_cap=50.0)              # the rest beside another's token
    for _ in range(3):
        step({"a": 1, "b": 1}, logits_soft_cap=50.0)            # single tokens
    # a tree of five drafted tokens: 0 - 1 - 2, 1 - 3, 0 - 4
    mask = torch.tensor([0b00001, 0b00011, 0b00111, 0b01011, 0b10001], dtype=torch.int64)[:, None]
    step({"a": 5}, tree_mask=mask)
    attention.check()
    # request a's rows, in sequence order
    _, kp, ki, kl = requests.metadata({"a": 0})
    n = requests.length["a"]
    key = torch.empty(n, KV_HEADS, HEAD_DIM, dtype=torch.bfloat16, device=device)
    value = torch.empty_like(key)
    kv.read_quantised_paged_kv_cache(key, value, torch.tensor([0, n], dtype=torch.int32, device=device),
                                     codes, exponents, ki.to(device), kp.to(device), kl.to(device))
    return done, {"key": key, "value": value, "kv_indptr": kp, "kv_indices": ki, "kv_last_page_len": kl}


if __name__ == "__main__":
    steps, rows = main()
    torch.cuda.synchronize()
    for s in steps:
        print(f"{s['out'].shape[0]:4d} tokens  out {tuple(s['out'].shape)}  "
              f"mean |out| {s['out'].float().abs().mean().item():.4f}")
    print(f"read back {tuple(rows['key'].shape)} keys and values")
