"""Paged attention of one engine step, planned once and run for every layer.

``PagedAttention`` follows PaceServe's attention wrapper: ``begin_forward``
takes the step's host metadata (the append/KV index arrays that
paceserve/model_executor/attention/flashinfer_attention_wrapper.py:75-209
builds) and plans the work, ``forward`` runs one layer on the plan (:211-275).
Prompts, prompt chunks and single tokens share a plan.  Beyond causal
attention it takes capped scores, a distance bias (ALiBi), a sliding window, a
bidirectional prefix and packed documents; ``begin_tree_forward`` plans a
step whose new tokens are trees of drafted tokens.  The cache is the engine's
16-bit cache or a quantised one (codes and exponents, as
``kv_transfer_ops.append_quantised_paged_kv_cache`` writes it).

    attn = PagedAttention(num_heads, num_kv_heads, head_dim, page_size)
    attn.begin_forward(qo_indptr, kv_indptr, kv_indices, kv_last_page_len)
    for layer in layers:
        out = attn.forward(query, layer.cache)
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _C

attention_ops = _C.attention_ops


def _host_ints(x) -> torch.Tensor:
    if isinstance(x, torch.Tensor):
        return x.to(device="cpu", dtype=torch.int32).contiguous()
    return torch.tensor(list(x), dtype=torch.int32)


class PagedAttention:
    """Plans and runs the attention of one engine's steps on one GPU.

    The plan, its copy on the device and the workspace belong to the object: a
    new ``begin_forward`` replaces them, and calls of ``forward`` that may
    overlap on the GPU (several streams) need an object each.  A step that ran
    while a CUDA graph was captured is kept as long as the object, which has to
    outlive the graph.
    """

    def __init__(self, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
                 device: torch.device | str | int = "cuda"):
        self.num_heads = num_heads
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.page_size = page_size
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("PagedAttention: a CUDA device is needed")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self.num_sms = torch.cuda.get_device_properties(device).multi_processor_count
        self._scale = 1.0 / math.sqrt(head_dim)
        self._workspace = torch.zeros(0, dtype=torch.uint8, device=device)
        self._fault = torch.zeros(1, dtype=torch.int32, device=device)
        self._step = None
        self._captured = []  # steps whose memory a CUDA graph reads
        self.plan = None

    def begin_forward(self, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, *,
                      window_left: int = -1, prefix_lens=None, doc_starts=None) -> None:
        """Plan a step.  Sequences or int32 CPU tensors (a CUDA tensor is copied
        to the host, which waits for it): request b's new tokens are rows
        ``qo_indptr[b] .. qo_indptr[b + 1]`` of the query, the last of its
        sequence, whose pages are ``kv_indices[kv_indptr[b] .. kv_indptr[b + 1]]``
        with ``kv_last_page_len[b]`` tokens on the last one.

        ``window_left`` >= 0 hides keys more than that many tokens back;
        ``prefix_lens[b]`` keys at the sequence's start are seen by all its
        tokens; ``doc_starts[t]`` is the first position of new token t's own
        document, and hides what lies before.  A token left without keys gets
        zeros."""
        self._begin(qo_indptr, kv_indptr, kv_indices, kv_last_page_len, window_left=window_left,
                    prefix_lens=prefix_lens, doc_starts=doc_starts)

    def begin_tree_forward(self, qo_indptr, kv_indptr, kv_indices, kv_last_page_len,
                           tree_mask: torch.Tensor) -> None:
        """Plan a step whose new tokens are drafted: all of a request's are
        already appended to its sequence, and token t sees the sequence before
        them and those drafted tokens k of its own request whose bit k of
        ``tree_mask[t]`` is set (its ancestors and itself).  ``tree_mask``:
        int64 [tokens, words], 64 drafted tokens a word; on the host it may be
        changed afterwards, on the GPU the step reads it as it is."""
        if tree_mask.dim() != 2 or tree_mask.dtype != torch.int64 or tree_mask.shape[1] == 0:
            raise RuntimeError("begin_tree_forward: tree_mask must be int64 [tokens, words]")
        self._begin(qo_indptr, kv_indptr, kv_indices, kv_last_page_len, tree_mask=tree_mask)

    def _begin(self, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, *, window_left=-1,
               prefix_lens=None, doc_starts=None, tree_mask=None) -> None:
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("PagedAttention: plan the step before the CUDA graph is captured: "
                                   "a replay would copy the plan from host memory of this call")
        if self._step is not None and self._step.captured:
            self._captured.append(self._step)
        self._step = self.plan = None
        plan = attention_ops.plan_paged_attention(
            _host_ints(qo_indptr), _host_ints(kv_indptr), _host_ints(kv_indices),
            _host_ints(kv_last_page_len), self.num_heads, self.num_kv_heads, self.head_dim,
            self.page_size, window_left,
            None if prefix_lens is None else _host_ints(prefix_lens),
            None if doc_starts is None else _host_ints(doc_starts),
            0 if tree_mask is None else tree_mask.shape[1], self.num_sms)
        if tree_mask is not None and tree_mask.shape[0] != plan.total_q:
            raise RuntimeError("begin_tree_forward: tree_mask needs a row for each new token")
        with torch.cuda.device(self.device):
            if self._workspace.numel() < plan.workspace_bytes:
                self._workspace = torch.zeros(plan.workspace_bytes, dtype=torch.uint8,
                                              device=self.device)
            if tree_mask is not None:
                if tree_mask.is_pinned():  # its copy would read the caller's memory later
                    tree_mask = torch.empty(tree_mask.shape, dtype=torch.int64).copy_(tree_mask)
                tree_mask = tree_mask.to(self.device, non_blocking=True).contiguous()
            self._step = attention_ops.AttentionStep(
                plan, plan.words.to(self.device, non_blocking=True), self._workspace, tree_mask)
        self.plan = plan

    def forward(self, query: torch.Tensor, paged_kv_cache: torch.Tensor, *,
                exponents: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                logits_soft_cap: float = 0.0, alibi_slopes: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                fault_flags: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One layer's attention: ``query`` [tokens, num_heads, head_dim] (token
        rows may be strided views of the qkv projection) over the layer's cache
        [pages, 2, page_size, num_kv_heads, head_dim], or over a quantised
        cache's codes with its ``exponents``.  ``out`` must not overlap the
        query.  ``lse`` (float32 [tokens, num_heads]) receives each row's
        log-sum-exp.  Every wait in the kernels is bounded; one that runs out
        sets bit 30 of ``fault_flags`` (int32 on the device), or of the object's
        own flag, which ``check`` reads."""
        if self._step is None:
            raise RuntimeError("PagedAttention.forward: begin_forward has not planned a step")
        return self._step.forward(query, paged_kv_cache, exponents,
                                  self._scale if sm_scale is None else sm_scale, logits_soft_cap,
                                  alibi_slopes, out, lse,
                                  self._fault if fault_flags is None else fault_flags)

    def check(self) -> None:
        """Raise if a kernel's wait ran out in a ``forward`` since the last call:
        the outputs since then are undefined.  Waits for the current stream,
        which has to come after those calls.  Afterwards the object is as new."""
        if int(self._fault) == 0:
            return
        self._fault.zero_()
        self._workspace.zero_()
        raise RuntimeError("PagedAttention: a kernel wait ran out; the outputs since the last "
                           "check are undefined")
