"""Block tables and a step's index arrays, kept on the GPU.

``BlockTables`` holds, for up to ``max_requests`` rows, each request's pages in
sequence order and the stack of pages that nobody has.  ``begin_step`` takes the
pages that a step's new tokens need and builds, from the lengths alone and in
one launch, what PaceServe's attention wrapper builds on the host
(paceserve/model_executor/attention/flashinfer_attention_wrapper.py:75-209): the
append and KV index arrays, and each new token's request, position and slot.

    tables = BlockTables(max_requests, max_blocks, page_size, num_pages, max_tokens)
    step = tables.begin_step(seq_lens, new_lens)
    for layer in layers:
        pos_encoding_ops.qk_norm_rotary_append(step.positions, q, k, v, ..., layer.cache,
                                               step.slot_mapping)
    tables.release(held_lens, kept_lens)       # drafts not accepted, requests that are done
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _C

kv_transfer_ops = _C.kv_transfer_ops

MAX_REQUESTS = 8192  # of a step: their prefix sums are in one CTA's shared memory

PROBLEMS = {1: "a length is negative, or more tokens are kept than held",
            2: "a request needs more pages than its row holds",
            4: "the step needs more pages than kv_indices holds",
            8: "the step has more new tokens than max_tokens",
            16: "there are not enough free pages, or more are given back than there are"}


class StepTables(NamedTuple):
    """One step's arrays: views of the object's, which the next step overwrites.
    Token entries past the step's last token are -1."""

    append_indptr: torch.Tensor
    kv_indptr: torch.Tensor
    kv_indices: torch.Tensor
    kv_last_page_len: torch.Tensor
    batch_indices: torch.Tensor
    positions: torch.Tensor
    slot_mapping: torch.Tensor


class BlockTables:
    """Row b of a step's lengths is row b of ``block_tables``: a request keeps its
    row while it lives, and a row without a request has lengths of 0.  There are
    at most ``MAX_REQUESTS`` rows.  Calls belong to one stream (or are ordered by
    the caller) and may be captured into a CUDA graph, which then reads the
    lengths' tensors anew at each replay."""

    def __init__(self, max_requests: int, max_blocks: int, page_size: int, num_pages: int,
                 max_tokens: int, device: torch.device | str | int = "cuda"):
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("BlockTables: a CUDA device is needed")
        if min(max_requests, max_blocks, page_size, num_pages, max_tokens) < 1:
            raise RuntimeError("BlockTables: all sizes must be positive")
        if max_requests > MAX_REQUESTS:
            raise RuntimeError(f"BlockTables: at most {MAX_REQUESTS} requests, not {max_requests}")
        if max(max_requests * max_blocks, num_pages, max_tokens) >= 1 << 31:
            raise RuntimeError("BlockTables: sizes past 32 bits")
        ints = lambda *n, kind=torch.int32: torch.zeros(*n, dtype=kind, device=device)  # noqa: E731
        self.page_size = page_size
        self.block_tables = ints(max_requests, max_blocks)
        # page 0 is taken first
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)
        self._step = StepTables(ints(max_requests + 1), ints(max_requests + 1),
                                ints(min(max_requests * max_blocks, num_pages)), ints(max_requests),
                                ints(max_tokens), ints(max_tokens, kind=torch.int64),
                                ints(max_tokens, kind=torch.int64))
        self._status, self._arrivals = ints(1), ints(1)

    def begin_step(self, seq_lens: torch.Tensor, new_lens: torch.Tensor) -> StepTables:
        """Take pages for ``new_lens[b]`` tokens after the ``seq_lens[b]`` that
        request b has (int32 on the device, one entry for each row in use) and
        build the step's arrays.  A step that does not fit takes nothing, leaves
        every token entry at -1 and shows in ``check``; until then all later steps
        and releases do the same, whatever their lengths."""
        s, n = self._step, seq_lens.numel()
        if n > self.block_tables.shape[0]:
            raise RuntimeError("BlockTables.begin_step: more lengths than rows")
        kv_transfer_ops.build_step_tables(
            self.block_tables, seq_lens, new_lens, self.page_size, self.free_pages, self.free_count,
            s.append_indptr, s.kv_indptr, s.kv_indices, s.kv_last_page_len, s.batch_indices,
            s.positions, s.slot_mapping, self._status, self._arrivals)
        return s._replace(append_indptr=s.append_indptr[:n + 1], kv_indptr=s.kv_indptr[:n + 1],
                          kv_last_page_len=s.kv_last_page_len[:n])

    def release(self, held_lens: torch.Tensor, kept_lens: torch.Tensor) -> None:
        """Give back the pages past the first ``kept_lens[b]`` of request b's
        ``held_lens[b]`` tokens: 0 for a request that is done."""
        kv_transfer_ops.release_pages(self.block_tables, held_lens, kept_lens, self.page_size,
                                      self.free_pages, self.free_count, self._status,
                                      self._arrivals)

    def check(self) -> None:
        """Raise if a step or a release since the last call did not fit.  Waits
        for the current stream, which has to come after those calls.

        From that step or release on nothing was taken, given or written to.  Go on
        with the lengths that the last step that fitted left (lengths that moved on
        since count pages that their requests were not given), and make the
        releases since then again."""
        bits = int(self._status)
        if bits:
            self._status.zero_()
            raise RuntimeError("BlockTables: " + "; ".join(
                text for bit, text in PROBLEMS.items() if bits & bit))
