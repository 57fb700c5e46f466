"""CPU: what paged attention plans and refuses where arguments are at an edge."""
import ctypes

import pytest
import torch

from paceserve_b200 import attention_ops, cabi


def ints(*v):
    return (ctypes.c_int32 * len(v))(*v)


def plan_c(lib, q, pages, page=16, last=7, heads=8, kv_heads=2, head_dim=128):
    """(plan, words) of one request, through the C entry point."""
    plan = cabi.AttentionPlan()
    n = lib.pace_paged_attention_plan_words(1, q, pages, 148)
    words = (ctypes.c_int32 * n)()
    assert lib.pace_paged_attention_plan(
        ctypes.byref(plan), words, n, ints(0, q), ints(0, pages), ints(*range(pages)), pages,
        ints(last), 1, heads, kv_heads, head_dim, page, -1, None, None, 0, 148) == cabi.PACE_OK
    return plan, words


def test_workspace_alignment_is_checked():
    """A prompt that is cut leaves partial rows in the workspace, 32 bytes at a time."""
    lib = cabi.load()
    plan, _ = plan_c(lib, 70, 2000)
    assert plan.many_slots > 0

    def run(workspace, nbytes=plan.workspace_bytes):
        return lib.pace_paged_attention(ctypes.byref(plan), 16, 16, 16, 1024, 1024, 16, None, 2000,
                                        1.0, 0.0, None, None, None, workspace, nbytes, None,
                                        cabi.PACE_BF16, None)

    for args in ((4096 + 16,), (4096 + 8,), (4096, plan.workspace_bytes - 1), (None,)):
        assert run(*args) == cabi.PACE_ERR_INVALID_ARGUMENT, args
        assert b"32-byte aligned workspace" in lib.pace_last_error()


def test_every_piece_of_a_tree_may_hide_keys():
    """Also a tree of one node: its own bit may be clear, and its key is in its piece."""
    ints32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    for heads, words in ((8, 1), (64, 2)):
        plan = attention_ops.plan_paged_attention(ints32(0, 1, 4), ints32(0, 2, 4), ints32(0, 1, 2, 3),
                                                  ints32(5, 16), heads, 2, 128, 16, tree_words=words)
        at = 4 * plan.total_q
        items = [plan.words[at + 12 * i:at + 12 * i + 12].tolist()
                 for i in range(plan.num_few + plan.num_many)]
        assert len(items) == 2 and all(w[9] == 1 for w in items)


def test_entries_of_no_request_are_not_looked_at():
    """kv_indices of a fixed size, filled up with -1 or whatever was there: only the entries
    between the first and the last kv_indptr name pages."""
    ints32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    call = attention_ops.plan_paged_attention
    rest = (ints32(5, 16), 8, 2, 128, 16)
    plan = call(ints32(0, 1, 4), ints32(1, 3, 5), ints32(-1, 0, 7, 2, 3, -1, 1 << 30), *rest)
    assert plan.words.tolist()[-7:] == [-1, 0, 7, 2, 3, -1, 1 << 30]
    for bad in (1, 4):
        indices = ints32(-1, 0, 7, 2, 3, -1, 1 << 30)
        indices[bad] = -1
        with pytest.raises(RuntimeError, match="negative page"):
            call(ints32(0, 1, 4), ints32(1, 3, 5), indices, *rest)
    lib = cabi.load()
    c_plan = cabi.AttentionPlan()
    n = lib.pace_paged_attention_plan_words(1, 1, 3, 148)
    words = (ctypes.c_int32 * n)()
    assert lib.pace_paged_attention_plan(ctypes.byref(c_plan), words, n, ints(0, 1), ints(0, 1),
                                         ints(4, -1, 99), 3, ints(2), 1, 8, 2, 128, 16, -1, None, None,
                                         0, 148) == cabi.PACE_OK
    assert c_plan.max_page == 4
