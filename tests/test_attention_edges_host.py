"""CPU: what paged attention plans and refuses where arguments are at an edge."""
import ctypes

from paceserve_b200 import cabi


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
