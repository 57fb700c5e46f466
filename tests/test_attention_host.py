"""CPU: the plan of paged attention covers every visible key of every row once,
and refuses metadata that no kernel may read."""
import ctypes

import pytest
import torch

from oracle import attention_ref as ref
from paceserve_b200 import attention_ops, cabi, kv_transfer_ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def meta(lens, page):
    n = [-(-x // page) for _, x in lens]
    return (torch.tensor([0] + [q for q, _ in lens]).cumsum(0).int(),
            torch.tensor([0] + n).cumsum(0).int(), torch.arange(sum(n)).int().flip(0),
            torch.tensor([(x - 1) % page + 1 if x else 1 for _, x in lens]).int())


def records(plan, lens, heads, kv_heads, page):
    """(token records, items) of a plan's words."""
    words = plan.words.tolist()
    tokens = [words[4 * i:4 * i + 4] for i in range(plan.total_q)]
    at, items = 4 * plan.total_q, []
    for _ in range(plan.num_few + plan.num_many):
        items.append(words[at:at + 12])
        at += 12
    assert words[at:] == meta(lens, page)[2].tolist()
    return tokens, items


@pytest.mark.parametrize("kw", [{}, {"window_left": 0}, {"window_left": 100},
                                {"prefix": 50, "window_left": 300}, {"docs": True}, {"tree": 2}])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (3, 1), (16, 16), (128, 1)])
def test_plan_covers_every_visible_key_once(kw, heads, kv_heads):
    page = 16
    lens = [(1, 5000), (1, 1), (0, 9), (100, 700), (128, 128), (3, 40), (1, 0)]
    if not kw.get("tree"):
        lens += [(700, 2000), (9, 4)]
    qp, kp, ki, kl = meta(lens, page)
    t = int(qp[-1])
    prefix = i32([kw["prefix"]] * len(lens)) if "prefix" in kw else None
    docs = None
    if kw.get("docs"):
        docs = torch.randint(0, 900, (t,), generator=torch.Generator().manual_seed(1)).int()
    if kw.get("tree"):
        lens[-1] = (1, 1)
        qp, kp, ki, kl = meta(lens, page)
    plan = attention_ops.plan_paged_attention(
        qp, kp, ki, kl, heads, kv_heads, 128, page, kw.get("window_left", -1), prefix, docs,
        kw.get("tree", 0))
    tokens, items = records(plan, lens, heads, kv_heads, page)
    seen = {i: set() for i in range(plan.total_q)}
    slots = set()
    for n, (tok0, ntok, k0, k1, page_base, tile, slot, split, splits, *_) in enumerate(items):
        few = n < plan.num_few
        assert ntok * (heads // kv_heads) <= (16 if few else 256)
        assert 0 <= split < splits
        if splits > 1:
            key = (few, slot + split)
            assert key not in slots and slot + split < (plan.few_slots if few else plan.many_slots)
            slots.add(key)
        for i in range(tok0, tok0 + ntok):
            assert page_base == tokens[i][2]
            keys = set(range(k0, k1))
            assert not keys & seen[i]
            seen[i] |= keys
    for b, (q, n) in enumerate(lens):
        see = ref.visible(q, n, kw.get("window_left", -1), kw.get("prefix", 0),
                          None if docs is None else docs[int(qp[b]):int(qp[b + 1])],
                          torch.full((q, kw["tree"]), -1) if kw.get("tree") else None)
        for i in range(q):
            t = int(qp[b]) + i
            lo, hi, page_base, pos = tokens[t]
            keys = set(torch.nonzero(see[i]).flatten().tolist())
            if kw.get("tree"):
                assert (lo, hi, pos) == (0, n - q, n)
            else:
                assert set(range(lo, hi)) == keys and pos == n - q + i
            assert page_base == int(kp[b])
            assert keys <= seen[t]


def test_plan_refusals():
    call = attention_ops.plan_paged_attention
    good = dict(qo_indptr=i32([0, 2]), kv_indptr=i32([0, 1]), kv_indices=i32([4]),
                kv_last_page_len=i32([7]), num_heads=8, num_kv_heads=2, head_dim=128, page_size=16)
    assert call(**good).total_q == 2
    for change, words in [
            (dict(qo_indptr=i32([1, 2])), "begin with 0"),
            (dict(qo_indptr=i32([0, 3, 2]), kv_indptr=i32([0, 1, 1]), kv_last_page_len=i32([1, 1])),
             "not ascending"),
            (dict(kv_indptr=i32([0, 2])), "passes kv_indices"),
            (dict(kv_indices=i32([-1])), "negative page"),
            (dict(kv_last_page_len=i32([17])), "kv_last_page_len 17"),
            (dict(kv_last_page_len=i32([0])), "kv_last_page_len 0"),
            (dict(num_heads=9), "9 query heads over 2"),
            (dict(num_heads=129, num_kv_heads=1), "at most 128"),
            (dict(head_dim=12), "head_dim 12"),
            (dict(head_dim=512), "head_dim 512"),
            (dict(page_size=0), "bad shape"),
            (dict(prefix_lens=i32([-1])), "negative prefix"),
            (dict(tree_words=1, window_left=3), "no other mask"),
            (dict(tree_words=1, qo_indptr=i32([0, 8])), "drafts 8 tokens"),
            (dict(tree_words=1, qo_indptr=i32([0, 65]), kv_indptr=i32([0, 5]),
                  kv_indices=i32([0, 1, 2, 3, 4])), "drafts 65 tokens"),
            (dict(qo_indptr=torch.tensor([0, 2])), "int32 CPU tensor"),
            (dict(doc_starts=i32([0])), "doc_starts"),
            (dict(kv_indptr=i32([0])), "batch \\+ 1"),
            (dict(page_size=1 << 30, kv_indptr=i32([0, 3]), kv_indices=i32([0, 1, 2]),
                  kv_last_page_len=i32([5])), "a sequence of")]:
        with pytest.raises(RuntimeError, match=words):
            call(**{**good, **change})


def test_c_abi_refusals_need_no_gpu():
    lib = cabi.load()
    plan = cabi.AttentionPlan()
    arr = lambda *v: (ctypes.c_int32 * len(v))(*v)  # noqa: E731
    n = lib.pace_paged_attention_plan_words(1, 1, 1, 148)
    words = (ctypes.c_int32 * n)()

    def make(num_words=n):
        return lib.pace_paged_attention_plan(
            ctypes.byref(plan), words, num_words, arr(0, 1), arr(0, 1), arr(3), 1, arr(2), 1, 8, 2,
            128, 16, -1, None, None, 0, 148)

    assert make(5) == cabi.PACE_ERR_INVALID_ARGUMENT and b"words" in lib.pace_last_error()
    assert make() == cabi.PACE_OK
    assert (plan.total_q, plan.max_page, plan.num_few, plan.num_many) == (1, 3, 1, 0)

    def run(pages=4, stride=1024, cap=0.0, mask=None, out=16):
        return lib.pace_paged_attention(ctypes.byref(plan), 16, out, 16, stride, stride, 16, None,
                                        pages, 1.0, cap, None, mask, None, None, 0, None,
                                        cabi.PACE_BF16, None)

    for kw, word in [(dict(pages=3), b"page 3"), (dict(stride=1023), b"stride"),
                     (dict(cap=-1.0), b"soft_cap"), (dict(mask=16), b"tree mask"),
                     (dict(out=None), b"null pointer")]:
        assert run(**kw) == cabi.PACE_ERR_INVALID_ARGUMENT and word in lib.pace_last_error(), kw
    assert lib.pace_append_quantised_paged_kv_cache(
        None, None, 1, 2, 12, 24, 24, None, None, None, 1, 16, None, 1, None, None, 1, None,
        cabi.PACE_BF16, None) == cabi.PACE_ERR_INVALID_ARGUMENT
    assert b"head_dim 12" in lib.pace_last_error()


def test_cpu_tensors_rejected():
    x = torch.zeros(4, 2, 8, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        kv_transfer_ops.append_quantised_paged_kv_cache(
            torch.ones(1, 128), torch.ones(1, 128), i32([0, 1]), x,
            torch.zeros(4, 2, 8, 2, dtype=torch.uint8), i32([0]), i32([0, 1]), i32([1]))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        kv_transfer_ops.read_quantised_paged_kv_cache(
            torch.ones(1, 128), torch.ones(1, 128), i32([0, 1]), x,
            torch.zeros(4, 2, 8, 2, dtype=torch.uint8), i32([0]), i32([0, 1]), i32([1]))
