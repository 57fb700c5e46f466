"""GPU: the quantised paged KV cache -- append and read back -- bit for bit
against the restatement in 64 bits."""
import pytest
import torch

from oracle import attention_ref as ref
from paceserve_b200 import kv_transfer_ops as kv

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def pages_of(lens, page, seed=0, spare=3):
    """(kv_indptr, kv_indices, kv_last_page_len, pages in all) of sequences of these lengths."""
    n = [-(-x // page) for x in lens]
    total = sum(n) + spare
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed))[:sum(n)].int()
    return (torch.tensor([0] + n).cumsum(0).int(), ids,
            torch.tensor([(x - 1) % page + 1 if x else 1 for x in lens]).int(), total)


def rows_with_extremes(g, tokens, heads, hd, dtype):
    x = torch.randn(tokens, heads, hd, generator=g) * torch.exp(torch.randn(heads, hd, generator=g))
    x = x.to(dtype)
    flat = x.view(-1, hd)
    flat[0] = 0
    flat[1] = torch.finfo(dtype).max
    flat[2] = torch.finfo(dtype).tiny  # below it the exponent stops at its least
    flat[3, 0] = 448.0
    flat[3, 1:] = 0.0
    flat[4] = torch.tensor([1.75, 1.76]).to(dtype).repeat(hd // 2)  # either side of a binade of codes
    # a tie in every binade: halfway between codes, to the even one
    flat[5] = torch.tensor([448.0, 17.0, 19.0, 2.125, 2.375, 2.0 ** -10, 3 * 2.0 ** -10, 0.0]).to(
        dtype).repeat(hd // 8)
    if tokens * heads > 8:
        flat[6, 1] = float("inf")
        flat[6, 2] = -float("inf")
        flat[7, 3] = float("nan")
        flat[8] = float("inf")
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,hd,page,lens,new", [
    (8, 128, 16, [40, 1, 17], [40, 1, 3]),
    (1, 64, 8, [9], [9]),
    (3, 80, 5, [13, 6, 2], [4, 6, 1]),   # odd page size, 80 = 10 lanes of 8
    (2, 256, 1, [7, 3], [7, 1]),
    (5, 8, 16, [33], [20]),
    (4, 120, 32, [64, 31], [0, 31]),     # a request that appends nothing
])
def test_append_and_read(dtype, heads, hd, page, lens, new):
    g = torch.Generator().manual_seed(heads * hd)
    kp, ki, kl, total = pages_of(lens, page)
    ai = torch.tensor([0] + new).cumsum(0).int()
    n = int(ai[-1])
    key = rows_with_extremes(g, n, heads, hd, dtype)
    value = rows_with_extremes(g, n, heads, hd, dtype).flip(0)
    codes = torch.randint(0, 126, (total, 2, page, heads, hd), generator=g).to(torch.uint8)
    exps = torch.randint(100, 140, codes.shape[:-1], generator=g).to(torch.uint8)
    got_c, got_e = codes.to(DEV).view(torch.float8_e4m3fn), exps.to(DEV)
    ref.append_quantised(key, value, ai, codes, exps, ki, kp, kl)
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    d = lambda *ts: [t.to(DEV) for t in ts]  # noqa: E731
    # K and V as views of a wider row, as the qkv projection leaves them; then odd strides
    for pad in (8, 3):
        wide = torch.zeros(n, 2 * heads * hd + pad, dtype=dtype)
        wide[:, :heads * hd] = key.view(n, -1)
        wide[:, heads * hd:2 * heads * hd] = value.view(n, -1)
        wide = wide.to(DEV)
        kv.append_quantised_paged_kv_cache(wide[:, :heads * hd], wide[:, heads * hd:2 * heads * hd],
                                           *d(ai), got_c, got_e, *d(ki, kp, kl), bad)
        assert torch.equal(got_c.view(torch.uint8).cpu(), codes)
        assert torch.equal(got_e.cpu(), exps)
    assert bad.item() == 0
    # read all back: exact in every type that holds the value, else rounded once
    rows = torch.tensor([0] + lens).cumsum(0).int()
    want = ref.dequantise(codes, exps)
    want = [torch.cat([ref.gather_rows(want, ki, kp, kl, b)[kind] for b in range(len(lens))])
            for kind in (0, 1)]
    for out_dtype in (dtype, torch.float32):
        # contiguous rows, then rows inside wider ones
        for pad in (0, 8, 5):
            out = torch.full((2, int(rows[-1]), heads * hd + pad), 7.0, dtype=out_dtype, device=DEV)
            kv.read_quantised_paged_kv_cache(out[0, :, :heads * hd], out[1, :, :heads * hd], *d(rows),
                                             got_c, got_e, *d(ki, kp, kl), bad)
            for kind in (0, 1):
                a = out[kind, :, :heads * hd].cpu().view(-1, heads, hd)
                w = want[kind].float().to(out_dtype)
                assert torch.equal(a.isnan(), w.isnan())
                assert torch.equal(a.nan_to_num(0.0, 1e30, -1e30), w.nan_to_num(0.0, 1e30, -1e30))
            assert bool((out[:, :, heads * hd:] == 7.0).all())
    assert bad.item() == 0


def test_many_requests_and_many_tokens():
    """More requests than the kernels stage in shared memory, and enough tokens
    for the four-tokens-a-CTA form; against the kernel on a part at a time."""
    g = torch.Generator().manual_seed(2)
    heads, hd, page, b = 8, 128, 16, 2600
    lens = torch.randint(1, 40, (b,), generator=g).tolist()
    new = [min(n, int(x)) for n, x in zip(lens, torch.randint(0, 9, (b,), generator=g))]
    kp, ki, kl, total = pages_of(lens, page)
    ai = torch.tensor([0] + new).cumsum(0).int()
    n = int(ai[-1])
    key = torch.randn(n, heads * hd, generator=g).bfloat16().to(DEV)
    value = torch.randn(n, heads * hd, generator=g).bfloat16().to(DEV)
    d = lambda *ts: [t.to(DEV) for t in ts]  # noqa: E731

    def cache():
        return (torch.zeros(total, 2, page, heads, hd, dtype=torch.uint8, device=DEV).view(
            torch.float8_e4m3fn), torch.zeros(total, 2, page, heads, dtype=torch.uint8, device=DEV))

    c0, e0 = cache()
    kv.append_quantised_paged_kv_cache(key, value, *d(ai), c0, e0, *d(ki, kp, kl))
    c1, e1 = cache()
    for lo in range(0, b, 300):
        hi = min(b, lo + 300)
        t0, t1 = int(ai[lo]), int(ai[hi])
        kv.append_quantised_paged_kv_cache(key[t0:t1], value[t0:t1], *d(ai[lo:hi + 1] - ai[lo]), c1,
                                           e1, *d(ki, kp[lo:hi + 1], kl[lo:hi]))
    assert torch.equal(c0.view(torch.uint8), c1.view(torch.uint8)) and torch.equal(e0, e1)
    rows = torch.tensor([0] + lens).cumsum(0).int()
    out = torch.empty(2, int(rows[-1]), heads * hd, dtype=torch.bfloat16, device=DEV)
    kv.read_quantised_paged_kv_cache(out[0], out[1], *d(rows), c0, e0, *d(ki, kp, kl))
    want = ref.dequantise(c0.view(torch.uint8).cpu(), e0.cpu())
    for kind in (0, 1):
        w = torch.cat([ref.gather_rows(want, ki, kp, kl, r)[kind] for r in range(b)])
        assert torch.equal(out[kind].cpu(), w.bfloat16().view(-1, heads * hd))


def test_bad_tokens_are_skipped_and_counted():
    heads, hd, page = 2, 64, 8
    codes = torch.zeros(4, 2, page, heads, hd, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    exps = torch.zeros(4, 2, page, heads, dtype=torch.uint8, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    key = torch.ones(3, heads * hd, device=DEV)
    bad = i32([0])
    # request 0's page is outside the cache; request 1's last-page length is; request 2 is good
    kv.append_quantised_paged_kv_cache(key, key, i32([0, 1, 2, 3]), codes, exps, i32([9, 1, 2]),
                                       i32([0, 1, 2, 3]), i32([1, 9, 1]), bad)
    assert bad.item() == 2
    assert int((exps != 0).sum()) == 2 * heads
    out = torch.full((3, heads * hd), 5.0, device=DEV)
    kv.read_quantised_paged_kv_cache(out, out.clone(), i32([0, 1, 2, 3]), codes, exps,
                                     i32([9, 1, 2]), i32([0, 1, 2, 3]), i32([1, 9, 1]), bad)
    assert bad.item() == 4
    assert bool((out[:2] == 5.0).all()) and bool((out[2] == 1.0).all())


def test_refusals():
    codes = torch.zeros(4, 2, 8, 2, 64, dtype=torch.uint8, device=DEV)
    exps = torch.zeros(4, 2, 8, 2, dtype=torch.uint8, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    key = torch.ones(1, 128, device=DEV)
    meta = [i32([0]), i32([0, 1]), i32([1])]
    call = kv.append_quantised_paged_kv_cache
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        call(key, key, i32([0, 1]), codes, exps, *meta)
    f8 = codes.view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="exponents"):
        call(key, key, i32([0, 1]), f8, exps[:, :, :, :1], *meta)
    with pytest.raises(RuntimeError, match="share one of"):
        call(key, key.half(), i32([0, 1]), f8, exps, *meta)
    with pytest.raises(RuntimeError, match="must be \\[nnz"):
        call(key[:, :64], key[:, :64], i32([0, 1]), f8, exps, *meta)
    with pytest.raises(RuntimeError, match="token counts differ"):
        call(key, key.repeat(2, 1), i32([0, 1]), f8, exps, *meta)
    with pytest.raises(RuntimeError, match="batch \\+ 1"):
        call(key, key, i32([0, 1, 1]), f8, exps, *meta)
    with pytest.raises(RuntimeError, match="head_dim 12"):
        call(torch.ones(1, 24, device=DEV), torch.ones(1, 24, device=DEV), i32([0, 1]),
             torch.zeros(4, 2, 8, 2, 12, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn),
             exps, *meta)
