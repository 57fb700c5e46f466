"""GPU: paged attention against the restatement in 64 bits.

Tolerance, per element of the output o = sum p v (p the softmax): the output is
rounded once to its type (half an ulp: u * |o|, u = eps / 2 of the type: 2^-8 for
bf16, 2^-11 for fp16, 2^-24 for fp32), and the kernels round each p once to the
query's type before it meets v (at most u * sum p|v| in the worst case).  The
fp32 score of D products is off by at most (D + 3) * 2^-24 * scale * sum|q k|,
here under 2e-4 with these inputs, and moves p by twice that.  fp16's subnormals
lie 2^-24 apart, so rounding to them moves the smallest outputs by up to 2^-25.  So
    |got - want| <= u * |o| + (u + 4e-4) * sum p|v| + (2^-25 in fp16).
"""
import math

import pytest
import torch

from oracle import attention_ref as ref
from paceserve_b200 import kv_transfer_ops as kv
from paceserve_b200.attention import PagedAttention
from tests.test_kv_quant_gpu import pages_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
U = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


class Step:
    """One step's inputs: requests (new tokens, sequence length), a filled cache."""

    def __init__(self, lens, heads, kv_heads, hd, page=16, dtype=torch.bfloat16, quantised=False,
                 seed=0, spread=1.5):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.kv_heads, self.hd, self.page = lens, heads, kv_heads, hd, page
        self.kp, self.ki, self.kl, self.total = pages_of([n for _, n in lens], page, seed)
        self.qp = torch.tensor([0] + [q for q, _ in lens]).cumsum(0).int()
        t = int(self.qp[-1])
        self.query = (torch.randn(t, heads, hd, generator=g) * spread).to(dtype)
        rows = torch.randn(self.total, 2, page, kv_heads, hd, generator=g)
        self.exponents = None
        if quantised:
            codes = torch.randint(0, 256, rows.shape, generator=g).to(torch.uint8)
            codes = torch.where(codes % 128 == 127, codes - 1, codes)  # 127 and 255 are NaN
            self.exponents = torch.randint(118, 121, rows.shape[:-1], generator=g).to(torch.uint8)
            self.cache = codes
        else:
            self.cache = rows.to(dtype)

    def values(self):
        return ref.dequantise(self.cache, self.exponents) if self.exponents is not None else self.cache

    def run(self, tree_mask=None, window_left=-1, prefix_lens=None, doc_starts=None, attn=None,
            query=None, out=None, **kw):
        attn = attn or PagedAttention(self.heads, self.kv_heads, self.hd, self.page, DEV)
        if tree_mask is not None:
            attn.begin_tree_forward(self.qp, self.kp, self.ki, self.kl, tree_mask)
        else:
            attn.begin_forward(self.qp, self.kp, self.ki, self.kl, window_left=window_left,
                               prefix_lens=prefix_lens, doc_starts=doc_starts)
        if kw.get("alibi_slopes") is not None:
            kw["alibi_slopes"] = kw["alibi_slopes"].to(DEV)
        lse = torch.full((self.query.shape[0], self.heads), 3.0, device=DEV)
        fault = torch.zeros(1, dtype=torch.int32, device=DEV)
        cache = self.cache.to(DEV)
        if self.exponents is not None:
            cache = cache.view(torch.float8_e4m3fn)
        out = attn.forward(self.query.to(DEV) if query is None else query, cache, out=out,
                           exponents=None if self.exponents is None else self.exponents.to(DEV),
                           lse=lse, fault_flags=fault, **kw)
        assert fault.item() == 0
        return out.cpu(), lse.cpu()

    def want(self, **kw):
        kw["soft_cap"] = kw.pop("logits_soft_cap", 0.0)
        kw["slopes"] = kw.pop("alibi_slopes", None)
        kw.setdefault("sm_scale", 1.0 / math.sqrt(self.hd))
        args = (self.qp, self.kp, self.ki, self.kl)
        values = self.values()
        out, lse = ref.attention(self.query, values, *args, **kw)
        size = values.clone()
        size[:, 1] = size[:, 1].abs()
        return out, lse, ref.attention(self.query, size, *args, **kw)[0]

    def check(self, attn=None, query=None, out=None, **kw):
        got, lse = self.run(attn=attn, query=query, out=out, **kw)
        out, want_lse, size = self.want(**kw)
        u = U[self.query.dtype]
        err = (got.double() - out).abs()
        assert torch.equal(got.isnan(), out.isnan())
        most = u * out.abs() + (u + 4e-4) * size + TINY[self.query.dtype]
        assert bool(((err <= most) | out.isnan()).all()), (err - most).max()
        none = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, none)
        assert bool((got[none] == 0).all())
        assert bool(((lse.double() - want_lse).abs()[~none] <= 5e-4 + 1e-6 * want_lse.abs()[~none]).all())


DTYPES = [torch.bfloat16, torch.float16]
# (new tokens, sequence length): single tokens over one key to several thousand, prompts, chunks
# after a context, and their mixtures
DECODE = [(1, 1), (1, 16), (1, 17), (1, 63), (1, 333), (1, 2500), (1, 64), (1, 129)]
PROMPTS = [(1, 1), (33, 33), (130, 130), (257, 300), (64, 1000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 128), (8, 8, 64), (6, 2, 128), (32, 2, 64),
                                               (16, 1, 128), (40, 1, 64), (20, 4, 128)])
@pytest.mark.parametrize("lens", [DECODE, PROMPTS], ids=["decode", "prompts"])
def test_causal(dtype, quantised, heads, kv_heads, hd, lens):
    Step(lens, heads, kv_heads, hd, dtype=dtype, quantised=quantised).check()


@pytest.mark.parametrize("page", [1, 5, 8, 16, 32, 48, 64, 128, 256])
@pytest.mark.parametrize("quantised", [False, True])
def test_page_sizes(page, quantised):
    lens = [(1, 300), (1, 1), (70, 211), (3, 129), (200, 200)]
    Step(lens, 8, 2, 128, page=page, quantised=quantised, seed=page).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["cap", "alibi", "window", "prefix", "docs", "all"])
def test_scores_and_masks(dtype, quantised, hd, kind):
    lens = [(1, 700), (1, 5), (90, 400), (150, 150), (2, 260), (1, 1)]
    step = Step(lens, 12, 4, hd, dtype=dtype, quantised=quantised, seed=5)
    kw = {}
    if kind in ("cap", "all"):
        kw["logits_soft_cap"] = 2.5  # within the scores' range: they bend
    if kind in ("alibi", "all"):
        kw["alibi_slopes"] = torch.tensor([2.0 ** -(i % 9) for i in range(12)])
    if kind in ("window", "all"):
        kw["window_left"] = 70
    if kind in ("prefix", "all"):
        kw["prefix_lens"] = torch.tensor([3, 99, 333, 100, 0, 1]).int()
    if kind in ("docs", "all"):
        starts = []
        for q, n in lens:
            starts += [max(0, (p // 61) * 61 - (7 if p % 2 else 0)) for p in range(n - q, n)]
        kw["doc_starts"] = torch.tensor(starts).int()
    step.check(**kw)


def test_rows_that_see_nothing():
    """A window or document start past the sequence, more new tokens than the
    sequence holds, an empty sequence, requests without new tokens."""
    lens = [(1, 40), (5, 3), (0, 50), (1, 0), (150, 150), (0, 0), (200, 120)]
    step = Step(lens, 8, 2, 128, seed=9)
    starts = torch.zeros(int(step.qp[-1]), dtype=torch.int32)
    starts[0] = 40
    starts[50:90] = 1000
    step.check(doc_starts=starts)
    step.check()
    Step([(0, 4), (0, 0)], 8, 2, 128).check()


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("tokens", [1, 70])
def test_long_sequence_is_cut_and_joined(quantised, tokens):
    Step([(tokens, 20000)], 8, 2, 128, quantised=quantised, seed=1).check()
    Step([(tokens, 5000), (tokens, 7001), (1, 1)], 8, 2, 64, quantised=quantised, seed=1).check(
        logits_soft_cap=20.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 128), (4, 4, 64), (40, 8, 128)])
def test_tree(dtype, quantised, heads, kv_heads, hd):
    lens = [(1, 1), (13, 344), (64, 64), (2, 700), (65, 90), (100, 300), (7, 7)]
    step = Step(lens, heads, kv_heads, hd, dtype=dtype, quantised=quantised, seed=3)
    step.check(tree_mask=random_trees(lens, 2), logits_soft_cap=0.0)
    step.check(tree_mask=random_trees(lens, 3), logits_soft_cap=5.0)


def random_trees(lens, words, seed=0):
    """Random trees' ancestor masks; bits of nodes that a request does not have
    are set too, and must not matter."""
    g = torch.Generator().manual_seed(seed)
    rows = []
    for q, _ in lens:
        masks = []
        for i in range(q):
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
        for m in masks:
            m |= (1 << 64 * words) - (1 << q)
            ws = [m >> 64 * w & (1 << 64) - 1 for w in range(words)]
            rows.append([w - (1 << 64) if w >> 63 else w for w in ws])
    return torch.tensor(rows, dtype=torch.int64)


def test_tree_row_that_sees_nothing():
    step = Step([(3, 3), (40, 40)], 8, 2, 128)
    mask = random_trees(step.lens, 1)
    mask[1] = 0
    mask[20:30] = 0
    step.check(tree_mask=mask)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_masked_does_not_matter(hd, bad):
    """NaN and infinities in slots past a sequence's end, before a window, in the
    causal future of a row, and in a draft tree's other branches."""
    lens = [(1, 200), (100, 230), (3, 40)]
    step = Step(lens, 8, 2, hd, seed=4)
    used = [set() for _ in range(step.total)]
    for b, (q, n) in enumerate(lens):
        for j in range(n):
            used[int(step.ki[int(step.kp[b]) + j // step.page])].add(j % step.page)
    for p, slots in enumerate(used):
        for s in range(step.page):
            if s not in slots:
                step.cache[p, :, s] = bad
    step.check()
    for b, (q, n) in enumerate(lens):
        for j in list(range(0, n - q - 30)) + [n - 1]:
            step.cache[step.ki[int(step.kp[b]) + j // step.page], :, j % step.page] = bad
    # the last token of each sees the last key (in `bad`); those before it do not
    got, _ = step.run(window_left=20)
    out, _, size = step.want(window_left=20)
    last = (step.qp[1:] - 1).long()
    seen = torch.ones(out.shape[0], dtype=torch.bool)
    seen[last] = False
    u = U[torch.bfloat16]
    assert bool(((got.double() - out).abs() <= u * out.abs() + (u + 4e-4) * size)[seen].all())
    # a row that sees it is not finite, in the value's own columns or all of them
    assert not bool(got[last].isfinite().any())
    # a tree: the last node's slot is seen by itself alone
    mask = torch.tensor([[(1 << i) | 1] for q, _ in lens for i in range(q)], dtype=torch.int64) \
        if max(q for q, _ in lens) <= 63 else None
    if mask is None:
        lens = [(1, 200), (60, 230), (3, 40)]
        step = Step(lens, 8, 2, hd, seed=4)
        for b, (q, n) in enumerate(lens):
            j = n - 1
            step.cache[step.ki[int(step.kp[b]) + j // step.page], :, j % step.page] = bad
        mask = torch.tensor([[(1 << i) | 1] for q, _ in lens for i in range(q)], dtype=torch.int64)
    got, _ = step.run(tree_mask=mask)
    out, _, size = step.want(tree_mask=mask)
    last = (step.qp[1:] - 1).long()
    seen = torch.ones(out.shape[0], dtype=torch.bool)
    seen[last] = False
    assert bool(((got.double() - out).abs() <= u * out.abs() + (u + 4e-4) * size)[seen].all())
    assert not bool(got[last].isfinite().any())


def test_scores_far_apart():
    """Scores of hundreds in size, rising along the sequence (the running maximum
    moves at every step) and falling (it never does)."""
    for sign in (1.0, -1.0):
        step = Step([(1, 900), (100, 900)], 8, 2, 128, seed=6, spread=1.0)
        ramp = torch.linspace(0, 40, 900) * sign
        for b in range(2):
            for j in range(900):
                page = step.ki[int(step.kp[b]) + j // step.page]
                step.cache[page, 0, j % step.page] = 0
                step.cache[page, 0, j % step.page, :, 0] = ramp[j]
        step.query[..., 0] = 30.0
        step.check()


def test_quantised_extremes():
    """Exponents at both ends of their range and NaN rows, in either half type."""
    for dtype in DTYPES:
        step = Step([(1, 120), (40, 120)], 4, 2, 128, dtype=dtype, quantised=True, seed=8)
        step.exponents[:, 0] = torch.randint(1, 60, step.exponents[:, 0].shape).to(torch.uint8)
        step.exponents[:, 1] = torch.randint(95, 118, step.exponents[:, 1].shape).to(torch.uint8)
        step.check()
    step = Step([(1, 120), (40, 120)], 4, 2, 128, quantised=True, seed=8)
    step.exponents[step.ki[int(step.kp[0])], 1, 3, 0] = 255  # request 0's key 3, V of head 0
    got, _ = step.run()
    out, _, _ = step.want()
    assert torch.equal(got.isnan(), out.isnan()) and bool(got.isnan().any())
    step = Step([(1, 60), (40, 60)], 4, 2, 128, quantised=True, seed=8)
    step.exponents[:, 1] = torch.randint(200, 236, step.exponents[:, 1].shape).to(torch.uint8)
    step.check()  # values up to 2^117: bf16 holds them


@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_a_large_value_of_a_small_weight(dtype):
    """A key whose weight is 2^-20 and whose value row is 2^20 times the others':
    both parts of the output count."""
    for tokens in (1, 40):
        step = Step([(tokens, 100)], 4, 2, 128, dtype=dtype, quantised=True, seed=21)
        step.exponents[:] = 119
        # every key scores 0 but the one in question, which scores 20 powers of two below
        page, slot = step.ki[3], 7
        step.query[:] = 0
        step.query[..., 0] = 1.0
        step.cache[:, 0] = 0
        step.cache[page, 0, slot, :, 0] = 0x80 | 0x70  # -128
        step.exponents[page, 0, slot] = 127
        step.exponents[page, 1, slot] = 139
        kw = {"sm_scale": 20.0 / 128 / math.log2(math.e)}
        step.check(**kw)


@pytest.mark.parametrize("hd,dtype,quantised", [(96, torch.bfloat16, False), (256, torch.float16, True),
                                                (8, torch.bfloat16, True), (128, torch.float32, False),
                                                (64, torch.float32, True)])
def test_other_head_sizes_and_float32(hd, dtype, quantised):
    lens = [(1, 77), (30, 60), (2, 2), (1, 0)]
    step = Step(lens, 6, 2, hd, dtype=dtype, quantised=quantised, seed=2)
    step.check(logits_soft_cap=4.0, window_left=33,
               alibi_slopes=torch.tensor([2.0 ** -(i + 1) for i in range(6)]))
    step = Step(lens[:3], 6, 2, hd, dtype=dtype, quantised=quantised, seed=2)
    step.check(tree_mask=random_trees(lens[:3], 1))


def test_strided_queries_and_outputs():
    """Queries as views of the qkv projection, outputs as views of wider rows;
    odd strides and offsets that no 16-byte access fits."""
    lens = [(1, 300), (90, 200), (3, 50)]
    step = Step(lens, 8, 2, 128, seed=7)
    t = int(step.qp[-1])
    for pad in (0, 8, 3):
        for shift in (0, 1):
            wide = torch.zeros(t, 8 * 128 + 512 + pad, dtype=torch.bfloat16)
            wide[:, shift:shift + 1024] = step.query.view(t, -1)
            out = torch.full((t, 1024 + pad + shift), 9.0, dtype=torch.bfloat16, device=DEV)
            step.check(query=wide.to(DEV)[:, shift:shift + 1024].view(t, 8, 128),
                       out=out[:, shift:shift + 1024].view(t, 8, 128))
            assert bool((out[:, :shift] == 9.0).all()) and bool((out[:, shift + 1024:] == 9.0).all())


def test_offsets_past_32_bits():
    """Pages whose elements lie past 2^31 of the cache's start."""
    heads, hd, page = 2, 128, 16
    total = (1 << 31) // (2 * page * heads * hd) + 40
    cache = torch.zeros(total, 2, page, heads, hd, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(1)
    ids = torch.randperm(39, generator=g)[:21] + total - 39
    cache[ids] = torch.randn(21, 2, page, heads, hd, generator=g).bfloat16().to(DEV)
    lens = [(1, 200), (60, 120)]
    step = Step(lens, 8, 2, hd, seed=1)
    step.ki = ids.int()
    step.cache = torch.zeros(0)
    attn = PagedAttention(8, 2, hd, page, DEV)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    got = attn.forward(step.query.to(DEV), cache).cpu()
    step.cache = cache[total - 40:].cpu()
    step.ki = (ids - (total - 40)).int()
    out, _, size = step.want()
    u = U[torch.bfloat16]
    assert bool(((got.double() - out).abs() <= u * out.abs() + (u + 4e-4) * size).all())


def test_same_bits_every_time_and_plans_follow_each_other():
    """One object through steps of different shape; each gives the bits that a
    new object gives, also on another stream than the plan's."""
    attn = PagedAttention(8, 2, 128, 16, DEV)
    for lens in ([(1, 9000)], [(300, 4000), (1, 3000)], [(1, 5)], [(70, 9000)], [(1, 9000)]):
        step = Step(lens, 8, 2, 128, seed=11)
        first, _ = step.run()
        again, _ = step.run(attn=attn)
        assert torch.equal(first, again)
        cache, q = step.cache.to(DEV), step.query.to(DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            third = attn.forward(q, cache)
        side.synchronize()
        assert torch.equal(first, third.cpu())


def test_graph_capture():
    step = Step([(1, 3000), (1, 40), (40, 200)], 8, 2, 128, seed=12)
    attn = PagedAttention(8, 2, 128, 16, DEV)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    cache, q = step.cache.to(DEV), step.query.to(DEV)
    want = attn.forward(q, cache)
    torch.cuda.synchronize()
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn.forward(q, cache, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_append_then_attend():
    """A decode step as an engine runs it over a quantised cache: append, then
    attention that sees the new tokens."""
    lens = [(1, 33), (1, 500), (20, 60)]
    step = Step(lens, 8, 2, 128, quantised=True, seed=13)
    t = int(step.qp[-1])
    g = torch.Generator().manual_seed(1)
    key, value = (torch.randn(t, 2 * 128, generator=g).bfloat16() for _ in range(2))
    codes, exps = step.cache.to(DEV).view(torch.float8_e4m3fn), step.exponents.to(DEV)
    kv.append_quantised_paged_kv_cache(key.to(DEV), value.to(DEV), step.qp.to(DEV), codes, exps,
                                       step.ki.to(DEV), step.kp.to(DEV), step.kl.to(DEV))
    ref.append_quantised(key, value, step.qp, step.cache, step.exponents, step.ki, step.kp, step.kl)
    assert torch.equal(codes.view(torch.uint8).cpu(), step.cache)
    step.check()


@pytest.mark.parametrize("cap", [0.3, 1.5, 6.0, 40.0, 3000.0])
@pytest.mark.parametrize("hd", [64, 128])
def test_caps_above_among_and_below_the_scores(cap, hd):
    """The capped score has a form for scores well below the cap, one for scores
    below it, and one for any."""
    Step([(1, 300), (130, 400)], 8, 2, hd, seed=19).check(logits_soft_cap=cap)
    Step([(1, 300), (130, 400)], 8, 2, hd, seed=19, dtype=torch.float16).check(logits_soft_cap=cap)


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.7])
def test_any_scale(scale):
    Step([(1, 70), (90, 200)], 8, 2, 128, seed=14, spread=0.3).check(sm_scale=scale)
    Step([(1, 70), (90, 200)], 8, 2, 64, seed=14, spread=0.3, quantised=True).check(
        sm_scale=scale, logits_soft_cap=3.0)


def test_cache_at_an_odd_address():
    """A cache that no 16-byte access fits: the CUDA-core kernel takes it."""
    step = Step([(1, 70), (30, 60)], 8, 2, 128, seed=15)
    flat = torch.zeros(step.cache.numel() + 1, dtype=torch.bfloat16, device=DEV)
    flat[1:] = step.cache.flatten().to(DEV)
    attn = PagedAttention(8, 2, 128, 16, DEV)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    got = attn.forward(step.query.to(DEV), flat[1:].view(step.cache.shape)).cpu()
    out, _, size = step.want()
    u = U[torch.bfloat16]
    assert bool(((got.double() - out).abs() <= u * out.abs() + (u + 4e-4) * size).all())


def test_the_widest_group():
    Step([(1, 300), (5, 130)], 128, 1, 64, seed=16).check()
    Step([(1, 300), (5, 130)], 256, 2, 128, seed=16, quantised=True).check()


def test_without_programmatic_launch():
    """A step with few and many rows, whose two kernels otherwise run beside each
    other, in plain order."""
    import paceserve_b200

    step = Step([(1, 900), (100, 300), (1, 40)], 8, 2, 128, seed=17)
    first, _ = step.run()
    paceserve_b200.set_pdl(False)
    try:
        second, _ = step.run()
    finally:
        paceserve_b200.set_pdl(True)
    assert torch.equal(first, second)
    step.check()


def test_append_and_attention_in_one_stream_order():
    """Layer after layer without a wait: each attention sees its layer's append, and
    the next append does not overtake it."""
    lens = [(1, 200), (120, 300)]
    step = Step(lens, 8, 2, 128, seed=18)
    t = int(step.qp[-1])
    g = torch.Generator().manual_seed(1)
    keys = [torch.randn(2, t, 2 * 128, generator=g).bfloat16() for _ in range(4)]
    on = [k.to(DEV) for k in keys]
    cache = step.cache.to(DEV)
    attn = PagedAttention(8, 2, 128, 16, DEV)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    q, meta = step.query.to(DEV), [x.to(DEV) for x in (step.qp, step.ki, step.kp, step.kl)]
    outs = []
    for k in on:  # the same cache again and again
        kv.append_paged_kv_cache_by_indptr(k[0], k[1], meta[0], cache, *meta[1:])
        outs.append(attn.forward(q, cache))
    torch.cuda.synchronize()
    for k, got in zip(keys, outs):
        for b, (n, length) in enumerate(lens):
            for i in range(n):
                pos = length - n + i
                page = step.ki[int(step.kp[b]) + pos // 16]
                step.cache[page, :, pos % 16] = k[:, int(step.qp[b]) + i].view(2, 2, 128)
        out, _, size = step.want()
        u = U[torch.bfloat16]
        assert bool(((got.cpu().double() - out).abs() <= u * out.abs() + (u + 4e-4) * size).all())


def test_example_steps():
    """examples/paged_attention_steps.py: every step's output and the rows read back."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "paged_attention_steps.py")
    spec = importlib.util.spec_from_file_location("paged_attention_steps", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    steps, rows = example.main(DEV)
    u = U[torch.bfloat16]
    for s in steps:
        values = ref.dequantise(s["codes"].cpu(), s["exponents"].cpu())
        args = dict(sm_scale=1 / math.sqrt(128), soft_cap=s["options"].get("logits_soft_cap", 0.0),
                    tree_mask=s["tree_mask"])
        out, _ = ref.attention(s["query"].cpu(), values, *s["meta"], **args)
        size = values.clone()
        size[:, 1] = size[:, 1].abs()
        size, _ = ref.attention(s["query"].cpu(), size, *s["meta"], **args)
        err = (s["out"].cpu().double() - out).abs()
        assert bool((err <= u * out.abs() + (u + 4e-4) * size).all())
    k, v = ref.gather_rows(values, rows["kv_indices"], rows["kv_indptr"], rows["kv_last_page_len"], 0)
    assert torch.equal(rows["key"].cpu(), k.bfloat16()) and torch.equal(rows["value"].cpu(), v.bfloat16())


def test_refusals():
    step = Step([(1, 30)], 8, 2, 128)
    attn = PagedAttention(8, 2, 128, 16, DEV)
    q, cache = step.query.to(DEV), step.cache.to(DEV)
    with pytest.raises(RuntimeError, match="has not planned"):
        attn.forward(q, cache)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    with pytest.raises(RuntimeError, match="the plan is for 1 tokens"):
        attn.forward(torch.cat([q, q]), cache)
    with pytest.raises(RuntimeError, match="query's dtype"):
        attn.forward(q.half(), cache)
    with pytest.raises(RuntimeError, match="not the plan's"):
        attn.forward(q, cache[:, :, :8].contiguous())
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        attn.forward(step.query, cache)
    with pytest.raises(RuntimeError, match="heads must be contiguous"):
        attn.forward(q.transpose(1, 2).contiguous().transpose(1, 2), cache)
    with pytest.raises(RuntimeError, match="of a cache of"):
        attn.forward(q, cache[:1])
    with pytest.raises(RuntimeError, match="logits_soft_cap"):
        attn.forward(q, cache, logits_soft_cap=-1.0)
    with pytest.raises(RuntimeError, match="alibi_slopes"):
        attn.forward(q, cache, alibi_slopes=torch.ones(3, device=DEV))
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        attn.forward(q, cache, exponents=torch.zeros(cache.shape[:-1], dtype=torch.uint8, device=DEV))
    with pytest.raises(RuntimeError, match="lse"):
        attn.forward(q, cache, lse=torch.zeros(1, 3, device=DEV))
    attn.begin_tree_forward(step.qp, step.kp, step.ki, step.kl, torch.ones(1, 1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no distance bias"):
        attn.forward(q, cache, alibi_slopes=torch.ones(8, device=DEV))
    with pytest.raises(RuntimeError, match="a row for each"):
        attn.begin_tree_forward(step.qp, step.kp, step.ki, step.kl, torch.ones(2, 1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="tree_mask must be int64"):
        attn.begin_tree_forward(step.qp, step.kp, step.ki, step.kl, torch.ones(1, 1))
