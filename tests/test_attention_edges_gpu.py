"""GPU: paged attention and the quantised cache where inputs are at an edge.

Tolerances are those derived in ``test_attention_gpu.py``.
"""
import math

import pytest
import torch

from oracle import attention_ref as ref
from paceserve_b200 import kv_transfer_ops as kv
from paceserve_b200.attention import PagedAttention, attention_ops
from tests.test_attention_gpu import DEV, U, Step, random_trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("quantised", [False, True])
def test_pieces_without_a_key_are_zero(dtype, hd, quantised):
    """Whole pieces of the tile kernel that see nothing, beside ones that do: zeros, not what
    else passes through the output's place in shared memory.  Queries at an odd address arrive
    late, element by element."""
    lens = [(900, 900), (130, 130), (300, 0), (200, 64)]
    step = Step(lens, 8, 2, hd, dtype=dtype, quantised=quantised, seed=31)
    t = int(step.qp[-1])
    starts = torch.zeros(t, dtype=torch.int32)
    starts[:900] = 10 ** 6
    cache = step.cache.to(DEV)
    exponents = None if step.exponents is None else step.exponents.to(DEV)
    if quantised:
        cache = cache.view(torch.float8_e4m3fn)
    want = step.want(doc_starts=starts)[0].ne(0).any(-1).any(-1)  # rows that see something
    assert 0 < int(want.sum()) < 300
    attn = PagedAttention(8, 2, hd, 16, DEV)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl, doc_starts=starts)
    for shift in (0, 1):
        wide = torch.full((t, 8 * hd + 9), 5.0, dtype=dtype)
        wide[:, shift:shift + 8 * hd] = step.query.view(t, -1)
        query = wide.to(DEV)[:, shift:shift + 8 * hd].view(t, 8, hd)
        for _ in range(20):
            out = torch.full((t, 8, hd), 9.0, dtype=dtype, device=DEV)
            lse = torch.zeros(t, 8, device=DEV)
            attn.forward(query, cache, exponents=exponents, out=out, lse=lse)
            assert not bool(out.cpu()[~want].any())
            assert bool((lse.cpu()[~want] == -float("inf")).all())
    step.check(doc_starts=starts)


def test_workspace_at_an_odd_address_is_refused():
    step = Step([(70, 20000)], 8, 2, 128, seed=1)
    plan = attention_ops.plan_paged_attention(step.qp, step.kp, step.ki, step.kl, 8, 2, 128, 16)
    assert plan.many_slots > 0
    workspace = torch.zeros(plan.workspace_bytes + 64, dtype=torch.uint8, device=DEV)
    query, cache = step.query.to(DEV), step.cache.to(DEV)
    outs = []
    for shift in (0, 16, 32, 8):
        args = (query, cache, plan, plan.words.to(DEV), workspace[shift:], 0.1)
        outs.append(torch.zeros_like(query))
        if shift % 32:
            with pytest.raises(RuntimeError, match="32-byte aligned workspace"):
                attention_ops.paged_attention(outs[-1], *args)
        else:
            attention_ops.paged_attention(outs[-1], *args)
            workspace.zero_()  # the next one's counters lie elsewhere
    assert bool(outs[0].any()) and torch.equal(outs[0], outs[2])


def test_a_wait_that_ran_out_is_told_and_forgotten():
    """The object's own flag, as a kernel would leave it (no wait runs out here), and a
    workspace whose counters are not zero: ``check`` raises once, and what follows is right."""
    step = Step([(70, 9000), (1, 5000)], 8, 2, 128, seed=11)
    attn = PagedAttention(8, 2, 128, 16, DEV)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    assert attn.plan.many_slots > 0 and attn.plan.few_slots > 0
    query, cache = step.query.to(DEV), step.cache.to(DEV)
    want = attn.forward(query, cache)
    attn.check()
    attn._fault.fill_(1 << 30)
    attn._workspace[:65536].view(torch.int32).fill_(1)
    with pytest.raises(RuntimeError, match="wait ran out"):
        attn.check()
    attn.check()
    assert torch.equal(attn.forward(query, cache), want)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    assert torch.equal(attn.forward(query, cache), want)
    # a caller's own flag takes its place
    mine = torch.zeros(1, dtype=torch.int32, device=DEV)
    attn.forward(query, cache, fault_flags=mine)
    assert mine.item() == 0


@pytest.mark.parametrize("tokens", [1, 70])
def test_a_plan_written_by_the_kernel_before(tokens):
    """Plan words that a kernel writes right before the call, over another step's: the call sees
    the new ones, also where it may start before that kernel has ended."""
    steps = [Step(lens, 8, 2, 128, seed=3) for lens in ([(tokens, 900), (tokens, 130)],
                                                       [(tokens, 130), (tokens, 900)])]
    cache = steps[0].cache.to(DEV)
    assert steps[0].total == steps[1].total
    plans = [attention_ops.plan_paged_attention(s.qp, s.kp, s.ki, s.kl, 8, 2, 128, 16) for s in steps]
    n = plans[0].words.numel()
    assert plans[1].words.numel() == n and not torch.equal(plans[0].words, plans[1].words)
    workspace = torch.zeros(max(p.workspace_bytes for p in plans), dtype=torch.uint8, device=DEV)
    query = steps[0].query.to(DEV)
    # both at the end of a buffer whose writing takes a while
    source = [torch.zeros(1 << 24, dtype=torch.int32, device=DEV) for _ in plans]
    for s, p in zip(source, plans):
        s[-n:] = p.words.to(DEV)
    words = source[0].clone()
    want = []
    for p in plans:
        want.append(torch.empty_like(query))
        attention_ops.paged_attention(want[-1], query, cache, p, p.words.to(DEV), workspace, 0.1)
    torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    outs = []
    for i in range(40):
        torch.add(source[i % 2], 0, out=words)
        outs.append(torch.empty_like(query))
        attention_ops.paged_attention(outs[-1], query, cache, plans[i % 2], words[-n:], workspace, 0.1)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))


@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_tree_of_one_hidden_node(heads, hd, bad):
    """A drafted token that does not see itself, whose value row is not finite: the few-row
    kernel (8 heads of 2) and the tile kernel (64)."""
    lens = [(1, 300), (1, 1), (1, 40), (1, 5000)]
    step = Step(lens, heads, 2, hd, seed=6)
    for b, (_, n) in enumerate(lens):
        step.cache[step.ki[int(step.kp[b]) + (n - 1) // 16], 1, (n - 1) % 16] = bad
    step.check(tree_mask=torch.zeros(len(lens), 1, dtype=torch.int64))


def zero_row_step(tokens, length, key, above, exponent, zero_exponent, hd=128, dtype=torch.bfloat16,
                  heads=8):
    """Requests whose key `key` has a value row of zeros and a score `above` powers of two over the
    others', which are near 0; the values' exponent byte, and the zero row's."""
    step = Step([(q, n) for q, n in zip(tokens, length)], heads, 2, hd, dtype=dtype, quantised=True,
                seed=41)
    step.exponents[:, 1] = exponent
    step.query[..., 0] = 1.0  # times the key's 128
    step.exponents[:, 0] = 114  # the others' keys are up to 448 * 2^-13
    for b in range(len(tokens)):
        page, slot = step.ki[int(step.kp[b]) + key // step.page], key % step.page
        step.cache[page, :, slot] = 0
        step.exponents[page, 0, slot] = 127
        step.cache[page, 0, slot, :, 0] = 0x70 if above else 0
        step.exponents[page, 1, slot] = zero_exponent
    return step, {"sm_scale": above / 128 / math.log2(math.e)} if above else {}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("above", [0, 6, 10])
@pytest.mark.parametrize("exponent", [118, 113, 108, 90])  # values up to 0.9, 0.03, 9e-4, 3e-9
@pytest.mark.parametrize("zero_exponent", [1, 127, 140])
def test_a_value_row_of_zeros(dtype, above, exponent, zero_exponent):
    """A visible key with a value row of zeros adds to the softmax's sum alone, whatever the row's
    exponent and however high its score: few rows and many, whole and cut, in trees."""
    for tokens, lengths, heads in (((1, 1, 1), (300, 33, 20), 8), ((1, 4), (6000, 5000), 8),
                                   ((2, 1), (70, 300), 16), ((80, 40), (300, 200), 8),
                                   ((70,), (6000,), 8)):
        if dtype == torch.float16 and exponent == 90:
            continue  # no values of fp16
        step, kw = zero_row_step(tokens, lengths, 17, above, exponent, zero_exponent, dtype=dtype,
                                 heads=heads)
        step.check(**kw)
    step, kw = zero_row_step((5, 3), (300, 90), 17, above, max(exponent, 100), zero_exponent, hd=64)
    step.check(tree_mask=random_trees(step.lens, 1), **kw)


def test_nothing_but_zeros():
    """A cache as it is allocated, and zero rows as the append leaves them."""
    for zero_exponent in (0, 1, 127):
        step = Step([(1, 300), (1, 4000), (50, 200)], 8, 2, 128, quantised=True, seed=1)
        step.cache[:] = 0
        step.exponents[:] = zero_exponent
        step.check()
    key = torch.zeros(3, 2 * 128, dtype=torch.bfloat16)
    key[1, 5] = 1.0
    codes = torch.zeros(4, 2, 16, 2, 128, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    exps = torch.zeros(4, 2, 16, 2, dtype=torch.uint8, device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    kv.append_quantised_paged_kv_cache(key.to(DEV), key.to(DEV), i32(0, 3), codes, exps, i32(2),
                                       i32(0, 1), i32(3))
    # e = -126 for zeros; 1 is 256 * 2^-8
    assert exps[2, :, :3].cpu().tolist() == [[[1, 1], [119, 1], [1, 1]]] * 2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_finite_rows_read_back_finite(dtype):
    """The type's largest magnitudes, within 2^-4 as any other value; beside infinities too."""
    heads, hd, most = 2, 64, torch.finfo(dtype).max
    x = torch.full((4, heads * hd), most, dtype=dtype)
    x[1] = -most
    # 247 and 249 of 256 parts either side of the last tie, and smaller ones
    x[2] = (torch.tensor([247.0, 249.0, 240.0, -249.0, 17.0, 1.0, 0.0, -255.0]) / 256).to(dtype).repeat(
        heads * hd // 8) * (most / 2) * 2
    x[3, ::3] = most
    x[3, 1] = float("inf")
    codes = torch.zeros(4, 2, 16, heads, hd, dtype=torch.uint8)
    exps = torch.zeros(4, 2, 16, heads, dtype=torch.uint8)
    got_c, got_e = codes.to(DEV).view(torch.float8_e4m3fn), exps.to(DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    meta = [i32(2), i32(0, 1), i32(4)]
    on = [t.to(DEV) for t in meta]
    kv.append_quantised_paged_kv_cache(x.to(DEV), x.to(DEV), i32(0, 4).to(DEV), got_c, got_e, *on)
    ref.append_quantised(x, x, i32(0, 4), codes, exps, *meta)
    assert torch.equal(got_c.view(torch.uint8).cpu(), codes) and torch.equal(got_e.cpu(), exps)
    out = torch.zeros(2, 4, heads * hd, dtype=dtype, device=DEV)
    kv.read_quantised_paged_kv_cache(out[0], out[1], i32(0, 4).to(DEV), got_c, got_e, *on)
    for got in out.cpu():
        finite = x.isfinite()
        assert bool(got[finite].isfinite().all())
        # relative to the row's largest, which bounds the subnormal codes' error too
        err = (got.double() - x.double()).abs()[finite]
        assert bool((err <= 2.0 ** -4 * x.double().abs()[finite] + 2.0 ** -18 * most).all())


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_small_weights_keep_their_bits(dtype, quantised):
    """Few rows and many, scores spread so far that one key has nearly all of the weight, and a
    value row of that key that is zero in half of the dimensions: what the others, down to 2^-20
    of it, give there is as exact as anything else."""
    for tokens in (1, 3, 70):
        for length in (200, 6000):
            step = Step([(tokens, length)], 8, 2, 128, dtype=dtype, quantised=quantised, seed=25)
            page, slot = step.ki[2], 5  # key 37
            step.query[..., 0] = 4.0
            step.cache[:, 0, :, :, 0] = 0
            if quantised:
                step.exponents[page, 0, slot] = 121
                step.cache[page, 0, slot] = 0
                step.cache[page, 0, slot, :, 0] = 0x7e  # 448 / 64 = 7
                step.cache[page, 1, slot, :, :64] = 0
                k = 7.0
            else:
                step.cache[page, 0, slot] = 0
                step.cache[page, 0, slot, :, 0] = k = 7.0
                step.cache[page, 1, slot, :, :64] = 0
            # the others' scores are near 0 for a scale so small but for this key's
            step.query[..., 1:] *= 0.02
            step.check(sm_scale=20.0 / (4.0 * k) / math.log2(math.e))


@pytest.mark.parametrize("cap", [513.0, 1e4, 1e5, 1e6, 1e9, 3e38, float("inf")])
@pytest.mark.parametrize("quantised", [False, True])
def test_large_caps(cap, quantised):
    """A cap far above the scores hardly bends them, in whichever kernel; an infinite one is none."""
    for hd, spread in ((64, 1.5), (128, 1.5), (128, 8.0)):
        step = Step([(1, 300), (3, 90), (130, 400), (1, 6000)], 8, 2, hd, quantised=quantised, seed=23,
                    spread=spread)
        got, lse = step.run(logits_soft_cap=cap)
        out, want_lse, size = step.want(logits_soft_cap=cap if cap < math.inf else 0.0)
        u = U[torch.bfloat16]
        assert bool(((got.double() - out).abs() <= u * out.abs() + (u + 4e-4) * size).all())
        assert bool(((lse.double() - want_lse).abs() <= 5e-4 + 1e-6 * want_lse.abs()).all())


@pytest.mark.parametrize("cap", [600.0, 1e4, 1e5])
@pytest.mark.parametrize("tokens", [1, 5, 70])
@pytest.mark.parametrize("hd", [64, 128])
def test_large_caps_beside_a_score_near_them(cap, tokens, hd):
    """One key whose score is minus half the cap; the others' are ordinary and all that counts."""
    step = Step([(tokens, 300), (tokens, 5000)], 8, 2, hd, seed=24)
    step.query[..., 0] = 8.0
    for b, (_, n) in enumerate(step.lens):
        for j in (3, n - tokens - 2):
            page, slot = step.ki[int(step.kp[b]) + j // 16], j % 16
            step.cache[page, 0, slot, :, 0] = -0.5 * cap / 8 * math.sqrt(hd)
    step.check(logits_soft_cap=cap)


def test_infinite_and_nan_rows_cost_what_others_do():
    """Rows that are not finite by what they see are not done again on the CUDA cores: NaN queries
    and keys, and an infinite value that all rows but the first see."""
    step = Step([(2048, 2048)], 32, 8, 128, seed=26)
    attn = PagedAttention(32, 8, 128, 16, DEV)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    query, cache = step.query.to(DEV), step.cache.to(DEV)

    def ms(q, c):
        times = []
        for _ in range(5):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            attn.forward(q, c)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    base = ms(query, cache)
    nan_query = query.clone()
    nan_query[:] = math.nan
    nan_key, inf_value = cache.clone(), cache.clone()
    nan_key[step.ki[0], 0, 0] = math.nan
    inf_value[step.ki[0], 1, 1] = math.inf
    for q, c in ((nan_query, cache), (query, nan_key), (query, inf_value)):
        assert ms(q, c) < 20 * base  # 500 times and more where every row was done again


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("lens", [[(1, 300), (4, 40)], [(90, 300), (300, 300)], [(70, 6000), (2, 9000)]])
def test_values_not_finite_where_seen(hd, quantised, lens):
    """An infinite (or, quantised, a NaN) value row in each sequence: seen by the later tokens,
    whose outputs are not finite, hidden from the others, whose outputs are as without it."""
    step = Step(lens, 8, 2, hd, quantised=quantised, seed=27, spread=0.3)
    at = [max(n - q + q // 2, 0) for q, n in lens]
    for b, j in enumerate(at):
        page, slot = step.ki[int(step.kp[b]) + j // 16], j % 16
        if quantised:
            step.exponents[page, 1, slot] = 255
            step.cache[page, 1, slot] = 0
        else:
            step.cache[page, 1, slot, :, ::3] = math.inf
    got, _ = step.run()
    out, _, _ = step.want()
    assert torch.equal(got.isfinite(), out.isfinite()) and bool(got.isfinite().any())
    assert not bool(got.isfinite().all())
    hidden = torch.cat([torch.arange(n - q, n) < j for (q, n), j in zip(lens, at)])
    clean = Step(lens, 8, 2, hd, quantised=quantised, seed=27, spread=0.3)
    out, _, size = clean.want()
    u = U[torch.bfloat16]
    err = (got.double() - out).abs()
    assert bool((err <= u * out.abs() + (u + 4e-4) * size)[hidden].all())


def test_a_graph_outlives_the_plan_it_was_captured_with():
    """Later steps on the same object, and whatever then takes freed memory, leave the captured
    step's plan, workspace and tree mask as they were."""
    step = Step([(1, 3000), (9, 4000), (40, 2000)], 8, 2, 128, seed=28)
    mask = random_trees(step.lens, 1)
    attn = PagedAttention(8, 2, 128, 16, DEV)
    cache, q = step.cache.to(DEV), step.query.to(DEV)
    for kw in ({}, {"tree": True}):
        if kw:
            attn.begin_tree_forward(step.qp, step.kp, step.ki, step.kl, mask)
        else:
            attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
        assert attn.plan.few_slots > 0 and attn.plan.many_slots > 0
        want = attn.forward(q, cache)
        torch.cuda.synchronize()
        out = torch.zeros_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attn.forward(q, cache, out=out)
        kept = attn._step
        for n in (20000, 30000):  # needs a larger workspace
            other = Step([(70, n), (1, 40)], 8, 2, 128, seed=29)
            attn.begin_forward(other.qp, other.kp, other.ki, other.kl)
            attn.forward(other.query.to(DEV), other.cache.to(DEV))
        assert kept in attn._captured
        del kept
        filler = [torch.full((k,), -1, dtype=torch.uint8, device=DEV)
                  for k in (512, 2048, 8192, 1 << 20, 1 << 22, 1 << 24) for _ in range(4)]
        torch.cuda.synchronize()
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        del filler, graph


def test_a_page_locked_tree_mask_may_be_written_again():
    """The engine fills the same page-locked buffer for the next step while the GPU is behind."""
    step = Step([(40, 300), (3, 90)], 8, 2, 128, seed=30)
    mask = random_trees(step.lens, 1)
    want, _ = step.run(tree_mask=mask)
    host = mask.clone().pin_memory()
    attn = PagedAttention(8, 2, 128, 16, DEV)
    cache, q = step.cache.to(DEV), step.query.to(DEV)
    for _ in range(3):
        host.copy_(mask)
        torch.cuda._sleep(200_000_000)
        attn.begin_tree_forward(step.qp, step.kp, step.ki, step.kl, host)
        host.zero_()
        assert torch.equal(attn.forward(q, cache).cpu(), want)


def test_output_over_the_query_is_refused():
    step = Step([(1, 30)], 8, 2, 128)
    attn = PagedAttention(8, 2, 128, 16, DEV)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    q = step.query.to(DEV)
    with pytest.raises(RuntimeError, match="out must not be the query"):
        attn.forward(q, step.cache.to(DEV), out=q)
    assert torch.equal(q.cpu(), step.query)


def test_planning_during_a_capture_is_refused():
    step = Step([(1, 300)], 8, 2, 128, seed=32)
    attn = PagedAttention(8, 2, 128, 16, DEV)
    attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
    cache, q = step.cache.to(DEV), step.query.to(DEV)
    want = attn.forward(q, cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before the CUDA graph"):
            attn.begin_forward(step.qp, step.kp, step.ki, step.kl)
        out = attn.forward(q, cache)  # the step planned before
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
