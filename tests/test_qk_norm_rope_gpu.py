"""GPU: head norms with rotation, in place and into the paged cache, against 64 bits.

Tolerance: half a step of the output, and 2^-18 of the rotated pair's sizes for fp32 (up to 16 squares
a lane and 5 more additions, halved by the root, rsqrt, and at most 6 roundings of products and sums:
under 40 * 2^-24)."""
import pytest
import torch

from oracle import heads_ref as ref
from oracle import ops_ref
from paceserve_b200 import pos_encoding_ops as pe

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-6


def check(got, want, size, dtype):
    got, f = got.double().cpu(), torch.finfo(dtype)
    tol = f.eps / 2 * want.abs() + 2.0 ** -18 * size + f.smallest_normal * f.eps / 2
    d = (got - want).abs()
    assert (d <= tol).all(), float((d - tol).max())


def make(t, heads, kv_heads, d, rot, dtype, seed=0, cache_dtype=torch.float32, pad=0, positions=512):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(t, (heads + 2 * kv_heads) * d + pad, generator=g) * 3).to(dtype)
    w = [(1 + torch.randn(d, generator=g) / 4).to(dtype) for _ in range(2)]
    cs = ops_ref.cos_sin_cache(rot, positions, 10000.0).to(cache_dtype)
    pos = torch.randint(0, positions, (t,), generator=g)
    return qkv, w, cs, pos


def split(qkv, heads, kv_heads, d):
    n = heads * d, (heads + kv_heads) * d, (heads + 2 * kv_heads) * d
    return qkv[:, :n[0]], qkv[:, n[0]:n[1]], qkv[:, n[1]:n[2]]


SHAPES = [  # heads, kv_heads, d, rot
    (32, 8, 128, 128), (24, 8, 64, 32), (5, 1, 128, 64), (3, 3, 96, 96), (2, 1, 80, 32), (7, 2, 256, 128),
    (4, 2, 112, 56), (1, 1, 8, 4), (3, 1, 20, 20), (2, 2, 33, 10), (64, 8, 128, 128), (1, 0, 64, 64),
    (0, 2, 64, 64), (2, 1, 512, 256)]


@pytest.mark.parametrize("heads,kv_heads,d,rot", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neox", [True, False])
def test_in_place(heads, kv_heads, d, rot, dtype, neox):
    for t in (1, 37):
        qkv, (qw, kw), cs, pos = make(t, heads, kv_heads, d, rot, dtype, seed=d + t)
        dev = qkv.to(DEV)
        q, k, v = split(dev, heads, kv_heads, d)
        pe.qk_norm_rotary_embedding(pos.to(DEV), q, k, qw.to(DEV), kw.to(DEV), EPS, d, cs.to(DEV), neox)
        hq, hk, hv = split(qkv, heads, kv_heads, d)
        for got, x, w, n in ((q, hq, qw, heads), (k, hk, kw, kv_heads)):
            want, size = ref.norm_rope(x.reshape(t, n, d), w, EPS, pos, cs, neox)
            check(got.reshape(t, n, d), want, size, dtype)
        assert torch.equal(v.cpu(), hv)


@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad", [0, 8, 3])  # rows further apart; by 3: no vector access
def test_strides_and_cache_types(cache_dtype, pad):
    t, heads, kv_heads, d = 19, 6, 2, 64
    qkv, (qw, kw), cs, pos = make(t, heads, kv_heads, d, d, torch.bfloat16, cache_dtype=cache_dtype, pad=pad)
    dev = qkv.to(DEV)
    q, k, _ = split(dev, heads, kv_heads, d)
    pe.qk_norm_rotary_embedding(pos.to(DEV), q.unflatten(1, (heads, d)), k, qw.to(DEV), kw.to(DEV), EPS, d,
                                cs.to(DEV), True)
    for got, x, w, n in zip((q, k), split(qkv, heads, kv_heads, d), (qw, kw), (heads, kv_heads)):
        want, size = ref.norm_rope(x.reshape(t, n, d), w, EPS, pos, cs, True)
        check(got.reshape(t, n, d), want, size, torch.bfloat16)
    n = (heads + kv_heads) * d
    assert torch.equal(dev[:, n:].cpu(), qkv[:, n:])


@pytest.mark.parametrize("d", [64, 33])
def test_positions_outside_the_table(d):
    t, heads, kv_heads = 9, 4, 2
    qkv, (qw, kw), cs, pos = make(t, heads, kv_heads, d, 32, torch.bfloat16)
    pos[2], pos[5], pos[7] = -1, 512, 1 << 40
    dev = qkv.to(DEV)
    q, k, _ = split(dev, heads, kv_heads, d)
    pe.qk_norm_rotary_embedding(pos.to(DEV), q, k, qw.to(DEV), kw.to(DEV), EPS, d, cs.to(DEV), True)
    for i in (2, 5, 7):
        assert torch.equal(dev[i].cpu(), qkv[i])
    want, size = ref.norm_rope(qkv[:, :heads * d].reshape(t, heads, d), qw, EPS, pos, cs, True)
    check(q.reshape(t, heads, d), want, size, torch.bfloat16)


@pytest.mark.parametrize("heads,kv_heads,d,rot", [(32, 8, 128, 128), (24, 8, 64, 32), (3, 1, 96, 48),
                                                  (5, 2, 33, 10), (0, 2, 64, 64), (2, 1, 80, 32)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neox,page", [(True, 16), (False, 8), (True, 5)])
def test_append(heads, kv_heads, d, rot, dtype, neox, page):
    for t in (1, 45):
        qkv, (qw, kw), cs, pos = make(t, heads, kv_heads, d, rot, dtype, seed=t)
        pages = -(-t // page) + 4
        g = torch.Generator().manual_seed(page)
        slots = torch.randperm(pages * page, generator=g)[:t]
        if t > 10:
            slots[3] = -1                 # padding: not counted
            pos[4] = -1
            slots[4] = -1                 # the same with no position
            slots[6] = pages * page       # past the cache
            slots[7] = -2
            pos[9] = 512                  # a slot but no position
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        cache = torch.full((pages, 2, page, kv_heads, d), 9.0).to(dtype)
        dev, cache_d = qkv.to(DEV), cache.to(DEV)
        q, k, v = split(dev, heads, kv_heads, d)
        pe.qk_norm_rotary_append(pos.to(DEV), q, k, v, qw.to(DEV), kw.to(DEV), EPS, d, cs.to(DEV), neox,
                                 cache_d, slots.to(DEV), bad)
        assert bad.item() == (3 if t > 10 else 0)
        hq, hk, hv = split(qkv, heads, kv_heads, d)
        want, size = ref.norm_rope(hq.reshape(t, heads, d), qw, EPS, pos, cs, neox)
        check(q.reshape(t, heads, d), want, size, dtype)
        assert torch.equal(dev[:, heads * d:].cpu(), qkv[:, heads * d:])
        want, size = ref.norm_rope(hk.reshape(t, kv_heads, d), kw, EPS, pos, cs, neox)
        cache_h, left = cache_d.cpu(), torch.ones(pages, page, dtype=torch.bool)
        for i in range(t):
            s = int(slots[i])
            if 0 <= s < pages * page and 0 <= int(pos[i]) < 512:
                left[s // page, s % page] = False
                check(cache_h[s // page, 0, s % page], want[i], size[i], dtype)
                assert torch.equal(cache_h[s // page, 1, s % page].flatten(), hv[i])
        assert (cache_h.transpose(1, 2)[left] == 9).all()


def test_offsets_past_32_bits():
    """The last page of a cache of more than 2^32 elements."""
    page, kv_heads, d = 16, 8, 128
    pages = (1 << 32) // (2 * page * kv_heads * d) + 8
    cache = torch.zeros(pages, 2, page, kv_heads, d, dtype=torch.bfloat16, device=DEV)
    t = 3
    qkv, (qw, kw), cs, pos = make(t, 4, kv_heads, d, d, torch.bfloat16)
    slots = torch.tensor([pages * page - 1, 5, (pages - 1) * page])
    dev = qkv.to(DEV)
    q, k, v = split(dev, 4, kv_heads, d)
    pe.qk_norm_rotary_append(pos.to(DEV), q, k, v, qw.to(DEV), kw.to(DEV), EPS, d, cs.to(DEV), True, cache,
                             slots.to(DEV))
    _, hk, hv = split(qkv, 4, kv_heads, d)
    want, size = ref.norm_rope(hk.reshape(t, kv_heads, d), kw, EPS, pos, cs, True)
    for i, s in enumerate(slots.tolist()):
        check(cache[s // page, 0, s % page], want[i], size[i], torch.bfloat16)
        assert torch.equal(cache[s // page, 1, s % page].cpu().flatten(), hv[i])


def test_many_tokens_match_few():
    """The same tokens in one call and in pieces: the same bits."""
    t, heads, kv_heads, d = 3000, 12, 4, 128
    qkv, (qw, kw), cs, pos = make(t, heads, kv_heads, d, d, torch.bfloat16)
    args = [x.to(DEV) for x in (qw, kw)] + [EPS, d, cs.to(DEV), True]
    one, many = qkv.to(DEV), qkv.to(DEV)
    pe.qk_norm_rotary_embedding(pos.to(DEV), *split(one, heads, kv_heads, d)[:2], *args)
    for i in range(0, t, 250):
        q, k, _ = split(many[i:i + 250], heads, kv_heads, d)
        pe.qk_norm_rotary_embedding(pos[i:i + 250].to(DEV), q, k, *args)
    assert torch.equal(one, many)


@pytest.mark.parametrize("t,heads,kv_heads,d,rot,page", [
    (3301, 64, 8, 128, 128, 16), (5601, 50, 3, 96, 48, 5), (6203, 9, 4, 256, 256, 1), (9000, 0, 70, 64, 32, 8),
    (1301, 5, 3, 64, 32, 3)])
@pytest.mark.parametrize("dtype,cache_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                               (torch.float32, torch.float32)])
@pytest.mark.parametrize("neox", [True, False])
def test_many_tokens(t, heads, kv_heads, d, rot, page, dtype, cache_dtype, neox):
    """The kernel for many tokens, in place and with the append, against the one for few."""
    qkv, (qw, kw), cs, pos = make(t, heads, kv_heads, d, rot, dtype, cache_dtype=cache_dtype, pad=16)
    pages = -(-t // page) + 2
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:t]
    pos[::97], pos[5] = -1, 512
    slots[::97] = -1
    slots[11], slots[12], slots[t - 1] = -1, pages * page, -7  # 5, 12 and the last count
    qw, kw, cs, pos, slots = (x.to(DEV) for x in (qw, kw, cs, pos, slots))
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = []
    for few in (False, True):
        dev, both = qkv.to(DEV), qkv.to(DEV)
        cache = torch.full((pages, 2, page, kv_heads, d), 9.0, device=DEV).to(dtype)
        for a, b in ((i, min(t, i + 500)) for i in range(0, t, 500)) if few else ((0, t),):
            q, k, _ = split(dev[a:b], heads, kv_heads, d)
            pe.qk_norm_rotary_embedding(pos[a:b], q, k, qw, kw, EPS, d, cs, neox)
            q, k, v = split(both[a:b], heads, kv_heads, d)
            pe.qk_norm_rotary_append(pos[a:b], q, k, v, qw, kw, EPS, d, cs, neox, cache, slots[a:b], bad)
        assert bad.item() == (6 if few else 3)
        got.append((dev, both, cache))
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_row_of_zeros_and_nan():
    qkv, (qw, kw), cs, pos = make(3, 2, 1, 64, 64, torch.bfloat16)
    qkv[0] = 0
    qkv[1, 5] = float("nan")
    dev = qkv.to(DEV)
    q, k, _ = split(dev, 2, 1, 64)
    pe.qk_norm_rotary_embedding(pos.to(DEV), q, k, qw.to(DEV), kw.to(DEV), EPS, 64, cs.to(DEV), True)
    assert (dev[0] == 0).all()
    assert q[1, :64].isnan().all() and q[1, 64:].isfinite().all() and k[1].isfinite().all()


def test_in_a_graph_after_what_writes_its_positions():
    t, heads, kv_heads, d = 64, 8, 2, 128
    qkv, (qw, kw), cs, pos = make(t, heads, kv_heads, d, d, torch.bfloat16)
    w = [x.to(DEV) for x in (qw, kw)]
    cs_d, src, dev = cs.to(DEV), qkv.to(DEV), torch.empty_like(qkv, device=DEV)
    base, where = torch.zeros(t, dtype=torch.int64, device=DEV), torch.zeros(t, dtype=torch.int64, device=DEV)
    q, k, _ = split(dev, heads, kv_heads, d)

    def step():
        dev.copy_(src)
        torch.add(base, 1, out=where)
        pe.qk_norm_rotary_embedding(where, q, k, *w, EPS, d, cs_d, True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for shift in (0, 100, 300):
        base.copy_(pos // 2 + shift - 1)
        graph.replay()
        want, size = ref.norm_rope(qkv[:, :heads * d].reshape(t, heads, d), qw, EPS, pos // 2 + shift, cs, True)
        check(q.reshape(t, heads, d), want, size, torch.bfloat16)


def test_refusals():
    t, heads, kv_heads, d = 4, 4, 2, 64
    qkv, (qw, kw), cs, pos = make(t, heads, kv_heads, d, d, torch.bfloat16)
    dev, qw, kw, cs, pos = (x.to(DEV) for x in (qkv, qw, kw, cs, pos))
    q, k, v = split(dev, heads, kv_heads, d)
    cache = torch.zeros(4, 2, 16, kv_heads, d, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(t, device=DEV)
    plain, append = pe.qk_norm_rotary_embedding, pe.qk_norm_rotary_append
    for call, what in [
        (lambda: plain(pos, q, k, qw[:32], kw, EPS, d, cs, True), "q_weight"),
        (lambda: plain(pos, q, k, qw.float(), kw, EPS, d, cs, True), "share a float dtype"),
        (lambda: plain(pos.int(), q, k, qw, kw, EPS, d, cs, True), "int64"),
        (lambda: plain(pos[:3], q, k, qw, kw, EPS, d, cs, True), "entries for"),
        (lambda: plain(pos, q, k[:3], qw, kw, EPS, d, cs, True), "token counts"),
        (lambda: plain(pos, q, k, qw, kw, EPS, d, cs.half(), True), "cos_sin_cache"),
        (lambda: append(pos, q, k, v[:, :64], qw, kw, EPS, d, cs, True, cache, slots), "differ in shape"),
        (lambda: append(pos, q, k, v, qw, kw, EPS, d, cs, True, cache[:, :, :, :1].contiguous(), slots), "heads of"),
        (lambda: append(pos, q, k, v, qw, kw, EPS, d, cs, True, cache.half(), slots), "share a dtype"),
        (lambda: append(pos, q, k, v, qw, kw, EPS, d, cs, True, cache, slots[:3]), "slot_mapping"),
        (lambda: append(pos, q, k, v, qw, kw, EPS, d, cs, True, cache, slots.int()), "slot_mapping"),
        (lambda: append(pos, q, k, v, qw, kw, EPS, d, cs, True, cache, slots, torch.zeros(1)), "bad_tokens"),
    ]:
        with pytest.raises(RuntimeError, match=what):
            call()
