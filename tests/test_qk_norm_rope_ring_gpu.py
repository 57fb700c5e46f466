"""GPU: the head norms' kernel for many tokens, and two heads a thread, against 64 bits.

The kernel for many tokens takes rows of 8 KB and more, 64 MB of them: 16-bit rows of every shape here
pass that in place and with the append.  Between 257 tokens and that, a thread has two heads.
Tolerances are those of ``tests/test_qk_norm_rope_gpu.py``."""
import pytest
import torch

from oracle import heads_ref as ref
from paceserve_b200 import pos_encoding_ops as pe
from tests.test_qk_norm_rope_gpu import DEV, EPS, make, split

pytestmark = pytest.mark.gpu
BF16, F16, FP32 = torch.bfloat16, torch.float16, torch.float32


def check(got, want, size, dtype):
    f = torch.finfo(dtype)
    tol = f.eps / 2 * want.abs() + 2.0 ** -18 * size + f.smallest_normal * f.eps / 2
    assert ((got.double() - want).abs() <= tol).all()


def run(t, heads, kv_heads, d, rot, page, dtype, cache_dtype, neox):
    qkv, (qw, kw), cs, pos = make(t, heads, kv_heads, d, rot, dtype, seed=t, cache_dtype=cache_dtype, pad=16)
    pages = -(-t // page) + 2
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:t]
    pos[::97], pos[5] = -1, 512
    slots[::97] = -1
    slots[11], slots[12], slots[t - 1] = -1, pages * page, -7  # 5, 12 and the last count
    qkv, qw, kw, cs, pos, slots = (x.to(DEV) for x in (qkv, qw, kw, cs, pos, slots))
    hq, hk, hv = split(qkv, heads, kv_heads, d)
    want_q = ref.norm_rope(hq.reshape(t, heads, d), qw, EPS, pos, cs, neox)
    want_k = ref.norm_rope(hk.reshape(t, kv_heads, d), kw, EPS, pos, cs, neox)
    after = (heads + kv_heads) * d
    # in place
    dev = qkv.clone()
    q, k, _ = split(dev, heads, kv_heads, d)
    fault = torch.zeros(1, dtype=torch.int32, device=DEV)
    pe.qk_norm_rotary_embedding(pos, q, k, qw, kw, EPS, d, cs, neox, fault)
    check(q.reshape(t, heads, d), *want_q, dtype)
    check(k.reshape(t, kv_heads, d), *want_k, dtype)
    assert torch.equal(dev[:, after:], qkv[:, after:])
    # with the append
    dev = qkv.clone()
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache = torch.full((pages, 2, page, kv_heads, d), 9.0, device=DEV).to(dtype)
    q, k, v = split(dev, heads, kv_heads, d)
    pe.qk_norm_rotary_append(pos, q, k, v, qw, kw, EPS, d, cs, neox, cache, slots, bad, fault)
    assert bad.item() == 3 and fault.item() == 0
    check(q.reshape(t, heads, d), *want_q, dtype)
    assert torch.equal(dev[:, heads * d:], qkv[:, heads * d:])
    goes = (slots >= 0) & (slots < pages * page) & (pos >= 0) & (pos < 512)
    flat = cache.transpose(0, 1).reshape(2, pages * page, kv_heads, d)
    check(flat[0, slots[goes]], want_k[0][goes], want_k[1][goes], dtype)
    assert torch.equal(flat[1, slots[goes]].reshape(-1, kv_heads * d), hv[goes])
    left = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    left[slots[goes]] = False
    assert (flat[:, left] == 9).all()


TYPES = [(BF16, FP32), (F16, F16), (FP32, FP32)]


@pytest.mark.parametrize("t,heads,kv_heads,d,rot,page", [
    (3801, 64, 8, 128, 128, 16),  # a token a stage of the ring
    (6701, 50, 3, 96, 48, 5),     # two; idle lanes
    (8001, 12, 4, 256, 256, 1),   # four in place, two with the append
    (9001, 0, 70, 64, 32, 8)])
@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("neox", [True, False])
def test_ring(t, heads, kv_heads, d, rot, page, dtype, cache_dtype, neox):
    run(t, heads, kv_heads, d, rot, page, dtype, cache_dtype, neox)


@pytest.mark.parametrize("heads,kv_heads,d,rot", [(5, 3, 64, 32), (7, 1, 96, 96), (1, 1, 128, 64), (0, 3, 64, 64)])
@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("neox", [True, False])
def test_two_heads_a_thread(heads, kv_heads, d, rot, dtype, cache_dtype, neox):
    for t in (257, 1301):
        run(t, heads, kv_heads, d, rot, 3, dtype, cache_dtype, neox)
