"""GPU: paged attention and the quantised cache where inputs are at an edge.

Tolerances are those derived in ``test_attention_gpu.py``.
"""
import pytest
import torch

from paceserve_b200.attention import PagedAttention
from tests.test_attention_gpu import DEV, Step

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
