"""GPU: the 8-bit products' residual add past 2^31 outputs."""
import pytest
import torch

from oracle import int8_ref as ref
from paceserve_b200 import int8_ops
from tests.test_int8_gpu import DEV, check_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [32768, 32769])  # rows that vector stores take, and rows that none takes
def test_residual_past_32_bits(n):
    t, k, some = 66000, 128, 200
    g = torch.Generator(device=DEV).manual_seed(n)
    draw = lambda r: torch.randint(-127, 128, (r, k), generator=g, device=DEV, dtype=torch.int8)  # noqa: E731
    x, w = draw(t), draw(n)
    sx, sw = torch.rand(t, generator=g, device=DEV) / 127, torch.rand(n, generator=g, device=DEV) / 127
    residual = torch.randn(t, n, generator=g, device=DEV, dtype=torch.bfloat16)
    # the first rows, those about offset 2^31, and the last ones
    at = (1 << 31) // n - some // 2
    pieces = [slice(0, some), slice(at, at + some), slice(t - some, t)]
    before = [residual[p].double() for p in pieces]
    int8_ops.linear_residual(residual, x, sx, w, sw)
    for p, b in zip(pieces, before):
        y = ref.linear(x[p], sx[p], w, sw)
        check_linear(residual[p], y + b, y.abs() + b.abs(), torch.bfloat16)
