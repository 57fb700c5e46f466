"""GPU: the 8-bit products' kernel for many tokens, on CTA pairs, against 64 bits.

It takes over from the cluster kernel where a call has more than a quarter as many tiles of 256 tokens by
128, 192 or 256 channels as there are SMs (37 of 148), so the widths here are in the thousands.
Tolerances are those of ``tests/test_int8_gpu.py``."""
import pytest
import torch

from oracle import int8_ref as ref
from paceserve_b200 import int8_ops
from tests.test_int8_gpu import DEV, F32, check_linear, half, make, silu_error

pytestmark = pytest.mark.gpu
BF16, F16, FP32 = torch.bfloat16, torch.float16, torch.float32


def check_gate_up(out, x, sx, w, sw, dtype):
    i = out.shape[1]
    y = ref.linear(x, sx, w, sw)
    gate = y[:, :i]
    # the gate is off by 3 * 2^-24 of itself, which moves silu by up to |gate| + 1 times that; where
    # e^-gate passes 2^126 the quotient is 0: what is lost is at most |gate| |up| 2^-126, with both below
    # 2^13 under 2^-100
    assert y.abs().max() < 2.0 ** 13
    want = ref.gate_up_silu(x, sx, w, sw)
    error = silu_error(gate) + 3 * F32 * (gate.abs() + 1) + 4 * F32
    least = torch.finfo(dtype).smallest_normal * half(dtype) + 2.0 ** -100
    assert ((out.double() - want).abs() <= (half(dtype) + error) * want.abs() + least).all()


@pytest.mark.parametrize("t,n,k", [
    (300, 2504, 512),                       # tiles of 128 channels
    (300, 2507, 512), (129, 5001, 272),     # rows that no vector store takes
    (300, 7011, 2048),                      # of 192
    (300, 9700, 4096), (300, 9703, 4112)])  # of 256, the last round's in halves
@pytest.mark.parametrize("dtype", [BF16, F16, FP32])
def test_strides_of_everything(t, n, k, dtype):
    """Rows of codes, weight, output and residual inside wider ones; what lies beside stays."""
    g = torch.Generator().manual_seed(t + n)
    x, sx, w, sw = make(g, t, n, k, dtype, pad=32)
    y = ref.linear(x, sx, w, sw)
    bias = torch.randn(n, generator=g).to(dtype).to(DEV)
    for shift in (0, 3):  # rows as they are, and a view that no vector store takes
        wide = torch.full((t, n + 16), 5.0, dtype=dtype, device=DEV)
        out = wide[:, shift:shift + n]
        beside = lambda: (wide[:, :shift] == 5).all() and (wide[:, shift + n:] == 5).all()  # noqa: E731
        int8_ops.linear(out, x, sx, w, sw)
        check_linear(out, y, y.abs(), dtype)
        assert beside()
        before = out.double()
        int8_ops.linear_residual(out, x, sx, w, sw)
        check_linear(out, y + before, y.abs() + before.abs(), dtype)
        assert beside()
        int8_ops.linear(out, x, sx, w, sw, bias)
        check_linear(out, y + bias.double(), y.abs() + bias.double().abs(), dtype)
        assert beside()


@pytest.mark.parametrize("t,i,k", [(300, 1252, 512), (300, 1253, 512), (300, 3001, 2048), (300, 4853, 4112)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_gate_up_strides(t, i, k, dtype):
    g = torch.Generator().manual_seed(t + i)
    x, sx, w, sw = make(g, t, 2 * i, k, dtype, pad=32)
    for shift in (0, 3):
        wide = torch.full((t, i + 16), 5.0, dtype=dtype, device=DEV)
        out = wide[:, shift:shift + i]
        int8_ops.gate_up_silu(out, x, sx, w, sw)
        check_gate_up(out, x, sx, w, sw, dtype)
        assert (wide[:, :shift] == 5).all() and (wide[:, shift + i:] == 5).all()


@pytest.mark.parametrize("k,pad", [(1111, 9), (4090, 6), (3, 13), (129, 15)])
def test_ragged_k_in_aligned_rows(k, pad):
    """What lies behind a row's k codes is not read into the sums."""
    g = torch.Generator().manual_seed(k)
    x, sx, w, sw = make(g, 300, 2512, k, FP32, pad)
    y = ref.linear(x, sx, w, sw)
    out = torch.empty(300, 2512, device=DEV)
    int8_ops.linear(out, x, sx, w, sw)
    check_linear(out, y, y.abs(), FP32)
    out = torch.empty(300, 1256, device=DEV)
    int8_ops.gate_up_silu(out, x, sx, w, sw)
    check_gate_up(out, x, sx, w, sw, FP32)


def test_largest_sums():
    """-128 x -128 over the longest K: 2^31 - 2^18, exactly."""
    t, n, k = 300, 2504, 131056  # k: a multiple of 16 below the limit
    x = torch.full((t, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    w[1], w[-1] = 127, 127
    out = torch.empty(t, n, device=DEV)
    int8_ops.linear(out, x, torch.ones(t, device=DEV), w, torch.ones(n, device=DEV))
    other = torch.tensor([1, n - 1], device=DEV)
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[other] = False
    assert (out[:, rest] == float(k << 14)).all()
    assert (out[:, other].double() + 128.0 * 127 * k).abs().max() <= F32 * 128 * 127 * k


@pytest.mark.parametrize("n,k", [(2504, 256), (2507, 256), (9700, 4096)])
def test_nan_scale_reaches_its_row_alone(n, k):
    g = torch.Generator().manual_seed(n)
    x, sx, w, sw = make(g, 300, n, k, BF16)
    y = ref.linear(x, sx, w, sw)
    sx[2] = sx[290] = float("nan")
    out = torch.empty(300, n, dtype=BF16, device=DEV)
    int8_ops.linear(out, x, sx, w, sw)
    bad = torch.zeros(300, dtype=torch.bool, device=DEV)
    bad[2] = bad[290] = True
    assert out[bad].isnan().all()
    check_linear(out[~bad], y[~bad], y[~bad].abs(), BF16)
