"""GPU: rows quantised to 8-bit integers and their products, against 64 bits.

Tolerances.  A code is the nearest integer to y / scale, so it is off by half a
step and by what fp32 makes of y and the quotient: 127 times a relative error.
A product's sum is exact; what follows are at most four fp32 roundings of 2^-24
(the sum as a float, two scales, bias or residual) and the output's half step.
"""
import pytest
import torch

from oracle import int8_ref as ref
from paceserve_b200 import int8_ops, quantise_weight

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# fp32 norm: up to 80 terms a thread and 10 in the tree, positive, each rounding at most 2^-24 of
# the sum, halved by the root; rsqrt and two products 2^-22: below 2^-18
NORM_ERROR = 2.0 ** -18
# silu * up: see silu_error
F32 = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def silu_error(g):
    """Relative error of fp32 silu(g) * u: the exponential's argument is off by |g| 2^-24 and the
    approximate forms by a few units more."""
    return (4 * g.abs() + 16) * F32


def inputs(g, rows, width, dtype, strided):
    x = torch.randn(rows, width + (8 if strided else 0), generator=g)
    x *= torch.exp(torch.randn(x.shape[1], generator=g))
    return x.to(dtype).to(DEV)[:, :width]


def check_codes(codes, scales, y, error):
    """`error`: relative error of fp32 y, a number or a tensor."""
    codes, scales, y = codes.cpu().double(), scales.cpu().double(), y.cpu()
    want = ref.scales_of(y)
    bad = want.isnan()
    assert torch.equal(bad, scales.isnan())
    assert (codes[bad] == 0).all()
    e = error if isinstance(error, float) else error.cpu()[~bad]
    most = e if isinstance(e, float) else e.amax(-1)
    assert ((scales[~bad] - want[~bad]).abs() <= (most + 2 * F32) * want[~bad]).all()
    steps = y[~bad] / want[~bad, None]
    m = most if isinstance(most, float) else most[:, None]
    assert ((codes[~bad] - steps).abs() <= 0.5 + 127 * (e + m + 4 * F32)).all()
    assert codes.abs().max() <= 127


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,strided", [
    (1, 4096, False), (3, 64, True), (5, 1, False), (7, 1111, False), (2, 8192, True), (2, 16392, False),
    (300, 256, False), (2, 20000, False), (4, 14336, False), (2, 32776, False), (160, 18432, True)])
def test_quantise_rows(dtype, rows, width, strided):
    g = torch.Generator().manual_seed(width)
    x = inputs(g, rows, width, dtype, strided)
    codes = torch.full((rows, width + 16), 99, dtype=torch.int8, device=DEV)[:, :width]
    scales = torch.empty(rows, device=DEV)
    int8_ops.quantise_rows(codes, scales, x)
    check_codes(codes, scales, x.double(), 0.0)
    # the definition in fp32, to the bit: IEEE division and rounding to even
    xf = x.float().cpu()
    s = (xf.abs().amax(-1) / 127).clamp_min(ref.LEAST_SCALE)
    assert torch.equal(scales.cpu(), s)
    assert torch.equal(codes.cpu().float(), (xf / s[:, None]).round())


@pytest.mark.parametrize("dtype", TYPES)
def test_quantise_extremes(dtype):
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = torch.zeros(9, 128)
    rows[1], rows[2, 5] = big, -big
    rows[3] = tiny
    rows[4, :2] = torch.tensor([float("inf"), 1.0])
    rows[5, 7] = float("nan")
    rows[6, 1] = -float("inf")
    rows[7] = torch.arange(128) - 64.0
    rows[7, 0] = 127.0  # scale 1: whole numbers
    rows[8, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])  # ties to even
    x = rows.to(dtype).to(DEV)
    codes = torch.empty(9, 128, dtype=torch.int8, device=DEV)
    scales = torch.empty(9, device=DEV)
    int8_ops.quantise_rows(codes, scales, x)
    check_codes(codes, scales, x.double(), 0.0)
    c = codes.cpu()
    assert (c[0] == 0).all() and scales[0].item() == ref.LEAST_SCALE
    assert (c[1] == 127).all() and c[2, 5] == -127
    assert scales[[4, 5, 6]].isnan().all() and (c[4:7] == 0).all()
    assert torch.equal(c[7].float(), rows[7])
    assert c[8, :4].tolist() == [127, 0, 2, -2]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,strided", [
    (1, 4096, False), (3, 64, True), (5, 7, False), (2, 1111, False), (130, 8192, False), (2, 20000, False),
    (2, 16384, False), (160, 18432, True)])
@pytest.mark.parametrize("add", [False, True])
def test_rms_norm_quantise(dtype, rows, width, strided, add):
    g = torch.Generator().manual_seed(width + add)
    x = inputs(g, rows, width, dtype, strided)
    res = inputs(g, rows, width, dtype, strided) if add else None
    w = (1 + torch.randn(width, generator=g) / 4).to(dtype).to(DEV)
    r = (x + res) if add else x  # one rounding, as the residual stream is held
    codes = torch.empty(rows, width, dtype=torch.int8, device=DEV)
    scales = torch.empty(rows, device=DEV)
    before = x.clone()
    int8_ops.rms_norm_quantise(codes, scales, x, w, 1e-5, res)
    assert torch.equal(x, before)
    if add:
        assert torch.equal(res, r)
    check_codes(codes, scales, ref.normed(r, w, 1e-5), NORM_ERROR)


def test_rms_norm_quantise_row_of_zeros_and_nan():
    x = torch.zeros(3, 256, device=DEV, dtype=torch.bfloat16)
    x[1, 3] = float("nan")
    x[2, 3] = float("inf")
    w = torch.ones(256, device=DEV, dtype=torch.bfloat16)
    codes = torch.empty(3, 256, dtype=torch.int8, device=DEV)
    scales = torch.empty(3, device=DEV)
    int8_ops.rms_norm_quantise(codes, scales, x, w, 1e-6)
    assert scales[0].item() == ref.LEAST_SCALE and scales[1:].isnan().all()
    assert (codes == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,strided", [
    (1, 14336, False), (3, 64, True), (5, 7, False), (2, 1111, False), (65, 4096, False), (2, 20000, False),
    (2, 32776, False), (160, 18432, True)])
def test_silu_and_mul_quantise(dtype, rows, width, strided):
    g = torch.Generator().manual_seed(width)
    x = inputs(g, rows, 2 * width, dtype, strided)
    codes = torch.empty(rows, width, dtype=torch.int8, device=DEV)
    scales = torch.empty(rows, device=DEV)
    int8_ops.silu_and_mul_quantise(codes, scales, x)
    check_codes(codes, scales, ref.silu_mul(x), silu_error(x[:, :width].double()))


def make(g, t, n, k, dtype, pad=0):
    """Codes and weights of every size, scales, on the GPU; rows `pad` bytes longer than k."""
    draw = lambda r: torch.randint(-127, 128, (r, k + pad), generator=g).to(torch.int8).to(DEV)[:, :k]  # noqa: E731
    x, w = draw(t), draw(n)
    sx = torch.exp(torch.randn(t, generator=g)).to(DEV) / 127
    sw = torch.exp(torch.randn(n, generator=g)).to(DEV) / (127 * k ** 0.5)
    return x, sx, w, sw


def check_linear(out, want, size, dtype):
    """size: the magnitudes that were added."""
    tol = half(dtype) * want.abs() + 5 * F32 * size + torch.finfo(dtype).smallest_normal * half(dtype)
    d = (out.double() - want).abs()
    assert (d <= tol).all(), float((d - tol).max())


SHAPES = [
    # t, n, k: every way the tokens lie (to 32, to 128, more), few and many tiles, short and long K
    (1, 6144, 4096), (1, 128, 128), (1, 1, 16), (3, 130, 48), (16, 4096, 14336), (17, 200, 256),
    (32, 6144, 4096), (33, 72, 8192), (64, 4096, 14336), (65, 4096, 4096), (128, 1000, 2048),
    (129, 300, 4096), (256, 4096, 4096), (300, 264, 14336), (777, 1003, 1040), (520, 4096, 1152), (200, 6144, 656), (1000, 1500, 304), (1000, 6144, 4096),
    # the last round's few tiles in halves, whole K blocks and not
    (300, 9700, 4096), (300, 9700, 4112), (601, 8900, 5008),
]


@pytest.mark.parametrize("t,n,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_linear(t, n, k, dtype):
    g = torch.Generator().manual_seed(t * 7 + n + k)
    x, sx, w, sw = make(g, t, n, k, dtype)
    bias = torch.randn(n, generator=g).to(dtype).to(DEV)
    y = ref.linear(x, sx, w, sw)
    out = torch.full((t, n), 7.0, dtype=dtype, device=DEV)
    int8_ops.linear(out, x, sx, w, sw)
    check_linear(out, y, y.abs(), dtype)
    first = out.clone()
    int8_ops.linear(out, x, sx, w, sw, bias)
    check_linear(out, y + bias.double(), y.abs() + bias.double().abs(), dtype)
    res = torch.randn(t, n, generator=g).to(dtype).to(DEV)
    want = y + res.double()
    size = y.abs() + res.double().abs()
    int8_ops.linear_residual(res, x, sx, w, sw)
    check_linear(res, want, size, dtype)
    for _ in range(3):  # whoever finishes a tile, the bits are the same
        int8_ops.linear(out, x, sx, w, sw)
        assert torch.equal(out, first)


@pytest.mark.parametrize("t,i,k", [(1, 14336, 4096), (2, 64, 64), (20, 200, 4096), (50, 1024, 2048),
                                   (128, 700, 1024), (130, 130, 256), (512, 14336, 4096), (601, 2056, 14336),
                                   (300, 4850, 4112)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gate_up_silu(t, i, k, dtype):
    g = torch.Generator().manual_seed(t + i + k)
    x, sx, w, sw = make(g, t, 2 * i, k, dtype)
    want = ref.gate_up_silu(x, sx, w, sw)
    gate = ref.linear(x, sx, w[:i], sw[:i])
    out = torch.empty(t, i, dtype=dtype, device=DEV)
    int8_ops.gate_up_silu(out, x, sx, w, sw)
    # the gate is off by 3 * 2^-24 of itself, which moves silu by up to |gate| + 1 times that
    error = silu_error(gate) + 3 * F32 * (gate.abs() + 1) + 4 * F32
    tol = (half(dtype) + error) * want.abs() + 2.0 ** -100 + torch.finfo(dtype).smallest_normal * half(dtype)
    d = (out.double() - want).abs()
    fine = want.abs() < torch.finfo(dtype).max
    assert fine.float().mean() > 0.9 and (d <= tol)[fine].all()


@pytest.mark.parametrize("t,n,k,pad", [(1, 77, 1111, 0), (70, 1003, 1111, 0), (33, 65, 4096, 3),
                                       (5, 130, 64, 8), (200, 70, 3, 0), (2, 3, 1, 0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_tma_does_not_take(t, n, k, pad, dtype):
    g = torch.Generator().manual_seed(t + n + k)
    x, sx, w, sw = make(g, t, 2 * n, k, dtype, pad)
    y = ref.linear(x, sx, w, sw)
    bias = torch.randn(2 * n, generator=g).to(dtype).to(DEV)
    out = torch.empty(t, 2 * n, dtype=dtype, device=DEV)
    int8_ops.linear(out, x, sx, w, sw, bias)
    check_linear(out, y + bias.double(), y.abs() + bias.double().abs(), dtype)
    res = torch.randn(t, 2 * n, generator=g).to(dtype).to(DEV)
    want = y + res.double()
    size = y.abs() + res.double().abs()
    int8_ops.linear_residual(res, x, sx, w, sw)
    check_linear(res, want, size, dtype)
    out = torch.empty(t, n, dtype=dtype, device=DEV)
    int8_ops.gate_up_silu(out, x, sx, w, sw)
    want = ref.gate_up_silu(x, sx, w, sw)
    error = silu_error(y[:, :n]) + 3 * F32 * (y[:, :n].abs() + 1) + 4 * F32
    # below the smallest normal number values are eps apart in its units: fp16 2^-14 * 2^-10 = 2^-24,
    # so half a step is smallest_normal * eps / 2 (2^-25)
    # Where 1 + e^-gate passes 2^126, the approximate quotient is 0: what is lost is at most
    # |gate| |up| 2^-126, with both below 2^13 under 2^-100
    assert y.abs().max() < 2.0 ** 13
    least = torch.finfo(dtype).smallest_normal * half(dtype) + 2.0 ** -100
    assert ((out.double() - want).abs() <= (half(dtype) + error) * want.abs() + least).all()


@pytest.mark.parametrize("t", [1, 20, 100, 300])
@pytest.mark.parametrize("k,pad", [(1111, 9), (4090, 6), (3, 13), (129, 15)])
def test_ragged_k_in_aligned_rows(t, k, pad):
    """What lies behind a row's k codes is not read into the sums."""
    g = torch.Generator().manual_seed(t + k)
    dtype = torch.float32
    x, sx, w, sw = make(g, t, 268, k, dtype, pad)
    y = ref.linear(x, sx, w, sw)
    out = torch.empty(t, 268, dtype=dtype, device=DEV)
    int8_ops.linear(out, x, sx, w, sw)
    check_linear(out, y, y.abs(), dtype)
    out = torch.empty(t, 134, dtype=dtype, device=DEV)
    int8_ops.gate_up_silu(out, x, sx, w, sw)
    gate = y[:, :134]
    error = silu_error(gate) + 3 * F32 * (gate.abs() + 1) + 4 * F32
    want = ref.gate_up_silu(x, sx, w, sw)
    # below the smallest normal number half a step is smallest_normal * eps / 2.  Where e^-gate passes
    # 2^128 in fp32 (gate below -88.7), the quotient is 0: what is lost is |gate| e^gate |up|, at most
    # |gate| |up| 2^-127, with both below 2^13 under 2^-100
    assert y.abs().max() < 2.0 ** 13
    least = torch.finfo(dtype).smallest_normal * half(dtype) + 2.0 ** -100
    assert ((out.double() - want).abs() <= (half(dtype) + error) * want.abs() + least).all()


@pytest.mark.parametrize("t", [1, 40, 100, 300])
def test_strides_of_everything(t):
    """Rows of codes, weight, output and residual inside wider ones; what lies beside stays."""
    g = torch.Generator().manual_seed(t)
    n, k = 264, 512
    x, sx, w, sw = make(g, t, n, k, torch.bfloat16, pad=32)
    y = ref.linear(x, sx, w, sw)
    for shift in (0, 3):  # aligned rows, and a view that no vector store takes
        wide = torch.full((t, n + 16), 5.0, dtype=torch.bfloat16, device=DEV)
        out = wide[:, shift:shift + n]
        int8_ops.linear(out, x, sx, w, sw)
        check_linear(out, y, y.abs(), torch.bfloat16)
        assert (wide[:, :shift] == 5).all() and (wide[:, shift + n:] == 5).all()
        before = out.double()
        int8_ops.linear_residual(out, x, sx, w, sw)
        check_linear(out, y + before, y.abs() + before.abs(), torch.bfloat16)
        assert (wide[:, :shift] == 5).all() and (wide[:, shift + n:] == 5).all()


def test_largest_sums():
    """-128 x -128 over the longest K: 2^31 - 2^14, exactly."""
    k = 131056  # a multiple of 16 below the limit
    for t in (2, 200):
        x = torch.full((t, k), -128, dtype=torch.int8, device=DEV)
        w = torch.full((8, k), -128, dtype=torch.int8, device=DEV)
        w[1] = 127
        one = torch.ones(t, device=DEV)
        out = torch.empty(t, 8, device=DEV)
        int8_ops.linear(out, x, one, w, torch.ones(8, device=DEV))
        assert (out[:, 0] == float(k << 14)).all()
        assert (out[:, 1].double() - -128.0 * 127 * k).abs().max() <= F32 * 128 * 127 * k


def test_nan_scale_reaches_its_row_alone():
    g = torch.Generator().manual_seed(0)
    for t in (4, 90, 300):
        x, sx, w, sw = make(g, t, 256, 256, torch.bfloat16)
        sx[2] = float("nan")
        out = torch.empty(t, 256, dtype=torch.bfloat16, device=DEV)
        int8_ops.linear(out, x, sx, w, sw)
        assert out[2].isnan().all() and out.isnan().any(-1).sum() == 1


@pytest.mark.parametrize("n", [32768, 32769])
def test_offsets_past_32_bits(n):
    """Over 2^31 outputs: the last rows are those of a call with them alone."""
    t, k, last = 66000, 128, 200
    x = torch.randint(-127, 128, (t, k), device=DEV, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), device=DEV, dtype=torch.int8)
    sx, sw = torch.rand(t, device=DEV) / 127, torch.rand(n, device=DEV) / 127
    out = torch.zeros(t, n, dtype=torch.bfloat16, device=DEV)
    int8_ops.linear(out, x, sx, w, sw)
    want = ref.linear(x[-last:], sx[-last:], w, sw)
    check_linear(out[-last:], want, want.abs(), torch.bfloat16)
    codes = torch.zeros(t, n, dtype=torch.int8, device=DEV)
    scales = torch.zeros(t, device=DEV)
    int8_ops.quantise_rows(codes, scales, out)
    check_codes(codes[-last:], scales[-last:], out[-last:].double(), 0.0)
    int8_ops.linear_residual(out, x, sx, w, sw)
    assert out[0].isfinite().all() and not torch.equal(out[-1].double(), want[-1])


def test_no_tokens():
    x = torch.empty(0, 64, dtype=torch.int8, device=DEV)
    s = torch.empty(0, device=DEV)
    w = torch.zeros(32, 64, dtype=torch.int8, device=DEV)
    sw = torch.ones(32, device=DEV)
    int8_ops.quantise_rows(x, s, torch.empty(0, 64, device=DEV))
    int8_ops.linear(torch.empty(0, 32, device=DEV), x, s, w, sw)
    int8_ops.gate_up_silu(torch.empty(0, 16, device=DEV), x, s, w, sw)


@pytest.mark.parametrize("t", [1, 64, 100, 256, 300])
def test_two_streams_and_graphs(t):
    """Calls on two streams at once, and in two graphs replayed at once."""
    g = torch.Generator().manual_seed(t)
    cases = []
    for i in range(2):
        x, sx, w, sw = make(g, t, 4096, 4096, torch.bfloat16)
        out = torch.empty(t, 4096, dtype=torch.bfloat16, device=DEV)
        int8_ops.linear(out, x, sx, w, sw)
        cases.append((x, sx, w, sw, out, out.clone()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (x, sx, w, sw, out, _) in zip(streams, cases):
            with torch.cuda.stream(s):
                int8_ops.linear(out, x, sx, w, sw)
    torch.cuda.synchronize()
    for c in cases:
        assert torch.equal(c[4], c[5])
        c[4].zero_()
    graphs = []
    for x, sx, w, sw, out, _ in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(3):
                int8_ops.linear(out, x, sx, w, sw)
        graphs.append(graph)
    for _ in range(10):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for c in cases:
        assert torch.equal(c[4], c[5])


def test_quantised_weight_near_the_linear():
    """x @ w^T through both quantisations: each code is off by half a step at most."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(9, 512, generator=g).bfloat16().to(DEV)
    w = torch.randn(300, 512, generator=g).bfloat16().to(DEV)
    codes, sw = quantise_weight(w)
    cx = torch.empty(9, 512, dtype=torch.int8, device=DEV)
    sx = torch.empty(9, device=DEV)
    int8_ops.quantise_rows(cx, sx, x)
    out = torch.empty(9, 300, device=DEV)
    int8_ops.linear(out, cx, sx, codes, sw)
    # |x w - x' w'| <= |x - x'| |w| + |x'| |w - w'|, summed
    bound = 0.501 * (sx.double()[:, None] * w.double().abs().sum(-1)
                     + (cx.double().abs().sum(-1) * sx.double())[:, None] * sw.double())
    assert ((out.double() - x.double() @ w.double().T).abs() <= bound).all()


@pytest.mark.parametrize("n,k", [(5, 500), (1, 77), (3, 64)])
def test_quantised_weight_rows_are_aligned(n, k):
    g = torch.Generator().manual_seed(k)
    w = torch.randn(n, k, generator=g).to(DEV)
    codes, scales = quantise_weight(w)
    assert codes.shape == (n, k) and codes.stride(0) % 16 == 0 and codes.data_ptr() % 16 == 0
    check_codes(codes, scales, w.double(), 0.0)


def test_refusals():
    x = torch.zeros(4, 64, dtype=torch.int8, device=DEV)
    sx, sw = torch.ones(4, device=DEV), torch.ones(32, device=DEV)
    w = torch.zeros(32, 64, dtype=torch.int8, device=DEV)
    out = torch.empty(4, 32, dtype=torch.bfloat16, device=DEV)
    for args, what in [
        ((out[:, :31], x, sx, w, sw), "shapes do not match"),
        ((out, x[:, :48], sx, w, sw), "shapes do not match"),
        ((out, x, sx[:3], w, sw), "token_scales"),
        ((out, x, sx, w, sw.double()), "channel_scales"),
        ((out, x.float(), sx, w, sw), "int8"),
        ((out.int(), x, sx, w, sw), "float32, float16 or bfloat16"),
        ((out, x, sx, w.cpu(), sw), "different devices"),
        ((out, x, sx, w, sw, torch.ones(32, device=DEV)), "bias"),
    ]:
        with pytest.raises(RuntimeError, match=what):
            int8_ops.linear(*args)
    with pytest.raises(RuntimeError, match="gate as up"):
        int8_ops.gate_up_silu(out[:, :15], x, sx, w[:31], sw[:31])
    with pytest.raises(RuntimeError, match="do not match input"):
        int8_ops.quantise_rows(x, sx, torch.zeros(4, 63, device=DEV))
    with pytest.raises(RuntimeError, match="do not match input"):
        int8_ops.silu_and_mul_quantise(x, sx, torch.zeros(4, 64, device=DEV))
    with pytest.raises(RuntimeError, match="residual shape"):
        int8_ops.rms_norm_quantise(x, sx, torch.zeros(4, 64, device=DEV), torch.ones(64, device=DEV), 1e-5,
                                   torch.zeros(3, 64, device=DEV))
    long = torch.zeros(1, 131072, dtype=torch.int8, device=DEV)
    with pytest.raises(RuntimeError, match="32 bits"):
        int8_ops.linear(torch.empty(1, 1, device=DEV), long, sx[:1], long, sw[:1])
