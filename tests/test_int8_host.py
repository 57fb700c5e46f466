"""CPU: the new entry points refuse what they cannot run before any GPU work."""
import pytest
import torch

from paceserve_b200 import cabi, int8_ops, kv_transfer_ops, pos_encoding_ops
from tests.test_cabi import _expect
from tests.test_shim_host import _params

BAD, LARGE = cabi.PACE_ERR_INVALID_ARGUMENT, cabi.PACE_ERR_TOO_LARGE


def test_signatures():
    assert _params(int8_ops.quantise_rows) == ["codes", "scales", "input"]
    assert _params(int8_ops.rms_norm_quantise) == ["codes", "scales", "input", "weight", "epsilon", "residual"]
    assert _params(int8_ops.linear)[:6] == ["out", "codes", "token_scales", "weight", "channel_scales", "bias"]
    assert _params(int8_ops.gate_up_silu)[:5] == ["out", "codes", "token_scales", "weight", "channel_scales"]
    assert _params(pos_encoding_ops.qk_norm_rotary_append)[-4:] == ["paged_kv_cache", "slot_mapping",
                                                                  "bad_tokens", "fault_flags"]
    assert _params(kv_transfer_ops.build_step_tables)[:4] == ["block_tables", "seq_lens", "new_lens", "page_size"]


def test_cpu_tensors_rejected():
    x, s = torch.zeros(4, 64, dtype=torch.int8), torch.ones(4)
    i = torch.zeros(4, dtype=torch.int32)
    calls = [
        lambda: int8_ops.quantise_rows(x, s, torch.zeros(4, 64)),
        lambda: int8_ops.rms_norm_quantise(x, s, torch.zeros(4, 64), torch.ones(64), 1e-5),
        lambda: int8_ops.silu_and_mul_quantise(x, s, torch.zeros(4, 128)),
        lambda: int8_ops.linear(torch.zeros(4, 4), x, s, x, s),
        lambda: int8_ops.linear_residual(torch.zeros(4, 4), x, s, x, s),
        lambda: int8_ops.gate_up_silu(torch.zeros(4, 2), x, s, x, s),
        lambda: pos_encoding_ops.qk_norm_rotary_embedding(
            torch.zeros(4, dtype=torch.long), torch.zeros(4, 64), torch.zeros(4, 64), torch.ones(64),
            torch.ones(64), 1e-5, 64, torch.zeros(8, 64), True),
        lambda: kv_transfer_ops.release_pages(torch.zeros(4, 2, dtype=torch.int32), i, i, 16, i, i, i, i),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()


def test_int8_argument_errors():
    lib = cabi.load()
    bf = cabi.PACE_BF16
    linear = lambda t, n, k, xs, ws, os, p=None: lib.pace_int8_linear(  # noqa: E731
        p, p, p, p, p, None, None, t, n, k, xs, ws, os, 0, bf, None, None)
    _expect(linear(-1, 8, 16, 16, 16, 8), BAD, "bad shape")
    _expect(linear(4, 0, 16, 16, 16, 8), BAD, "bad shape")
    _expect(linear((1 << 29) + 1, 8, 16, 16, 16, 8), BAD, "bad shape")
    _expect(linear(4, (1 << 29) + 1, 16, 16, 16, 1 << 30), BAD, "bad shape")
    _expect(linear(4, 8, 16, 15, 16, 8), BAD, "row stride")
    _expect(linear(4, 8, 16, 16, 16, 7), BAD, "row stride")
    _expect(linear(4, 8, 131072, 131072, 131072, 8), LARGE, "32 bits")
    _expect(linear(4, 8, 16, 16, 16, 8), BAD, "null pointer")
    assert linear(0, 8, 16, 16, 16, 8) == 0
    quant = lambda t, w, xs, cs: lib.pace_quantise_rows(None, None, None, t, w, xs, cs, bf, None)  # noqa: E731
    _expect(quant(-1, 8, 8, 8), BAD, "bad shape")
    _expect(quant(2, (1 << 30) + 1, 1 << 31, 1 << 31), BAD, "bad shape")
    _expect(quant(2, 8, 7, 8), BAD, "row stride")
    _expect(quant(2, 8, 8, 8), BAD, "null pointer")
    _expect(lib.pace_silu_and_mul_quantise(None, None, None, 2, 8, 15, 8, bf, None), BAD, "row stride")
    _expect(lib.pace_quantise_rows(64, 64, 64, 2, 8, 8, 8, cabi.PACE_I32, None),
            cabi.PACE_ERR_UNSUPPORTED_DTYPE, "dtype")


def test_head_argument_errors():
    lib = cabi.load()
    call = lambda t, h, hk, d, qs, ks, rot, pos: lib.pace_qk_norm_rotary_embedding(  # noqa: E731
        None, None, None, None, None, 1e-5, t, h, hk, d, qs, ks, None, cabi.PACE_F32, rot, pos, 1,
        cabi.PACE_BF16, None, None)
    _expect(call(-1, 8, 2, 64, 512, 128, 64, 16), BAD, "bad shape")
    _expect(call(2, 1 << 25, 2, 64, 1 << 31, 128, 64, 16), BAD, "bad shape")
    _expect(call(2, 8, 2, 64, 511, 128, 64, 16), BAD, "row stride")
    _expect(call(2, 8, 2, 64, 512, 128, 63, 16), BAD, "rot_dim")
    _expect(call(2, 8, 2, 64, 512, 128, 66, 16), BAD, "rot_dim")
    _expect(call(2, 8, 2, 64, 512, 128, 64, 0), BAD, "empty cos_sin_cache")
    _expect(call(2, 8, 2, 64, 512, 128, 64, 16), BAD, "null pointer")
    assert call(0, 8, 2, 64, 512, 128, 64, 16) == 0
    append = lambda pages, page: lib.pace_qk_norm_rotary_append(  # noqa: E731
        None, None, None, None, None, None, 1e-5, 2, 8, 2, 64, 512, 128, 128, None, cabi.PACE_F32, 64, 16,
        1, None, pages, page, None, None, cabi.PACE_BF16, None, None)
    _expect(append(-1, 16), BAD, "bad cache shape")
    _expect(append(4, 0), BAD, "bad cache shape")
    _expect(append(4, 16), BAD, "null pointer")


def test_table_argument_errors():
    lib = cabi.load()
    build = lambda r, page, stride, blocks, tokens: lib.pace_build_step_tables(  # noqa: E731
        None, stride, blocks, None, None, r, page, None, 4, None, None, None, None, 4, None, None, None,
        None, tokens, None, None, None)
    _expect(build(-1, 16, 4, 4, 4), BAD, "bad shape")
    _expect(build(2, 0, 4, 4, 4), BAD, "bad shape")
    _expect(build(2, 16, 3, 4, 4), BAD, "row stride")
    _expect(build(8193, 16, 4, 4, 4), LARGE, "at most 8192")
    _expect(build(2, 16, 4, 4, 1 << 31), LARGE, "2^31")
    _expect(build(2, 16, 4, 4, 4), BAD, "null pointer")
    _expect(lib.pace_release_pages(None, 4, 4, None, None, 2, 16, None, 4, None, None, None, None), BAD,
            "null pointer")
