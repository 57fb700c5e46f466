"""CPU: in the example of a layer every call that can give up is given the word that tells, and it is looked at."""
from types import SimpleNamespace

import pytest
import torch

from examples import int8_layer_steps as ex


def test_every_call_tells(monkeypatch):
    layer = ex.Layer.__new__(ex.Layer)
    layer.fault = torch.zeros(1, dtype=torch.int32)
    for name in ("input_norm", "post_norm", "q_norm", "k_norm", "cache", "cos_sin"):
        setattr(layer, name, None)
    for name in ("qkv", "out", "gate_up", "down"):
        setattr(layer, name, (None, None))
    told = []
    tells = lambda name: lambda *a, fault_flags: told.append((name, fault_flags is layer.fault))  # noqa: E731
    monkeypatch.setattr(ex, "int8_ops", SimpleNamespace(
        rms_norm_quantise=lambda *a: None, quantise_rows=lambda *a: None, linear=tells("linear"),
        linear_residual=tells("linear_residual"), gate_up_silu=tells("gate_up_silu")))
    monkeypatch.setattr(ex, "pos_encoding_ops", SimpleNamespace(qk_norm_rotary_append=tells("append")))
    attention = SimpleNamespace(forward=lambda q, cache: q)
    ex.forward(layer, torch.zeros(2, ex.HIDDEN), SimpleNamespace(positions=None, slot_mapping=None), attention)
    assert told == [(n, True) for n in ("linear", "append", "linear_residual", "gate_up_silu", "linear_residual")]
    layer.check()
    layer.fault.fill_(1 << 30)
    with pytest.raises(RuntimeError, match="wait ran out"):
        layer.check()
    layer.check()
