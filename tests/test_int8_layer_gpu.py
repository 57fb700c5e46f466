"""GPU: the 8-bit projections, head norms and step tables as a layer's steps use them together.

Each operator of the example is checked against 64 bits on what it was given, so that the tolerances
are those of one operator."""
import torch
import pytest

from examples import int8_layer_steps as ex
from oracle import attention_ref, heads_ref, int8_ref
from tests.test_int8_gpu import F32, NORM_ERROR, check_codes, check_linear, half, silu_error
from tests.test_qk_norm_rope_gpu import check as check_heads

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def split(qkv):
    return qkv.split([ex.HEADS * ex.HEAD_DIM, ex.KV_HEADS * ex.HEAD_DIM, ex.KV_HEADS * ex.HEAD_DIM], 1)


def test_steps():
    layer, tables, steps = ex.main()
    rows = [[], []]  # every token's key and value of each request, by position
    for s in steps:
        append_indptr, kv_indptr, kv_indices, last, owners, positions, slots = [x.cpu() for x in s["tables"]]
        t = sum(s["new"])
        # tables
        assert append_indptr.tolist() == [0, s["new"][0], t]
        want = [(b, p) for b in range(2) for p in range(s["lens"][b], s["lens"][b] + s["new"][b])]
        assert list(zip(owners.tolist()[:t], positions.tolist()[:t])) == want
        assert (owners[t:] == -1).all() and (slots[t:] == -1).all() and (positions[t:] == -1).all()
        used = kv_indices[:kv_indptr[-1]].tolist()
        assert len(set(used)) == len(used)
        # projections in
        check_codes(s["in_codes"], s["in_scales"], int8_ref.normed(s["hidden"], layer.input_norm, ex.EPS), NORM_ERROR)
        y = int8_ref.linear(s["in_codes"], s["in_scales"], *layer.qkv)
        check_linear(s["qkv"], y, y.abs(), BF16)
        # heads and cache
        q, k, v = (x.cpu() for x in split(s["qkv"]))
        pos = positions[:t]
        want, size = heads_ref.norm_rope(q.reshape(t, ex.HEADS, ex.HEAD_DIM), layer.q_norm.cpu(), ex.EPS, pos,
                                         layer.cos_sin.cpu(), True)
        check_heads(s["query"].reshape(t, ex.HEADS, ex.HEAD_DIM), want, size, BF16)
        want, size = heads_ref.norm_rope(k.reshape(t, ex.KV_HEADS, ex.HEAD_DIM), layer.k_norm.cpu(), ex.EPS, pos,
                                         layer.cos_sin.cpu(), True)
        cache = s["cache"].cpu()
        at, place = slots[:t] // ex.PAGE, slots[:t] % ex.PAGE
        check_heads(cache[at, 0, place], want, size, BF16)
        assert torch.equal(cache[at, 1, place].reshape(t, -1), v)
        # every earlier token of the two requests is still where the tables say
        for b in range(2):
            rows[b] = rows[b][:s["lens"][b]] + [(cache[at[i], 0, place[i]], cache[at[i], 1, place[i]])
                                                for i in range(t) if owners[i] == b]
            keys, values = attention_ref.gather_rows(cache, kv_indices, kv_indptr, last, b)
            assert keys.shape[0] == s["lens"][b] + s["new"][b] == len(rows[b])
            for i, (x, z) in enumerate(rows[b]):
                assert torch.equal(keys[i], x) and torch.equal(values[i], z)
        # attention, on the same tables
        want, _ = attention_ref.attention(s["query"].cpu().view(t, ex.HEADS, ex.HEAD_DIM), cache, append_indptr,
                                          kv_indptr, kv_indices, last, ex.HEAD_DIM ** -0.5)
        want = want.reshape(t, -1)
        # outputs are means of values: two 16-bit roundings (P and the output) of at most their size
        top = cache[:, 1].abs().max().double()
        assert ((s["attended"].double().cpu() - want).abs() <= half(BF16) * (want.abs() + 2 * top) + 1e-6).all()
        # projections out
        check_codes(s["out_codes"], s["out_scales"], s["attended"].double(), 0.0)
        y = int8_ref.linear(s["out_codes"], s["out_scales"], *layer.out)
        check_linear(s["middle"], y + s["hidden"].double(), y.abs() + s["hidden"].double().abs(), BF16)
        check_codes(s["post_codes"], s["post_scales"], int8_ref.normed(s["middle"], layer.post_norm, ex.EPS), NORM_ERROR)
        y = int8_ref.linear(s["post_codes"], s["post_scales"], *layer.gate_up)
        want, gate = int8_ref.silu_mul(y), y[:, :ex.INTER]
        error = silu_error(gate) + 3 * F32 * (gate.abs() + 1) + 4 * F32
        assert ((s["act"].double() - want).abs() <= (half(BF16) + error) * want.abs() + 2.0 ** -100).all()
        check_codes(s["act_codes"], s["act_scales"], s["act"].double(), 0.0)
        y = int8_ref.linear(s["act_codes"], s["act_scales"], *layer.down)
        check_linear(s["result"], y + s["middle"].double(), y.abs() + s["middle"].double().abs(), BF16)
    # pages: what the two requests hold and what is free are all there are
    held = [33, steps[-1]["lens"][1] + 1]
    assert tables.free_count.item() == 64 - sum(-(-n // ex.PAGE) for n in held)


def test_a_decode_step_in_a_graph():
    """Tables, norms, products, heads and cache captured once, with the lengths and rows of each replay;
    the bits are those of the same calls outside of a graph."""
    g = torch.Generator().manual_seed(5)
    dev, t = "cuda:0", 3
    layer = ex.Layer(32, dev, g)
    other = torch.zeros_like(layer.cache)

    def calls(tables, cache, seq, hidden):
        step = tables.begin_step(seq, torch.ones(t, dtype=torch.int32, device=dev))
        codes, scales = ex._codes(t, ex.HIDDEN, dev)
        ex.int8_ops.rms_norm_quantise(codes, scales, hidden, layer.input_norm, ex.EPS)
        qkv = torch.empty(t, (ex.HEADS + 2 * ex.KV_HEADS) * ex.HEAD_DIM, dtype=BF16, device=dev)
        ex.int8_ops.linear(qkv, codes, scales, *layer.qkv)
        q, k, v = split(qkv)
        ex.pos_encoding_ops.qk_norm_rotary_append(step.positions, q, k, v, layer.q_norm, layer.k_norm, ex.EPS,
                                                  ex.HEAD_DIM, layer.cos_sin, True, cache, step.slot_mapping)
        codes, scales = ex._codes(t, ex.HIDDEN, dev)
        ex.int8_ops.quantise_rows(codes, scales, q)
        ex.int8_ops.linear_residual(hidden, codes, scales, *layer.out)
        ex.int8_ops.rms_norm_quantise(codes, scales, hidden, layer.post_norm, ex.EPS)
        act = torch.empty(t, ex.INTER, dtype=BF16, device=dev)
        ex.int8_ops.gate_up_silu(act, codes, scales, *layer.gate_up)
        return act

    make = lambda: ex.BlockTables(t, 8, ex.PAGE, 32, t, dev)  # noqa: E731
    tables, eager = make(), make()
    seq = torch.zeros(t, dtype=torch.int32, device=dev)
    hidden = torch.zeros(t, ex.HIDDEN, dtype=BF16, device=dev)
    calls(make(), other, seq, hidden)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        act = calls(tables, layer.cache, seq, hidden)
    other.zero_()
    for i in range(40):
        x = torch.randn(t, ex.HIDDEN, generator=g).bfloat16().to(dev)
        seq.fill_(i)
        hidden.copy_(x)
        graph.replay()
        y = x.clone()
        want = calls(eager, other, seq, y)
        assert torch.equal(act, want) and torch.equal(hidden, y)
    tables.check()
    eager.check()
    assert torch.equal(layer.cache, other)
    assert torch.equal(tables.block_tables, eager.block_tables)
