"""Cases, plain forms and exact values of the 8-bit projections, the head norms with rotation, and
the step tables.

The operators serve one decoder layer of PaceServe with weights in 8 bits, and the step's index arrays:

* ``project``: rows are quantised to 8-bit integers with a scale each (as they are, out of the RMSNorm
  with the residual added first, or out of SiLU-and-mul) and multiplied with a weight in 8-bit integers
  with a scale for each output channel; the product is stored (with a bias or not), added to the
  residual stream, or taken through SiLU-and-mul;
* ``rotate``: each query and key head is normalised and rotated in one pass, in place, or with the keys
  and values going to their slots of the paged cache ``[pages, 2, page_size, kv_heads, head_dim]``;
* ``tables``: a step's page tables, index arrays and slots are built from the requests' lengths, new
  pages coming from a stack of free ones; then what the step took is given back (drafts that were not
  accepted), so that a pass leaves the tables as it found them.

``run`` computes each in elementary torch operations, or, where ``own`` is true, by this package's
kernels.
"""
import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
DEV = "cuda:0"
EPS = 1e-5
LEAST_SCALE = 2.0 ** -126


def _case(name, op, **kw):
    case = {"name": name, "op": op, "dtype": "bfloat16", "tokens": 1,
            # project
            "source": "rows", "end": "plain", "k": 4096, "n": 4096,
            # rotate
            "heads": 32, "kv_heads": 8, "head_dim": 128, "rot": 128, "neox": True, "append": False,
            "page": 16,
            # tables
            "requests": 0, "ctx": 0, "new": 1, "prompts": 0, "ragged": 1}
    assert set(kw) <= set(case)
    case.update(kw)
    return case


def listed():
    return [
        # one decode token's qkv projection: residual add, input norm, product
        _case("project_norm_qkv_1", "project", source="norm", n=6144),
        # a full decode batch's down projection into the residual stream
        _case("project_silu_down_64", "project", tokens=64, source="silu", end="residual", k=14336),
        # one chunked-prefill step of 512 tokens: the MLP's first half
        _case("project_norm_gate_up_512", "project", tokens=512, source="norm", end="gate_up",
              n=28672),
        # a prompt of odd length in fp16, its down projection
        _case("project_silu_down_1999_fp16", "project", dtype="float16", tokens=1999, source="silu",
              end="residual", k=14336),
        # a small head over odd widths, with a bias
        _case("project_odd_bias_77", "project", tokens=77, end="bias", k=1111, n=1003),
        # one long prompt through the MLP's first half: the largest product
        _case("project_gate_up_8192", "project", tokens=8192, end="gate_up", n=28672),
        # one decode token: norms, rotation, its key and value to the cache
        _case("rotate_append_1", "rotate", append=True),
        # a chunked-prefill step of 512 tokens
        _case("rotate_append_512", "rotate", tokens=512, append=True),
        # a prompt of odd length in fp16: adjacent pairs, 64-wide heads, half of each rotated
        _case("rotate_gptj_4999_fp16", "rotate", dtype="float16", tokens=4999, heads=24, kv_heads=8,
              head_dim=64, rot=32, neox=False),
        # long prompts of a model with 64 heads
        _case("rotate_append_16384", "rotate", tokens=16384, heads=64, append=True),
        # 64 requests, a token each
        _case("tables_decode_64", "tables", requests=64, ctx=8191),
        # a large batch with prompt chunks beside the single tokens
        _case("tables_mixed_1000", "tables", requests=1000, ctx=16000, new=448, prompts=30),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["project", "project", "project", "rotate", "rotate", "tables"])
    kw = {"dtype": rng.choice(["bfloat16", "float16"]), "ragged": rng.randrange(1, 1 << 20)}
    if op == "project":
        kw.update(tokens=_log(rng, 1, 8192), source=rng.choice(["rows", "norm", "silu"]),
                  end=rng.choice(["plain", "bias", "residual", "gate_up"]))
        if rng.random() < 0.2:  # odd widths
            kw.update(tokens=_log(rng, 1, 256), k=_log(rng, 100, 2000), n=_log(rng, 100, 2000))
        else:
            kw.update(k=rng.choice([2048, 4096, 8192, 14336]),
                      n=rng.choice([2048, 4096, 6144, 8192, 28672]))
            while kw["tokens"] * kw["k"] * kw["n"] > 8192 * 4096 * 28672:
                kw["tokens"] //= 2
        kw["n"] += kw["n"] % 2
    elif op == "rotate":
        kw.update(tokens=_log(rng, 1, 16384), neox=rng.random() < 0.7, append=rng.random() < 0.6,
                  head_dim=rng.choice([64, 96, 128]), kv_heads=rng.choice([2, 4, 8]),
                  page=rng.choice([8, 16, 32]))
        kw["heads"] = kw["kv_heads"] * rng.choice([1, 3, 4, 8])
        kw["rot"] = rng.choice([kw["head_dim"], kw["head_dim"], kw["head_dim"] // 2])
    else:
        kw.update(requests=_log(rng, 1, 1000), ctx=_log(rng, 1, 16000), page=rng.choice([8, 16, 32]),
                  new=_log(rng, 1, 448), prompts=rng.randrange(0, 31))
        kw["prompts"] = min(kw["prompts"], kw["requests"])
    return {k: v for k, v in _case("", op, **kw).items() if k != "name"}


def _lengths(case):
    """(tokens in the cache, new tokens) of each request: prompt chunks first, then single tokens."""
    r, got = random.Random(case["ragged"]), []
    for i in range(case["requests"]):
        new = 1
        if i < case["prompts"]:
            new = case["new"] if i == 0 else r.randrange(case["new"]) + 1
        got.append((case["ctx"] if i == 0 else r.randrange(case["ctx"] + 1), new))
    return got


def _outputs(case):
    """Columns that a projection stores."""
    return case["n"] // 2 if case["end"] == "gate_up" else case["n"]


def work(case):
    size, t = (4 if case["dtype"] == "float32" else 2), case["tokens"]
    if case["op"] == "project":
        k, n = case["k"], case["n"]
        rows = {"rows": k, "norm": 3 * k, "silu": 2 * k}[case["source"]]  # norm: x and residual in, residual out
        outs = _outputs(case) * (2 if case["end"] == "residual" else 1)
        return {"bytes": size * t * (rows + outs) + n * k + 4 * n, "flops": 2 * t * n * k}
    if case["op"] == "rotate":
        heads, d = case["heads"] + case["kv_heads"] * (2 if case["append"] else 1), case["head_dim"]
        return {"bytes": t * (2 * size * heads * d + 8 + 4 * case["rot"]), "flops": 8 * t * heads * d}
    lens, page = _lengths(case), case["page"]
    pages = sum(-(-(n + q) // page) for n, q in lens)
    old = sum(-(-n // page) for n, _ in lens)
    new = sum(q for _, q in lens)
    # lengths, old pages, new pages from the stack and back; indices, the table's new entries, slots
    return {"bytes": 4 * (8 * len(lens) + old + pages + 4 * (pages - old)) + 20 * new,
            "flops": 4 * (pages + new)}


# ------------------------------------------------------------------ inputs --
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype, t = DTYPES[case["dtype"]], case["tokens"]
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    st = {"case": case}
    if case["op"] == "project":
        k, n = case["k"], case["n"]
        # activations with a few channels that stand out, as layers have
        spread = torch.exp(rnd(2 * k if case["source"] == "silu" else k) / 2)
        st["x"] = (rnd(t, spread.numel()) * spread).to(dtype)
        if case["source"] == "norm":
            st["stream"] = rnd(t, k).to(dtype)
            st["norm_weight"] = (1 + rnd(k) / 8).to(dtype)
        # a weight quantised at load: codes of every size, a scale for each channel
        st["weight"] = (rnd(n, k) * 40).round_().clamp_(-127, 127).to(torch.int8)
        st["weight_scales"] = torch.exp(rnd(n) / 4) / (40 * math.sqrt(k))
        if case["end"] == "bias":
            st["bias"] = rnd(n).to(dtype)
        if case["end"] == "residual":
            st["residual"] = rnd(t, n).to(dtype)
        return st
    page = case["page"]
    if case["op"] == "rotate":
        h, hk, d, rot = case["heads"], case["kv_heads"], case["head_dim"], case["rot"]
        st["qkv"] = (rnd(t, (h + 2 * hk) * d) * 2).to(dtype)  # views of the projection's rows
        st["q_weight"], st["k_weight"] = (1 + rnd(d) / 8).to(dtype), (1 + rnd(d) / 8).to(dtype)
        ends = torch.randint(t, 32768, (1,), generator=g, device=DEV)
        st["positions"] = ends - t + torch.arange(t, device=DEV)
        angle = torch.arange(32768, device=DEV, dtype=torch.float64)[:, None] \
            * 500000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
        st["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        if case["append"]:
            pages = -(-t // page) + 3
            st["cache"] = torch.zeros(pages, 2, page, hk, d, device=DEV, dtype=dtype)
            order = torch.randperm(pages, generator=g, device=DEV)
            i = torch.arange(t, device=DEV)
            st["slots"] = order[i // page] * page + i % page
        return st
    lens = _lengths(case)
    held = [-(-n // page) for n, _ in lens]
    need = [-(-(n + q) // page) for n, q in lens]
    longest, total, tokens = max(need), sum(need), sum(q for _, q in lens)
    pool = torch.randperm(total + 64, generator=g, device=DEV).int()
    table = torch.full((len(lens), longest), -1, dtype=torch.int32, device=DEV)
    width = torch.tensor(held, device=DEV)
    table[torch.arange(longest, device=DEV)[None] < width[:, None]] = pool[:sum(held)]
    st.update(block_tables=table, free_pages=pool[sum(held):].clone(),
              free_count=torch.tensor([total + 64 - sum(held)], dtype=torch.int32, device=DEV),
              seq_lens=torch.tensor([n for n, _ in lens], dtype=torch.int32, device=DEV),
              new_lens=torch.tensor([q for _, q in lens], dtype=torch.int32, device=DEV))
    ints = lambda n, kind=torch.int32: torch.full((n,), -7, dtype=kind, device=DEV)  # noqa: E731
    # the step's arrays, kept from step to step; room for some tokens more
    st.update(append_indptr=ints(len(lens) + 1), kv_indptr=ints(len(lens) + 1), kv_indices=ints(total),
              kv_last_page_len=ints(len(lens)), batch_indices=ints(tokens + 5),
              positions=ints(tokens + 5, torch.int64), slot_mapping=ints(tokens + 5, torch.int64),
              status=torch.zeros(1, dtype=torch.int32, device=DEV),
              arrivals=torch.zeros(1, dtype=torch.int32, device=DEV),
              step_lens=torch.tensor([n + q for n, q in lens], dtype=torch.int32, device=DEV))
    return st


# ------------------------------------------------------------- plain forms --
def _quantised(y):
    """Whole numbers of -127 .. 127 (as floats) and a scale for each row of 32-bit `y`."""
    top = y.abs().amax(-1, keepdim=True)
    scale = (top / 127).clamp_min(LEAST_SCALE)
    return (y / scale).round(), scale


def _project_plain(st):
    case, x = st["case"], st["x"].float()
    stream = None
    if case["source"] == "norm":
        stream = st["stream"].copy_(x + st["stream"].float())
        x = stream.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * st["norm_weight"].float()
    elif case["source"] == "silu":
        gate, up = x.chunk(2, -1)
        x = gate * torch.sigmoid(gate) * up
    codes, scale = _quantised(x)
    # sums of products of whole numbers pass 24 bits: in 64
    y = (codes.double() @ st["weight"].double().T).float() * scale * st["weight_scales"]
    if case["end"] == "bias":
        y = y + st["bias"].float()
    elif case["end"] == "residual":
        st["residual"].copy_(st["residual"].float() + y)
        y = st["residual"]
    elif case["end"] == "gate_up":
        gate, up = y.chunk(2, -1)
        y = gate * torch.sigmoid(gate) * up
    got = {"out": y.to(st["x"].dtype)}
    if stream is not None:
        got["stream"] = stream
    return got


def _head_views(st):
    case = st["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    return [x.view(case["tokens"], -1, d) for x in st["qkv"].split([h * d, hk * d, hk * d], 1)]


def _rotated(st, x, weight):
    case, rot = st["case"], st["case"]["rot"]
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    cos, sin = st["cos_sin"][st["positions"]][:, None].chunk(2, -1)
    turn, rest = x[..., :rot], x[..., rot:]
    if case["neox"]:
        a, b = turn.chunk(2, -1)
        turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turn[..., ::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turn, rest], -1)


def _rotate_plain(st):
    q, k, v = _head_views(st)
    if not st["case"]["append"]:
        q.copy_(_rotated(st, q, st["q_weight"]))
        k.copy_(_rotated(st, k, st["k_weight"]))
        return {"qkv": st["qkv"]}
    q.copy_(_rotated(st, q, st["q_weight"]))
    at, slot = st["slots"] // st["case"]["page"], st["slots"] % st["case"]["page"]
    st["cache"][at, 0, slot] = _rotated(st, k, st["k_weight"]).to(st["cache"].dtype)
    st["cache"][at, 1, slot] = v
    return {"qkv": st["qkv"], "cache": st["cache"]}


TABLES = ("block_tables", "append_indptr", "kv_indptr", "kv_indices", "kv_last_page_len",
          "batch_indices", "positions", "slot_mapping", "status")


def _tables_plain(st):
    page, table = st["case"]["page"], st["block_tables"]
    n, q = st["seq_lens"].long(), st["new_lens"].long()
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    held, need = (n + page - 1) // page, (n + q + page - 1) // page
    # new pages, from the stack's top in the requests' order
    col = torch.arange(table.shape[1], device=DEV)[None]
    fresh = (col >= held[:, None]) & (col < need[:, None])
    rank = fresh.flatten().cumsum(0).view_as(fresh) - 1
    top = st["free_count"].long()
    pick = torch.where(fresh, top - 1 - rank, 0)
    table.copy_(torch.where(fresh, st["free_pages"][pick], table))
    st["free_count"] -= fresh.sum().int()
    # index arrays
    st["kv_indptr"].copy_(torch.cat([zero, need.cumsum(0)]))
    st["append_indptr"].copy_(torch.cat([zero, q.cumsum(0)]))
    st["kv_last_page_len"].copy_((n + q - 1) % page + 1)
    st["kv_indices"].copy_(table[col < need[:, None]])
    # one entry for each new token; -1 behind the last
    i = torch.arange(st["positions"].numel(), device=DEV)
    ip = st["append_indptr"].long()
    b = torch.searchsorted(ip, i, right=True) - 1
    real = i < ip[-1]
    b = torch.where(real, b, zero)
    pos = torch.where(real, n[b] + i - ip[b], zero)
    st["slot_mapping"].copy_(torch.where(real, table[b, pos // page] * page + pos % page, -1))
    st["batch_indices"].copy_(torch.where(real, b, -1))
    st["positions"].copy_(torch.where(real, pos, -1))
    got = {k: st[k] for k in TABLES}
    # the new pages back onto the stack, as they lay
    k = torch.where(fresh, pick, st["free_pages"].numel())
    stack = torch.cat([st["free_pages"], zero.int()])
    stack[k.flatten()] = table.flatten()
    st["free_pages"].copy_(stack[:-1])
    st["free_count"] += fresh.sum().int()
    got["free_pages"], got["free_count"] = st["free_pages"], st["free_count"]
    return got


def run(state):
    st, case = state, state["case"]
    if not own:
        return {"project": _project_plain, "rotate": _rotate_plain, "tables": _tables_plain}[
            case["op"]](st)
    if case["op"] == "project":
        from paceserve_b200 import int8_ops

        t, k, x = case["tokens"], case["k"], st["x"]
        codes = torch.empty(t, k, dtype=torch.int8, device=DEV)
        scales = torch.empty(t, dtype=torch.float32, device=DEV)
        got = {}
        if case["source"] == "norm":
            got["stream"] = st["stream"]
            int8_ops.rms_norm_quantise(codes, scales, x, st["norm_weight"], EPS, st["stream"])
        elif case["source"] == "silu":
            int8_ops.silu_and_mul_quantise(codes, scales, x)
        else:
            int8_ops.quantise_rows(codes, scales, x)
        if case["end"] == "residual":
            got["out"] = st["residual"]
            int8_ops.linear_residual(st["residual"], codes, scales, st["weight"], st["weight_scales"])
            return got
        got["out"] = torch.empty(t, _outputs(case), dtype=x.dtype, device=DEV)
        if case["end"] == "gate_up":
            int8_ops.gate_up_silu(got["out"], codes, scales, st["weight"], st["weight_scales"])
        else:
            int8_ops.linear(got["out"], codes, scales, st["weight"], st["weight_scales"],
                            st.get("bias"))
        return got
    if case["op"] == "rotate":
        from paceserve_b200 import pos_encoding_ops as pe

        h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
        q, k, v = st["qkv"].split([h * d, hk * d, hk * d], 1)
        if case["append"]:
            pe.qk_norm_rotary_append(st["positions"], q, k, v, st["q_weight"], st["k_weight"], EPS, d,
                                     st["cos_sin"], case["neox"], st["cache"], st["slots"])
            return {"qkv": st["qkv"], "cache": st["cache"]}
        pe.qk_norm_rotary_embedding(st["positions"], q, k, st["q_weight"], st["k_weight"], EPS, d,
                                    st["cos_sin"], case["neox"])
        return {"qkv": st["qkv"]}
    from paceserve_b200 import kv_transfer_ops as kv

    kv.build_step_tables(st["block_tables"], st["seq_lens"], st["new_lens"], case["page"],
                         st["free_pages"], st["free_count"], st["append_indptr"], st["kv_indptr"],
                         st["kv_indices"], st["kv_last_page_len"], st["batch_indices"],
                         st["positions"], st["slot_mapping"], st["status"], st["arrivals"])
    got = {k: st[k] for k in TABLES}
    kv.release_pages(st["block_tables"], st["step_lens"], st["seq_lens"], case["page"],
                     st["free_pages"], st["free_count"], st["status"], st["arrivals"])
    got["free_pages"], got["free_count"] = st["free_pages"], st["free_count"]
    return got


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "tables":
        return None  # whole numbers: nothing is rounded
    if case["op"] == "project":
        x, k = st["x"].double(), case["k"]
        got = {"out": None}
        if case["source"] == "norm":
            got["stream"] = x + st["stream"].double()
            # what is normalised is the stream as it is held
            x = got["stream"].to(st["x"].dtype).double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / k + EPS).sqrt() * st["norm_weight"].double()
        elif case["source"] == "silu":
            x = x[:, :k] / (1 + torch.exp(-x[:, :k])) * x[:, k:]
        scale = torch.maximum(x.abs().max(-1).values / 127, torch.tensor(LEAST_SCALE, device=DEV))
        codes = torch.round(x / scale[:, None]).float()
        out = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device=DEV)
        for c in range(0, k, 1024):  # 1024 products of 7 bits by 7 fit 24: exact in 32 bits
            out += codes[:, c:c + 1024] @ st["weight"][:, c:c + 1024].float().T
        out *= scale[:, None]
        out *= st["weight_scales"].double()
        if case["end"] == "bias":
            out += st["bias"].double()
        elif case["end"] == "residual":
            out += st["residual"].double()
        elif case["end"] == "gate_up":
            half = case["n"] // 2
            out = out[:, half:] * out[:, :half] / (1 + torch.exp(-out[:, :half]))
        got["out"] = out
        return got
    t, rot, d = case["tokens"], case["rot"], case["head_dim"]
    heads = st["qkv"].double().view(t, -1, d)
    nq, nk = case["heads"], case["kv_heads"]
    weight = torch.ones(nq + 2 * nk, d, dtype=torch.float64, device=DEV)
    weight[:nq], weight[nq:nq + nk] = st["q_weight"].double(), st["k_weight"].double()
    y = heads / (heads.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * weight
    at = torch.arange(rot // 2, device=DEV)
    first = at if case["neox"] else 2 * at
    second = at + rot // 2 if case["neox"] else 2 * at + 1
    table = st["cos_sin"].double()[st["positions"]][:, None]
    z = torch.complex(y[..., first], y[..., second]) * torch.complex(table[..., :rot // 2],
                                                                     table[..., rot // 2:])
    y[..., first], y[..., second] = z.real, z.imag
    y[:, nq + nk:] = heads[:, nq + nk:]  # values stay
    if not case["append"]:
        return {"qkv": y.view(t, -1)}
    cache = torch.zeros(st["cache"].shape, dtype=torch.float64, device=DEV)
    flat = cache.permute(1, 0, 2, 3, 4).reshape(2, -1, nk, d)  # a copy: [2, slots, heads, dims]
    flat[0, st["slots"]], flat[1, st["slots"]] = y[:, nq:nq + nk], y[:, nq + nk:]
    cache = flat.view(2, -1, case["page"], nk, d).permute(1, 0, 2, 3, 4)
    y[:, nq:] = heads[:, nq:]  # with the cache, the keys' rows stay as they were
    return {"qkv": y.view(t, -1), "cache": cache}
