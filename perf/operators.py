"""Cases, plain forms and exact values of the paged-attention operators.

The operators serve one decoder layer's attention over PaceServe's paged KV
cache ``[pages, 2, page_size, kv_heads, head_dim]``:

* ``append``: new K/V rows are quantised to e4m3 codes with one power-of-two
  exponent per (token, K or V, kv head) while they are written to their pages;
* ``read``: a request's quantised rows are read back in sequence order;
* ``attend``: attention of prompts, prompt chunks and single tokens over the
  cache (16-bit or quantised), with capped scores, distance bias, sliding
  window, prefix and document masks;
* ``tree``: attention of a tree of drafted tokens, the last of each sequence.

``run`` computes each in elementary torch operations in 32 bits, or, where
``own`` is true, by this package's kernels.
"""
import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
DEV = "cuda:0"
CODE_MAX = 448.0  # the largest e4m3 value


def _case(name, op, **kw):
    case = {"name": name, "op": op, "dtype": "bfloat16", "heads": 32, "kv_heads": 8,
            "head_dim": 128, "page": 16, "quantised": False, "prefills": 0, "prefill_len": 0,
            "done": 0, "decodes": 0, "ctx": 0, "nodes": 1, "ragged": 1, "soft_cap": 0.0,
            "alibi": False, "window": -1, "prefix": 0, "docs": 0}
    assert set(kw) <= set(case)
    case.update(kw)
    return case


def listed():
    return [
        # one decode token of one request: only launch latency counts
        _case("append_one_token", "append", quantised=True, decodes=1, ctx=700),
        # a chunked-prefill step with a budget of 512 tokens: a 448-token chunk and 64 decodes
        _case("append_mixed_512", "append", quantised=True, prefills=1, prefill_len=448,
              decodes=64, ctx=8191),
        # long prompts in fp16, 16384 tokens and a few, of odd lengths
        _case("append_prompts_fp16", "append", quantised=True, dtype="float16", prefills=5,
              prefill_len=3999),
        # one short request read back, e.g. its prefix going to a 16-bit cache
        _case("read_one_short", "read", quantised=True, decodes=1, ctx=137),
        # eight promoted requests of up to 8192 tokens
        _case("read_promoted", "read", quantised=True, decodes=8, ctx=8192, ragged=5),
        # one user chatting: one token, a short context
        _case("decode_one_short", "attend", decodes=1, ctx=333),
        # a full decode batch with long contexts and distance bias over a quantised cache
        _case("decode_64_quantised", "attend", quantised=True, decodes=64, ctx=8191, alibi=True),
        # the 512-token chunked-prefill step: a chunk and 64 decodes, capped scores
        _case("mixed_512_capped", "attend", prefills=1, prefill_len=448, decodes=64, ctx=4096,
              soft_cap=30.0),
        # prompts of odd lengths in fp16 with 64-wide heads, each packed from documents, under a
        # sliding window
        _case("prefill_docs_window_fp16", "attend", dtype="float16", heads=24, kv_heads=8,
              head_dim=64, prefills=4, prefill_len=1777, window=1023, docs=4, ragged=3),
        # one long prompt with a bidirectional prefix, capped scores: the largest prefill
        _case("prefill_8192_prefix_capped", "attend", prefills=1, prefill_len=8192, prefix=500,
              soft_cap=50.0),
        # one request's small draft tree
        _case("tree_one", "tree", decodes=1, ctx=331, nodes=13),
        # a batch of larger trees over long contexts in a quantised cache
        _case("tree_32_quantised", "tree", quantised=True, decodes=32, ctx=4500, nodes=48),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["append", "read", "attend", "attend", "attend", "tree", "tree"])
    kw = {"dtype": rng.choice(["bfloat16", "float16"]), "head_dim": rng.choice([64, 128]),
          "page": rng.choice([8, 16, 16, 32]), "ragged": rng.randrange(1, 1 << 20)}
    kw["kv_heads"] = rng.choice([2, 4, 8])
    kw["heads"] = kw["kv_heads"] * rng.choice([1, 3, 4, 4, 8])
    if kw["heads"] > 32:
        kw["heads"] = 32
    if op == "append":
        kw.update(quantised=True, prefills=rng.choice([0, 1, 3]), prefill_len=_log(rng, 1, 5000),
                  decodes=rng.randrange(1, 65), ctx=_log(rng, 1, 8191))
        kw["dtype"] = rng.choice(["bfloat16", "float16", "float32"])
    elif op == "read":
        kw.update(quantised=True, decodes=_log(rng, 1, 8), ctx=_log(rng, 1, 8192))
    elif op == "tree":
        kw.update(quantised=rng.random() < 0.5, decodes=_log(rng, 1, 32), ctx=_log(rng, 1, 4500),
                  nodes=_log(rng, 1, 64), soft_cap=rng.choice([0.0, 0.0, 50.0]))
    else:
        kw.update(quantised=rng.random() < 0.4, soft_cap=rng.choice([0.0, 0.0, 30.0]),
                  alibi=rng.random() < 0.3)
        if rng.random() < 0.5:
            kw.update(decodes=_log(rng, 1, 64), ctx=_log(rng, 1, 8191))
            kw["window"] = rng.choice([-1, -1, 1023])
        else:
            kw.update(prefills=rng.randrange(1, 5), prefill_len=_log(rng, 1, 4000))
            kw["done"] = rng.choice([0, 0, _log(rng, 1, 500)])
            kw["window"] = rng.choice([-1, -1, 511])
            kw["prefix"] = rng.choice([0, 0, 100])
            kw["docs"] = rng.choice([0, 0, 5])
    return {k: v for k, v in _case("", op, **kw).items() if k != "name"}


def _lengths(case):
    """(new tokens, sequence length) of each request: prompts first, then the others."""
    r = random.Random(case["ragged"])
    got = []
    for i in range(case["prefills"]):
        n = case["prefill_len"] if i == 0 else r.randrange(case["prefill_len"] // 2,
                                                           case["prefill_len"]) + 1
        got.append((n, n + case["done"]))
    for i in range(case["decodes"]):
        n = case["ctx"] if i == 0 else r.randrange(case["ctx"]) + 1
        q = case["nodes"] if i == 0 else r.randrange((case["nodes"] + 1) // 2, case["nodes"] + 1)
        got.append((q, n + q if case["op"] == "tree" else max(n, q)))
    return got


def _doc_starts(case):
    """The first position of each new token's own document; None without documents."""
    if not case["docs"]:
        return None
    r, got = random.Random(case["ragged"] + 1), []
    for q, n in _lengths(case):
        cuts = sorted({0} | {r.randrange(n) for _ in range(case["docs"] - 1)})
        k = 0
        for p in range(n - q, n):
            while k + 1 < len(cuts) and cuts[k + 1] <= p:
                k += 1
            got.append(cuts[k])
    return got


def work(case):
    h, d, hk = case["heads"], case["head_dim"], case["kv_heads"]
    size = 4 if case["dtype"] == "float32" else 2
    lens = _lengths(case)
    tokens, total = sum(q for q, _ in lens), sum(n for _, n in lens)
    row = hk * (d + 1) if case["quantised"] else hk * d * size  # one token's K (or V) in the cache
    if case["op"] == "append":
        return {"bytes": 2 * tokens * (hk * d * size + row), "flops": 4 * tokens * hk * d}
    if case["op"] == "read":
        return {"bytes": 2 * total * (hk * d * size + row), "flops": 2 * total * hk * d}
    starts = _doc_starts(case)
    pairs = seen = at = 0
    for q, n in lens:
        first = n
        for i in range(q):
            p = n - q + i
            lo = max(0, p - case["window"]) if case["window"] >= 0 else 0
            if starts:
                lo = max(lo, starts[at + i])
            hi = min(n, max(p + 1, case["prefix"]))
            pairs += max(0, hi - lo)
            first = min(first, lo)
        seen += n - first
        at += q
    return {"bytes": 2 * tokens * h * d * size + 2 * seen * row, "flops": 4 * d * h * pairs}


# ------------------------------------------------------------------ inputs --
def _plain_codes(x):
    """e4m3 codes (as float8) and biased exponents of rows of `x` (last axis): the exponent is the
    smallest e with max|x| <= 448 * 2^e."""
    x = x.float()
    m, k = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > 0.875, k - 8, k - 9).clamp(-126, 127)
    e = torch.where(m == 0, torch.zeros_like(e), e)
    y = torch.ldexp(x, -e[..., None]).clamp(-CODE_MAX, CODE_MAX)
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _tree(r, nodes):
    """Ancestor masks (each node's own bit among them) of a random tree in topological order."""
    masks = []
    for i in range(nodes):
        parent = r.randrange(-1, i) if i else -1
        masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
    return masks


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = _lengths(case)
    dtype, page = DTYPES[case["dtype"]], case["page"]
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    npages = [-(-n // page) for _, n in lens]
    total = sum(npages) + 3
    host = {
        "qo_indptr": torch.tensor([0] + [q for q, _ in lens]).cumsum(0).int(),
        "kv_indptr": torch.tensor([0] + npages).cumsum(0).int(),
        "kv_last_page_len": torch.tensor([(n - 1) % page + 1 for _, n in lens]).int(),
        "kv_indices": torch.randperm(total, generator=g, device=DEV)[:total - 3].int().cpu(),
    }
    st = {"case": case, "lens": lens, "host": host, **{k: v.to(DEV) for k, v in host.items()}}
    tokens = sum(q for q, _ in lens)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=dtype)  # noqa: E731
    shape = (total, 2, page, hk, d)
    if case["op"] == "append":
        # K and V are views of the projection's rows, as in a decoder layer; channels of
        # different size, as keys have
        qkv = rnd(tokens, (h + 2 * hk) * d) * torch.exp(rnd((h + 2 * hk) * d))
        st["key"], st["value"] = qkv[:, h * d:(h + hk) * d], qkv[:, (h + hk) * d:]
        st["codes"] = torch.zeros(shape, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
        st["exponents"] = torch.zeros(shape[:-1], device=DEV, dtype=torch.uint8)
        return st
    if case["quantised"]:
        st["codes"], st["exponents"] = _plain_codes(
            torch.randn(shape, generator=g, device=DEV) * torch.exp(rnd(1, 2, 1, hk, d).float() / 2))
    else:
        st["cache"] = rnd(shape)
    if case["op"] == "read":
        st["rows"] = torch.tensor([0] + [n for _, n in lens]).cumsum(0).int().to(DEV)
        return st
    # queries of the projection's rows too; sharp enough that some keys stand out
    st["query"] = (rnd(tokens, (h + 2 * hk) * d) * 1.5)[:, :h * d].view(tokens, h, d)
    st["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device=DEV) \
        if case["alibi"] else None
    starts = _doc_starts(case)
    host["doc_starts"] = None if starts is None else torch.tensor(starts).int()
    st["doc_starts"] = None if starts is None else host["doc_starts"].to(DEV)
    host["prefix_lens"] = torch.tensor([min(case["prefix"], n) for _, n in lens]).int() \
        if case["prefix"] else None
    if case["op"] == "tree":
        r = random.Random(seed)
        words = [w - (1 << 64) if w >> 63 else w for q, _ in lens for w in _tree(r, q)]
        st["tree_mask"] = torch.tensor(words, dtype=torch.int64, device=DEV)[:, None]
    if own:
        # the step's plan, made once for all layers
        from paceserve_b200.attention import PagedAttention

        st["attention"] = PagedAttention(h, hk, d, page, device=DEV)
        args = [host[k] for k in ("qo_indptr", "kv_indptr", "kv_indices", "kv_last_page_len")]
        if case["op"] == "tree":
            st["attention"].begin_tree_forward(*args, st["tree_mask"])
        else:
            st["attention"].begin_forward(*args, window_left=case["window"],
                                          prefix_lens=host["prefix_lens"],
                                          doc_starts=host["doc_starts"])
    return st


# ------------------------------------------------------------- plain forms --
def _seq_lens(st):
    n = st["kv_indptr"].diff()
    return (n - 1) * st["case"]["page"] + st["kv_last_page_len"]


def _append_plain(st):
    page = st["case"]["page"]
    hk, d = st["case"]["kv_heads"], st["case"]["head_dim"]
    ip = st["qo_indptr"].long()
    token = torch.arange(st["key"].shape[0], device=DEV)
    b = torch.searchsorted(ip, token, right=True) - 1
    pos = _seq_lens(st)[b] - ip[b + 1] + token
    where = st["kv_indices"][st["kv_indptr"][b] + pos // page].long()
    both = torch.stack([st["key"], st["value"]], 1).view(-1, 2, hk, d)
    codes, exps = _plain_codes(both)
    kinds = torch.arange(2, device=DEV)[None]
    slot = (where[:, None], kinds, (pos % page)[:, None])
    st["codes"].view(torch.uint8)[slot] = codes.view(torch.uint8)
    st["exponents"][slot] = exps
    return {"codes": st["codes"], "exponents": st["exponents"]}


def _rows(st, kind, page_ids, slots):
    """K (0) or V (1) rows at these places of the cache, in 32 bits."""
    if not st["case"]["quantised"]:
        return st["cache"][page_ids, kind, slots].float()
    x = st["codes"].view(torch.uint8)[page_ids, kind, slots].view(torch.float8_e4m3fn).float()
    return torch.ldexp(x, st["exponents"][page_ids, kind, slots].int()[..., None] - 127)


def _read_plain(st):
    page, ip = st["case"]["page"], st["rows"].long()
    row = torch.arange(sum(n for _, n in st["lens"]), device=DEV)
    b = torch.searchsorted(ip, row, right=True) - 1
    pos = row - ip[b]
    where = st["kv_indices"][st["kv_indptr"][b] + pos // page].long()
    dtype = DTYPES[st["case"]["dtype"]]
    return {"key": _rows(st, 0, where, pos % page).to(dtype),
            "value": _rows(st, 1, where, pos % page).to(dtype)}


def _attend_plain(st, first, last):
    """Attention of requests first .. last, padded to their longest."""
    case, lens = st["case"], st["lens"][first:last]
    h, hk, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    qm, km = max(q for q, _ in lens), max(n for _, n in lens)
    n = _seq_lens(st)[first:last].long()[:, None]
    q0, q1 = st["qo_indptr"][first:last].long(), st["qo_indptr"][first + 1:last + 1].long()
    i = torch.arange(qm, device=DEV)[None]
    j = torch.arange(km, device=DEV)
    real = i < (q1 - q0)[:, None]
    token = torch.where(real, q0[:, None] + i, q0[:, None])
    base = n - (q1 - q0)[:, None]
    place = st["kv_indptr"][first:last, None].long() + torch.minimum(j[None], n - 1) // page
    where = st["kv_indices"][place].long()
    slots = torch.minimum(j[None], n - 1) % page
    k = _rows(st, 0, where, slots).permute(0, 2, 3, 1)  # [b, hk, d, km]
    v = _rows(st, 1, where, slots).permute(0, 2, 1, 3)  # [b, hk, km, d]
    g, b = h // hk, last - first
    q = st["query"][token].float().view(b, qm, hk, g, d).permute(0, 2, 3, 1, 4)
    s = (q.reshape(b, hk, g * qm, d) @ k).view(b, hk, g, qm, km)
    s *= 1.0 / math.sqrt(d)
    if case["soft_cap"]:
        s.div_(case["soft_cap"]).tanh_().mul_(case["soft_cap"])
    pos = base + i
    if case["alibi"]:
        s -= st["slopes"].view(1, hk, g, 1, 1) * (pos[..., None] - j).abs()[:, None, None]
    if case["op"] == "tree":
        node = j - base[..., None]  # [b, 1, km], the drafted tokens from 0
        bits = st["tree_mask"][token, 0][..., None] >> node.clamp(0, 63)
        seen = (j < n[..., None]) & ((node < 0) | (bits & 1).bool())
    else:
        hi = pos + 1
        if case["prefix"]:
            hi = torch.maximum(hi, torch.full_like(hi, case["prefix"]))
        lo = torch.zeros_like(pos)
        if case["window"] >= 0:
            lo = pos - case["window"]
        if st["doc_starts"] is not None:
            lo = torch.maximum(lo, st["doc_starts"][token].long())
        seen = (j >= lo[..., None]) & (j < torch.minimum(hi, n)[..., None])
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(top.isinf(), torch.zeros_like(top), top)).exp_()
    total = s.sum(-1)
    o = (s.view(b, hk, g * qm, km) @ v).view(b, hk, g, qm, d)
    o = torch.where(total[..., None] > 0, o / total[..., None], torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(b, qm, h, d)[real].to(st["query"].dtype)


def run(state):
    st, case = state, state["case"]
    if own:
        from paceserve_b200 import kv_transfer_ops as kv

        if case["op"] == "append":
            kv.append_quantised_paged_kv_cache(
                st["key"], st["value"], st["qo_indptr"], st["codes"], st["exponents"],
                st["kv_indices"], st["kv_indptr"], st["kv_last_page_len"])
            return {"codes": st["codes"], "exponents": st["exponents"]}
        if case["op"] == "read":
            rows = sum(n for _, n in st["lens"])
            shape = (rows, case["kv_heads"], case["head_dim"])
            key = torch.empty(shape, dtype=DTYPES[case["dtype"]], device=DEV)
            value = torch.empty_like(key)
            kv.read_quantised_paged_kv_cache(
                key, value, st["rows"], st["codes"], st["exponents"], st["kv_indices"],
                st["kv_indptr"], st["kv_last_page_len"])
            return {"key": key, "value": value}
        out = st["attention"].forward(
            st["query"], st["codes"] if case["quantised"] else st["cache"],
            exponents=st["exponents"] if case["quantised"] else None,
            logits_soft_cap=case["soft_cap"], alibi_slopes=st["slopes"])
        return {"out": out}
    if case["op"] == "append":
        return _append_plain(st)
    if case["op"] == "read":
        return _read_plain(st)
    p, n = case["prefills"], len(st["lens"])
    if not p or p == n:
        return {"out": _attend_plain(st, 0, n)}
    return {"out": torch.cat([_attend_plain(st, 0, p), _attend_plain(st, p, n)])}


# ------------------------------------------------------------------- exact --
def _e4m3_64(y):
    """`y` (64 bits, |y| <= 448) rounded to the nearest multiple of its binade's step, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30))).clamp(min=-6.0) - 3.0)
    return torch.round(y / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    lens, page = st["lens"], case["page"]
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    table = st["host"]["kv_indices"].tolist()
    first = st["host"]["kv_indptr"].tolist()

    def places(r, lo, hi):
        pos = torch.arange(lo, hi, device=DEV)
        ids = torch.tensor(table[first[r]:first[r + 1]], device=DEV)
        return ids[pos // page], pos % page

    if case["op"] == "append":
        codes = torch.zeros(st["codes"].shape, dtype=torch.float64, device=DEV)
        exps = torch.zeros(st["exponents"].shape, dtype=torch.int64, device=DEV)
        at = 0
        for r, (q, n) in enumerate(lens):
            ids, slots = places(r, n - q, n)
            for kind, x in enumerate((st["key"], st["value"])):
                x = x[at:at + q].double().view(q, hk, d)
                top = x.abs().amax(-1)
                e = torch.ceil(torch.log2(top / CODE_MAX))
                e += (top > CODE_MAX * torch.exp2(e)).double()  # where log2 was rounded
                e -= (top <= CODE_MAX * torch.exp2(e - 1)).double()
                codes[ids, kind, slots] = _e4m3_64(x / torch.exp2(e)[..., None])
                exps[ids, kind, slots] = e.long() + 127
            at += q
        return {"codes": codes, "exponents": exps}

    def rows(r, kind, lo, hi):
        ids, slots = places(r, lo, hi)
        if not case["quantised"]:
            return st["cache"][ids, kind, slots].double()
        c = st["codes"].view(torch.uint8)[ids, kind, slots].long()
        e, m = c // 8 % 16, (c % 8).double()
        x = torch.where(e > 0, (8 + m) * torch.exp2(e.double() - 10), m * 2.0 ** -9)
        x = torch.where(c >= 128, -x, x)
        return x * torch.exp2(st["exponents"][ids, kind, slots].double() - 127)[..., None]

    if case["op"] == "read":
        return {name: torch.cat([rows(r, kind, 0, n) for r, (_, n) in enumerate(lens)])
                for kind, name in enumerate(("key", "value"))}
    outs, at = [], 0
    for r, (q, n) in enumerate(lens):
        k, v = rows(r, 0, 0, n), rows(r, 1, 0, n)
        for c0 in range(0, q, 1024):  # queries a block at a time
            c1 = min(q, c0 + 1024)
            pos = torch.arange(n - q + c0, n - q + c1, device=DEV)[:, None]
            j = torch.arange(n, device=DEV)[None]
            if case["op"] == "tree":
                bits = st["tree_mask"][at + c0:at + c1]
                hidden = (j >= n - q) & ((bits >> (j - (n - q)).clamp(min=0)) % 2 == 0)
            else:
                hidden = (j > pos) & (j >= case["prefix"])
                if case["window"] >= 0:
                    hidden |= pos - j > case["window"]
                if st["doc_starts"] is not None:
                    hidden |= j < st["doc_starts"][at + c0:at + c1, None]
            heads = []
            for head in range(h):
                x = st["query"][at + c0:at + c1, head].double()
                s = x @ k[:, head * hk // h].T / d ** 0.5
                if case["soft_cap"]:
                    s = case["soft_cap"] * torch.tanh(s / case["soft_cap"])
                if case["alibi"]:
                    s = s - st["slopes"][head].double() * (pos - j).abs()
                s = s.masked_fill(hidden, -math.inf)
                p = torch.softmax(s, -1).nan_to_num(0.0)  # a row that sees nothing is 0
                heads.append(p @ v[:, head * hk // h])
            outs.append(torch.stack(heads, 1))
        at += q
    return {"out": torch.cat(outs)}
