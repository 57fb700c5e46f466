"""GPU: step tables against a walk over the requests, entry by entry."""
import random

import pytest
import torch

from oracle import heads_ref as ref
from paceserve_b200 import cabi
from paceserve_b200 import kv_transfer_ops as kv
from paceserve_b200.block_tables import BlockTables

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ints(x, kind=torch.int32):
    return torch.tensor(x, dtype=kind, device=DEV)


class Tables:
    """The op's arrays with room to spare, filled so that what is not written shows."""

    def __init__(self, seq, new, page, spare=3, pad_tokens=5, blocks=None, seed=0):
        r = random.Random(seed)
        held = [-(-n // page) for n in seq]
        need = [-(-(n + q) // page) for n, q in zip(seq, new)]
        self.page, self.seq, self.new = page, seq, new
        self.blocks = max(need + [1]) if blocks is None else blocks
        ids = list(range(sum(need) + spare))
        r.shuffle(ids)
        self.rows = [[ids.pop() for _ in range(h)] + [-5] * (self.blocks - h) for h in held]
        self.free = ids
        self.tokens = sum(new) + pad_tokens
        wide = torch.full((max(1, len(seq)), self.blocks + 2), -9, dtype=torch.int32, device=DEV)
        self.table = wide[:len(seq), :self.blocks]
        if seq:
            self.table.copy_(ints(self.rows))
        self.wide = wide
        self.free_pages = ints(self.free + [-3] * 2)
        self.count = ints([len(self.free)])
        n = len(seq)
        self.out = {k: torch.full((m,), -7, dtype=kind, device=DEV) for k, m, kind in [
            ("append_indptr", n + 1, torch.int32), ("kv_indptr", n + 1, torch.int32),
            ("kv_indices", sum(need) + 4, torch.int32), ("kv_last_page_len", n, torch.int32),
            ("batch_indices", self.tokens, torch.int32), ("positions", self.tokens, torch.int64),
            ("slot_mapping", self.tokens, torch.int64)]}
        self.status, self.arrivals = ints([0]), ints([0])

    def build(self):
        o = self.out
        kv.build_step_tables(self.table, ints(self.seq), ints(self.new), self.page, self.free_pages,
                             self.count, o["append_indptr"], o["kv_indptr"], o["kv_indices"],
                             o["kv_last_page_len"], o["batch_indices"], o["positions"],
                             o["slot_mapping"], self.status, self.arrivals)

    def release(self, held, kept):
        kv.release_pages(self.table, ints(held), ints(kept), self.page, self.free_pages, self.count,
                         self.status, self.arrivals)


def check_build(t):
    want, height = ref.build(t.rows, t.seq, t.new, t.page, t.free, len(t.free), t.tokens)
    got = {k: v.tolist() for k, v in t.out.items()}
    pages = len(want["kv_indices"])
    assert got["kv_indices"][pages:] == [-7] * (len(got["kv_indices"]) - pages)
    got["kv_indices"] = got["kv_indices"][:pages]
    for k, v in want.items():
        assert got[k] == v, k
    assert t.table.tolist() == t.rows and (t.wide[:, t.blocks:] == -9).all()
    assert t.count.item() == height and t.status.item() == 0 and t.arrivals.item() == 0
    assert t.free_pages.tolist()[:len(t.free)] == t.free


def lens(n, ctx, new, seed):
    r = random.Random(seed)
    return [r.randrange(ctx + 1) for _ in range(n)], [r.randrange(new + 1) for _ in range(n)]


@pytest.mark.parametrize("seq,new,page", [
    ([0], [1], 16), ([15], [1], 16), ([16], [1], 16), ([17], [0], 16), ([0], [0], 16), ([], [], 16),
    ([0, 0, 5], [0, 33, 0], 8), ([100, 0, 31], [1, 300, 1], 32), ([7, 7, 7], [1, 1, 1], 1),
    ([10, 3], [5, 11], 5), ([9] * 40, [1] * 40, 3), ([0, 1000], [0, 0], 16)])
def test_few_requests(seq, new, page):
    t = Tables(seq, new, page)
    t.build()
    check_build(t)


@pytest.mark.parametrize("n,ctx,new,page", [(64, 8191, 1, 16), (1000, 300, 40, 16), (513, 70, 3, 7),
                                            (4097, 40, 2, 8), (8192, 20, 1, 16), (33, 40000, 600, 8)])
def test_many_requests(n, ctx, new, page):
    seq, add = lens(n, ctx, new, n)
    t = Tables(seq, add, page)
    t.build()
    check_build(t)
    # giving it back leaves the stack as it was
    t.release([a + b for a, b in zip(seq, add)], seq)
    assert t.count.item() == len(t.free) and t.free_pages.tolist()[:len(t.free)] == t.free
    assert t.status.item() == 0 and t.arrivals.item() == 0


def test_release_some_and_all():
    seq, page = [40, 17, 0, 64, 5], 16
    t = Tables(seq, [0] * 5, page, spare=2)
    free = list(t.free)
    t.free_pages = torch.cat([t.free_pages, torch.zeros(40, dtype=torch.int32, device=DEV)])
    kept = [17, 16, 0, 0, 5]
    t.release(seq, kept)
    given = [t.rows[0][2], t.rows[1][1]] + t.rows[3][:4]  # pages 2 of 3, 1 of 2, 0-3 of 4
    assert t.count.item() == len(free) + 6
    assert t.free_pages.tolist()[:len(free) + 6] == free + given[::-1]
    assert t.table.tolist() == t.rows


def nothing_done(t, free):
    assert t.table.tolist() == t.rows and t.count.item() == len(free)
    assert t.free_pages.tolist()[:len(free)] == free and t.arrivals.item() == 0


@pytest.mark.parametrize("what,bit", [
    ("negative", cabi.PACE_TABLES_BAD_LENGTH), ("negative_new", cabi.PACE_TABLES_BAD_LENGTH),
    ("row", cabi.PACE_TABLES_SHORT_ROW), ("indices", cabi.PACE_TABLES_SHORT_INDICES),
    ("tokens", cabi.PACE_TABLES_SHORT_TOKENS), ("pages", cabi.PACE_TABLES_NO_PAGES),
    ("huge", cabi.PACE_TABLES_SHORT_ROW), ("height", cabi.PACE_TABLES_NO_PAGES)])
def test_what_does_not_fit_changes_nothing(what, bit):
    seq, new = lens(300, 200, 30, 1)
    t = Tables(seq, new, 16, spare=0)
    free = list(t.free)
    if what == "negative":
        t.seq = seq[:7] + [-1] + seq[8:]
    elif what == "negative_new":
        t.new = new[:7] + [-(1 << 31)] + new[8:]
    elif what == "row":
        t.new = new[:7] + [16 * t.blocks + 1 - seq[7]] + new[8:]
    elif what == "huge":
        t.seq, t.new = [(1 << 31) - 1] * 300, [(1 << 31) - 1] * 300
    elif what == "indices":
        t.out["kv_indices"] = t.out["kv_indices"][:-5]
    elif what == "tokens":
        for k in ("batch_indices", "positions", "slot_mapping"):
            t.out[k] = t.out[k][:sum(new) - 1]
    elif what == "pages":
        free = free[1:]
        t.count.fill_(len(free))
        t.free_pages = ints(free)
    else:
        t.count.fill_(len(free) + 100)  # more than the stack holds
    t.build()
    assert t.status.item() & bit
    if what == "height":
        assert t.count.item() == len(free) + 100
        t.count.fill_(len(free))
    nothing_done(t, free)
    for k in ("append_indptr", "kv_indptr", "kv_last_page_len"):
        assert (t.out[k] == 0).all(), k
    for k in ("batch_indices", "positions", "slot_mapping"):
        assert (t.out[k] == -1).all(), k
    assert (t.out["kv_indices"] == -7).all()


@pytest.mark.parametrize("held,kept,bit", [
    ([20, 5], [21, 0], cabi.PACE_TABLES_BAD_LENGTH), ([20, -1], [0, -1], cabi.PACE_TABLES_BAD_LENGTH),
    ([20, 100], [0, 0], cabi.PACE_TABLES_SHORT_ROW), ([32, 32], [0, 0], cabi.PACE_TABLES_NO_PAGES)])
def test_release_that_does_not_fit(held, kept, bit):
    t = Tables([32, 32], [0, 0], 16, spare=1)
    free = list(t.free)
    t.release(held, kept)
    assert t.status.item() & bit
    nothing_done(t, free)


def test_steps_of_an_engine_in_a_graph():
    """Requests come, grow by a token a step and go; the step is captured once."""
    page, rows = 4, 6
    tables = BlockTables(rows, 16, page, 40, 24, DEV)
    seq, new = ints([0] * rows), ints([0] * rows)
    tables.begin_step(seq, new)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = tables.begin_step(seq, new)
        seq.add_(new)
    r = random.Random(0)
    have, pages = [0] * rows, [[] for _ in range(rows)]
    for i in range(60):
        add = [0] * rows
        for b in range(rows):
            if have[b] == 0:
                add[b] = r.randrange(0, 9) if sum(add) < 10 else 0
            elif r.random() < 0.1:
                tables.release(ints([have[b] if c == b else 0 for c in range(rows)]), ints([0] * rows))
                have[b], pages[b] = 0, []
            else:
                add[b] = 1
        if any(a and h + a > 64 for a, h in zip(add, have)):
            break
        seq.copy_(ints(have))
        new.copy_(ints(add))
        graph.replay()
        tables.check()
        have = [a + b for a, b in zip(have, add)]
        assert seq.tolist() == have
        table = tables.block_tables.tolist()
        used = []
        for b in range(rows):
            n = -(-have[b] // page)
            assert table[b][:len(pages[b])] == pages[b]
            pages[b] = table[b][:n]
            used += pages[b]
        free = tables.free_pages.tolist()[:tables.free_count.item()]
        assert sorted(used + free) == list(range(40))  # every page has one owner
        assert step.kv_indices.tolist()[:len(used)] == used
        slots = [pages[b][p // page] * page + p % page for b in range(rows)
                 for p in range(have[b] - add[b], have[b])]
        assert step.slot_mapping.tolist() == slots + [-1] * (24 - len(slots))


def test_class_refuses_and_tells():
    tables = BlockTables(2, 4, 16, 3, 100, DEV)
    tables.begin_step(ints([0, 0]), ints([40, 16]))  # 4 pages of 3
    with pytest.raises(RuntimeError, match="not enough free pages"):
        tables.check()
    tables.check()
    tables.begin_step(ints([0, 0]), ints([40, 0]))
    tables.check()
    with pytest.raises(RuntimeError, match="more lengths than rows"):
        tables.begin_step(ints([0] * 3), ints([0] * 3))
    with pytest.raises(RuntimeError, match="differ in length"):
        tables.begin_step(ints([0, 0]), ints([0]))
    with pytest.raises(RuntimeError, match="seq_lens"):
        tables.begin_step(ints([0, 0], torch.int64), ints([0, 0]))
    with pytest.raises(RuntimeError, match="all sizes"):
        BlockTables(0, 4, 16, 3, 100, DEV)


def test_many_steps_without_a_pause():
    """Every CTA of every call has the height that the call before left."""
    n, page = 700, 16
    held, new = lens(n, 500, 60, 5)
    t = BlockTables(n, 40, page, 40 * n, 501 * n)
    seq, new = ints(held), ints(new)
    t.begin_step(torch.zeros_like(seq), seq)
    t.check()
    height, stack = t.free_count.item(), t.free_pages.clone()
    total = seq + new
    for _ in range(300):
        step = t.begin_step(seq, new)
        t.release(total, seq)
    t.check()
    assert t.free_count.item() == height and torch.equal(t.free_pages, stack)
    assert step.append_indptr[-1].item() == new.sum().item()
    used = step.kv_indices[:step.kv_indptr[-1].item()].tolist()
    assert len(set(used)) == len(used)  # no page twice
