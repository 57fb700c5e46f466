"""GPU: after a step or a release that did not fit, nothing is taken, given or written until it is looked at."""
import pytest
import torch

from oracle import heads_ref as ref
from paceserve_b200 import cabi
from paceserve_b200.block_tables import BlockTables
from tests.test_step_tables_gpu import DEV, Tables, check_build, ints, lens, nothing_done

pytestmark = pytest.mark.gpu


def state(t):
    return [x.clone() for x in (t.block_tables, t.free_pages, t.free_count)]


def leads_nowhere(step):
    for x in (step.append_indptr, step.kv_indptr, step.kv_last_page_len):
        assert (x == 0).all()
    for x in (step.batch_indices, step.positions, step.slot_mapping):
        assert (x == -1).all()


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_steps_after_one_that_did_not_fit():
    """The lengths move on, as an engine's that runs a step ahead: the pages that were not given are no one's."""
    t = BlockTables(3, 8, 4, 6, 32, DEV)
    t.begin_step(ints([0, 0, 0]), ints([8, 4, 0]))
    t.check()
    before = state(t)
    leads_nowhere(t.begin_step(ints([8, 4, 0]), ints([4, 4, 16])))  # 6 pages of 3
    leads_nowhere(t.begin_step(ints([12, 8, 16]), ints([1, 1, 1])))  # 3 pages, held ones not given
    leads_nowhere(t.begin_step(ints([12, 8, 16]), ints([0, 0, 0])))  # none needed
    t.release(ints([12, 8, 16]), ints([8, 4, 0]))
    t.begin_step(ints([-1, 8, 16]), ints([0, 0, 0]))
    assert same(before, state(t))
    with pytest.raises(RuntimeError, match="not enough free pages") as e:
        t.check()
    assert "negative" not in str(e.value)  # what stopped it, not what came after
    t.check()
    # with the lengths that the last step left, it goes on
    step = t.begin_step(ints([8, 4, 0]), ints([1, 0, 5]))
    t.check()
    rows, free = before[0].tolist(), before[1].tolist()
    want, height = ref.build(rows, [8, 4, 0], [1, 0, 5], 4, free, 3, 32)
    got = {k: v.tolist() for k, v in step._asdict().items()}
    got["kv_indices"] = got["kv_indices"][:len(want["kv_indices"])]
    assert got == want and t.free_count.item() == height and t.block_tables.tolist() == rows


def test_steps_after_a_release_that_did_not_fit():
    t = BlockTables(2, 4, 16, 8, 64, DEV)
    t.begin_step(ints([0, 0]), ints([40, 5]))
    before = state(t)
    t.release(ints([40, 5]), ints([41, 0]))  # more kept than held
    t.release(ints([40, 5]), ints([0, 0]))
    leads_nowhere(t.begin_step(ints([40, 5]), ints([1, 1])))
    assert same(before, state(t))
    with pytest.raises(RuntimeError, match="more tokens are kept than held$"):
        t.check()
    t.release(ints([40, 5]), ints([0, 0]))
    t.check()
    assert t.free_count.item() == 8


@pytest.mark.parametrize("n", [3, 900])  # one CTA, and many
def test_replays_past_the_last_page(n):
    """A captured step whose lengths grow by themselves runs out of pages; no later replay writes a slot."""
    page, ctx = 4, 37
    held, _ = lens(n, ctx, 1, n)
    need = [-(-h // page) for h in held]
    t = BlockTables(n, 64, page, sum(need) + 2 * n, max(sum(held), n), DEV)
    zero, one = ints([0] * n), ints([1] * n)
    t.begin_step(zero, ints(held))
    t.check()
    seq = ints(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = t.begin_step(seq, one)
        seq.add_(one)
    rows, free, height = t.block_tables.tolist(), t.free_pages.tolist(), t.free_count.item()
    have, fits = list(held), True
    for i in range(30):
        graph.replay()
        short = sum(h % page == 0 for h in have) > height
        fits = fits and not short
        if fits:
            want, height = ref.build(rows, have, [1] * n, page, free, height, step.positions.numel())
            assert step.slot_mapping.tolist() == want["slot_mapping"]
            have = [h + 1 for h in have]
        else:
            leads_nowhere(step)
            # what would fit the pages that are left: one request, with a page it was not given
            seq.zero_()
            one.zero_()
            seq[0], one[0] = have[0] + page, 1
        assert t.free_count.item() == height
    assert not fits and t.block_tables.tolist() == rows and t.free_pages.tolist() == free
    with pytest.raises(RuntimeError, match="not enough free pages"):
        t.check()
    # a request is done, the lengths are those of the last step that fitted: the next one fits again
    have_now = ints(have)
    done = torch.arange(n, device=DEV) % 3 == 0
    t.release(have_now, torch.where(done, 0, have_now).int())
    seq.copy_(torch.where(done, 0, have_now))
    one.fill_(1)
    graph.replay()
    t.check()
    slots = step.slot_mapping.tolist()[:n]
    assert len(set(slots)) == n and min(slots) >= 0
    table, left = t.block_tables.tolist(), torch.where(done, 0, have_now).tolist()
    used = [p for b in range(n) for p in table[b][:-(-(left[b] + 1) // page)]]
    assert sorted(used + t.free_pages.tolist()[:t.free_count.item()]) == list(range(t.free_pages.numel()))


@pytest.mark.parametrize("n", [40, 1000])
def test_status_that_is_set_is_left(n):
    """The op: any bit that is set in *status stops it, and stays the only one."""
    seq, new = lens(n, 200, 30, n)
    t = Tables(seq, new, 16)
    free = list(t.free)
    t.status.fill_(cabi.PACE_TABLES_SHORT_TOKENS)
    t.build()
    nothing_done(t, free)
    assert t.status.item() == cabi.PACE_TABLES_SHORT_TOKENS
    for k in ("append_indptr", "kv_indptr", "kv_last_page_len"):
        assert (t.out[k] == 0).all()
    for k in ("batch_indices", "positions", "slot_mapping"):
        assert (t.out[k] == -1).all()
    t.release(seq, [0] * n)
    nothing_done(t, free)
    t.release([-1] * n, [0] * n)
    nothing_done(t, free)
    assert t.status.item() == cabi.PACE_TABLES_SHORT_TOKENS
    t.status.zero_()
    t.build()
    check_build(t)
