"""GPU: block tables and slot maps from lengths, pages given back, against the oracle."""

import numpy as np
import pytest
import torch

from oracle import step as O
from tests.conftest import SEED

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def state(B, W, F, ctx, seed, spread=10**6):
    """A pool of F pages in use: rows hold their contexts' pages, the ring has been gone round."""
    rng = np.random.default_rng(seed)
    held = [min(-(-c // 64), W) for c in ctx]
    ids = rng.permutation(F)
    table, at = np.full((B, W), -1), 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    taken = int(rng.integers(0, spread))
    ring = np.full(F, -7)
    for k in range(F - at):
        ring[(taken + k) % F] = ids[at + k]
    return table, held, ring, (taken, taken + F - at)


def run(dev, table, held, ctx, new, ring, cursor, **size):
    import torch_spyre_amd as tsa

    t, h, r = i32(table, dev), i32(held, dev), i32(ring, dev)
    c = torch.tensor(cursor, dtype=torch.int64, device=dev)
    for _ in range(2):  # the same inputs, the same results
        plan = tsa.plan_pages(t, h, i32(ctx, dev), i32(new, dev), r, c, **size)
    want = O.plan_pages(table, held, ctx, new, ring, cursor, **size)
    assert np.array_equal(t.cpu().numpy(), want[0])
    for got, ref in zip((plan.positions, plan.slots, plan.held, plan.cursor, plan.starts), want[1:]):
        assert np.array_equal(got.cpu().numpy(), np.asarray(ref))
    assert plan.slots.dtype == torch.int64 and plan.positions.dtype == torch.int32
    assert np.array_equal(r.cpu().numpy(), ring) and h.tolist() == list(held) and c.tolist() == list(cursor)
    return t, plan, r


CASES = [  # B, most context, most new tokens
    (1, 0, 1), (1, 64, 1), (1, 63, 1), (1, 1000, 200), (7, 130, 65), (64, 5000, 25), (257, 100, 3), (1000, 300, 1), (4096, 70, 2)]


@pytest.mark.parametrize("B,ctx,new", CASES)
@pytest.mark.parametrize("packed", [False, True])
def test_plan(cuda, B, ctx, new, packed):
    rng = np.random.default_rng(SEED + B)
    c, n = rng.integers(0, ctx + 1, B), rng.integers(0, new + 1, B)
    c[0], n[-1] = ctx, new
    W = -(-(ctx + new) // 64) + 2
    total = sum(-(-(x + y) // 64) for x, y in zip(c, n))
    s = state(B, W, total + 3, c, SEED + B + 1)
    size = {"tokens": int(n.sum()) + (B % 3)} if packed else {"length": int(n.max()) + (B % 3)}
    run(cuda, s[0], s[1], c, n, s[2], s[3], **size)


@pytest.mark.parametrize("free", [0, 1, 2, 5])
def test_ring_runs_out(cuda, free):
    c, n = [100, 0, 64, 10], [100, 130, 1, 0]
    table, held, ring, _ = state(4, 4, 5 + 5, c, SEED)
    for size in ({"length": 130}, {"tokens": 231}):
        run(cuda, table, held, c, n, ring, (1003, 1003 + free), **size)


def test_rows_run_out_and_odd_lengths(cuda):
    """A row of the table that is too narrow, negative lengths, more tokens than places."""
    table, held, ring, cursor = state(4, 2, 20, [100, 0, 64, 0], SEED + 2)
    for size in ({"length": 5}, {"length": 0}, {"tokens": 9}, {"tokens": 0}):
        run(cuda, table, held, [100, 0, 64, -5], [200, -3, 64, 3], ring, cursor, **size)
    run(cuda, table, held, [100, 0, 64, 0], [0, 0, 0, 0], ring, cursor, tokens=3)


def test_no_sequences_no_pages(cuda):
    import torch_spyre_amd as tsa

    e = torch.empty((0,), dtype=torch.int32, device=cuda)
    c = torch.tensor([5, 5], dtype=torch.int64, device=cuda)
    plan = tsa.plan_pages(e.view(0, 3), e, e, e, e, c, tokens=2)
    assert plan.positions.tolist() == [-1, -1] and plan.slots.tolist() == [-1, -1] and plan.starts.tolist() == [0]
    assert plan.cursor.tolist() == [5, 5] and plan.held.shape == (0,)
    one = torch.tensor([3], dtype=torch.int32, device=cuda)
    plan = tsa.plan_pages(one.view(1, 1)[:, :0], one * 0, one, one, e, c, length=2)
    assert plan.slots.tolist() == [[-1, -1]] and plan.positions.tolist() == [[3, 4]] and plan.held.tolist() == [0]
    held, cur = tsa.release_pages(e.view(0, 3), e, e, e, c)
    assert held.shape == (0,) and cur.tolist() == [5, 5]


@pytest.mark.parametrize("B,ctx", [(1, 1), (3, 200), (64, 3000), (300, 500)])
def test_release(cuda, B, ctx):
    import torch_spyre_amd as tsa

    rng = np.random.default_rng(SEED + B + 5)
    c = rng.integers(0, ctx + 1, B)
    table, held, ring, cursor = state(B, -(-ctx // 64) + 1, sum(-(-int(x) // 64) for x in c) + 4, c, SEED + B + 6)
    lens = np.where(rng.random(B) < 0.3, 0, rng.integers(0, ctx + 100, B))
    t, r = i32(table, cuda), i32(ring, cuda)
    for _ in range(2):
        h, cur = tsa.release_pages(t, i32(held, cuda), i32(lens, cuda), r, torch.tensor(cursor, dtype=torch.int64, device=cuda))
    want = O.release_pages(table, held, lens, ring, cursor)
    assert np.array_equal(r.cpu().numpy(), want[0]) and np.array_equal(h.cpu().numpy(), want[1])
    assert tuple(cur.tolist()) == want[2] and np.array_equal(t.cpu().numpy(), table)


def test_pool_over_many_steps(cuda):
    """PagePool through steps of admissions, drafts and ends: no page is held twice, none is lost."""
    import torch_spyre_amd as tsa

    rng = np.random.default_rng(SEED + 9)
    pool = tsa.PagePool(40, 6, 12, device=cuda)
    lens = np.zeros(6, dtype=np.int64)
    for step in range(30):
        new = rng.integers(0, 90, 6)
        new = np.where(lens + new > 12 * 64, 0, new)
        plan = pool.plan(i32(lens, cuda), i32(new, cuda), length=90)
        held = pool.held.tolist()
        lens = np.minimum(lens + new, np.array(held) * 64)  # what found pages
        slots = plan.slots[plan.slots >= 0]
        assert len(set(slots.tolist())) == len(slots)
        lens = np.where(rng.random(6) < 0.25, 0, np.maximum(lens - rng.integers(0, 30, 6), 0))
        pool.release(i32(lens, cuda))
        held, (taken, returned) = pool.held.tolist(), pool.cursor.tolist()
        ring = pool.free_pages.tolist()
        ids = [x for b, h in enumerate(held) for x in pool.block_table[b, :h].tolist()]
        ids += [ring[c % 40] for c in range(taken, returned)]
        assert sorted(ids) == list(range(40)) and held == [-(-int(x) // 64) for x in lens]
