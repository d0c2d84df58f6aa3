"""CPU: pins of the oracle of pages, draft verification and latent attention."""

import numpy as np

from oracle import step as O
from tests.conftest import SEED


def test_pages_by_hand():
    table = [[7, -1, -1], [-1, -1, -1]]
    t, pos, slots, held, cursor, starts = O.plan_pages(table, [1, 0], [63, 0], [2, 65], [5, 4, 3, 2], (6, 9), tokens=70)
    # the ring is at 6 mod 4: page 3, then 2, then (8 mod 4) 5; the second sequence needs two
    assert t.tolist() == [[7, 3, -1], [2, 5, -1]] and held.tolist() == [2, 2] and cursor == (9, 9)
    assert pos[:3].tolist() == [63, 64, 0] and slots[:3].tolist() == [7 * 64 + 63, 3 * 64, 2 * 64]
    assert slots[66] == 5 * 64 and starts.tolist() == [0, 2, 67] and pos[67:].tolist() == [-1] * 3
    ring, held, cursor = O.release_pages(t, held, [64, 0], [5, 4, 3, 2], cursor)
    assert ring.tolist() == [5, 3, 2, 5] and held.tolist() == [1, 0] and cursor == (9, 12)


def test_pages_run_out():
    t, pos, slots, held, cursor, _ = O.plan_pages([[-1] * 4] * 2, [0, 0], [0, 0], [100, 100], [9, 8, 7], (0, 3), length=100)
    assert held.tolist() == [2, 1] and cursor == (3, 3) and slots[1, 63] == 7 * 64 + 63 and slots[1, 64] == -1
    assert pos[1, 99] == 99


def test_chain_is_the_targets_distribution():
    """Kept or drawn, the first token is distributed as the target's row, whatever the draft's."""
    rng = np.random.default_rng(SEED)
    V, N = 5, 40000
    p, q = rng.dirichlet(np.ones(V), 2), rng.dirichlet(np.ones(V), 1)
    counts = np.zeros(V)
    for x, u in zip(rng.choice(V, N, p=q[0]), rng.random((N, 2))):
        path, drawn = O.verify([x], p, u, draft=q)
        counts[x if path else drawn] += 1
    # five standard deviations of a count
    assert (np.abs(counts - N * p[0]) <= 5 * np.sqrt(N * p[0] * (1 - p[0]))).all()


def test_tree_is_the_targets_distribution():
    rng = np.random.default_rng(SEED + 1)
    V, N = 5, 40000
    p = rng.dirichlet(np.ones(V), 4)
    counts = np.zeros(V)
    for u in rng.random((N, 4)):  # three siblings, one token twice
        path, drawn = O.verify([2, 4, 2], p, u, parents=[-1, -1, -1])
        counts[[2, 4, 2][path[0]] if path else drawn] += 1
    assert (np.abs(counts - N * p[0]) <= 5 * np.sqrt(N * p[0] * (1 - p[0]))).all()


def test_verify_by_hand():
    p = np.array([[0.5, 0.5, 0.0], [0.0, 0.25, 0.75], [1.0, 0.0, 0.0]])
    assert O.verify([1, 2], p, [0.49, 0.7, 0.0]) == ([0, 1], 0)
    assert O.verify([1, 2], p, [0.5, 0.7, 0.3]) == ([], 0)       # u < p is strict; 1 is out
    assert O.verify([1, 2], p, [0.1, 0.75, 0.0]) == ([0], 1)
    assert O.verify([1, 2], p, [0.1, 0.9, 0.9], n=1) == ([0], 2)
    assert O.verify([2], p[:2], [0.0, 0.5]) == ([], 1)           # half of the total is not above it
    assert O.verify([0], p[1:], [0.3, 1.0], draft=p[1:2]) == ([], 2)  # p == q: drawn from p; a limit at the total
    assert O.verify([-1], p[:2], [0.0, 0.2]) == ([], 0)
    assert O.verify([], np.array([[np.nan, -1.0, np.inf]]), [0.5]) == ([], -1)


def test_attend_expanded_and_absorbed():
    """The two forms are the same attention."""
    rng = np.random.default_rng(SEED + 2)
    n, rank, D = 9, 16, 6
    c, r, q, s = rng.normal(size=(n, rank)), rng.normal(size=(n, 4)), rng.normal(size=(1, D)), rng.normal(size=(1, 4))
    wk, wv = rng.normal(size=(D, rank)), rng.normal(size=(D, rank))
    keep = rng.random((1, n)) < 0.6
    a = O.attend(np.concatenate((q @ wk, s), 1), np.concatenate((c, r), 1), c, keep, 0.3)
    e = O.attend(np.concatenate((q, s), 1), np.concatenate((c @ wk.T, r), 1), c @ wv.T, keep, 0.3)
    np.testing.assert_allclose(a[0] @ wv.T, e[0], rtol=1e-12)
    np.testing.assert_allclose(a[1], e[1], rtol=1e-12)
    out, lse, _, _ = O.attend(q, c[:, :D], c, np.zeros((1, n), bool), 1.0)
    assert not out.any() and lse[0] == -np.inf
