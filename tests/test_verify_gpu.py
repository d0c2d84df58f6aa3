"""GPU: drafted tokens checked against the target's probabilities, equal to the
oracle (64-bit sums; a limit is nearer to a border than the sums' rounding once in
10^9 tokens)."""

import numpy as np
import pytest
import torch

from oracle import step as O
from tests.conftest import SEED

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def inputs(dev, B, T, V, dtype, seed, drawn, tree, ids=torch.int64):
    g = torch.Generator(device=dev).manual_seed(seed)
    logits = torch.randn((B, T + 1, V), generator=g, device=dev) * 2
    p = torch.softmax(logits, -1).to(TYPES[dtype])
    u = torch.rand((B, T + 1), generator=g, device=dev)
    q = torch.softmax(logits[:, :T] + 0.5 * torch.randn((B, T, V), generator=g, device=dev), -1).to(TYPES[dtype]) if drawn else None
    parents = (torch.rand((B, T), generator=g, device=dev) * torch.arange(1, T + 1, device=dev)).int() - 1 if tree else None
    rows = parents.long() + 1 if tree else torch.arange(T, device=dev).expand(B, T)
    source = (q if drawn else p.gather(1, rows.unsqueeze(-1).expand(-1, -1, V))).float()
    x = torch.multinomial(source.reshape(-1, V) + 1e-9, 1, generator=g).view(B, T) if B * T else torch.zeros((B, T), device=dev)
    return x.to(ids), p, u, q, parents


def check(x, p, u, q=None, parents=None, lens=None):
    import torch_spyre_amd as tsa

    out, kept, path = tsa.verify_drafts(x, p, u, draft_probs=q, parents=parents, draft_lens=lens)
    host = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    P, Q, U, X = host(p), host(q), host(u), x.cpu().numpy()
    A = None if parents is None else parents.cpu().numpy()
    B, T = X.shape
    for b in range(B):
        want, drawn = O.verify(X[b], P[b], U[b], None if Q is None else Q[b], None if A is None else A[b],
                               None if lens is None else int(lens[b]))
        n = len(want)
        assert int(kept[b]) == n and path[b].tolist() == want + [-1] * (T - n), (b, want, path[b].tolist())
        assert out[b].tolist() == [int(X[b][i]) for i in want] + [drawn] + [-1] * (T - n), (b, n, drawn)
    assert out.dtype == x.dtype and kept.dtype == path.dtype == torch.int32
    return kept


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("kind", ["chain, q", "chain", "tree"])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (1, 7, 100), (3, 5, 4096), (2, 4, 4097), (5, 3, 8191), (4, 25, 1000), (2, 70, 50),
                                   (1, 2, 300001)])
def test_kinds(cuda, dtype, kind, B, T, V):
    x, p, u, q, parents = inputs(cuda, B, T, V, dtype, SEED + V + T, kind == "chain, q", kind == "tree")
    check(x, p, u, q, parents)


@pytest.mark.parametrize("kind", ["chain, q", "chain", "tree"])
@pytest.mark.parametrize("B,T,V", [(64, 2, 40001), (290, 1, 61441)])
def test_many_sequences_of_large_vocabularies(cuda, kind, B, T, V):
    x, p, u, q, parents = inputs(cuda, B, T, V, "f16", SEED + V, kind == "chain, q", kind == "tree")
    check(x, p, u, q, parents)


@pytest.mark.parametrize("T", [64, 65, 150, 1024])
def test_many_siblings(cuda, T):
    """All of them continue the context, most are rejected, tokens occur again."""
    x, p, _, _, _ = inputs(cuda, 3, T, 3 * T, "f32", SEED + T, False, True)
    u = torch.rand((3, T + 1), device=cuda)
    u[:, :T] = u[:, :T].clamp(min=0.02)
    check(x, p, u, None, torch.full((3, T), -1, dtype=torch.int32, device=cuda))


@pytest.mark.parametrize("kind", ["chain, q", "chain", "tree"])
def test_uneven_drafts_and_int32(cuda, kind):
    x, p, u, q, parents = inputs(cuda, 9, 6, 777, "f32", SEED, kind == "chain, q", kind == "tree", torch.int32)
    lens = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, -1], dtype=torch.int32, device=cuda)
    check(x, p, u, q, parents, lens)


def test_many_runs_and_every_outcome(cuda):
    """Many short lines: every number of kept tokens occurs."""
    x, p, u, q, _ = inputs(cuda, 400, 4, 30, "f32", SEED + 1, True, False)
    assert set(check(x, p, u, q).tolist()) == set(range(5))


def test_no_drafts_is_sampling(cuda):
    x, p, u, _, _ = inputs(cuda, 50, 0, 5000, "f32", SEED + 2, False, False)
    check(x, p, u)


def test_strides(cuda):
    B, T, V = 3, 4, 501
    x, p, u, q, parents = inputs(cuda, B, T, V, "bf16", SEED + 3, True, True)
    wide = torch.zeros((T + 1, B, V + 7), dtype=p.dtype, device=cuda)
    wide[..., 3:V + 3] = p.transpose(0, 1)
    p2 = wide[..., 3:V + 3].transpose(0, 1)
    check(x.t().contiguous().t(), p2, u.t().contiguous().t(), q.transpose(1, 2).contiguous().transpose(1, 2))
    check(x.t().contiguous().t(), p2, u.t().contiguous().t(), None, parents.t().contiguous().t())
    check(x[:1].expand(B, T), p[:1].expand(B, T + 1, V), u)


def test_limits(cuda):
    """Uniforms at 0 and at 1 and beyond, NaN; rows of one token; ties at a border."""
    p = torch.zeros((1, 2, 9000), device=cuda)
    p[0, :, [3, 4096, 8999]] = torch.tensor([0.25, 0.25, 0.5], device=cuda)
    x = torch.tensor([[4096]], device=cuda)
    for u0 in (0.0, 0.2499, 0.25, 1.0, float("nan")):
        for u1 in (0.0, 0.25, 0.3333, 0.5, 0.9999, 1.0, 2.0, -1.0):
            check(x, p, torch.tensor([[u0, u1]], device=cuda))


def test_tokens_outside_and_parents_outside(cuda):
    x, p, u, _, _ = inputs(cuda, 4, 5, 64, "f32", SEED + 4, False, False)
    x[0, 0], x[1, 2], x[2, 1] = -1, 64, 2**40
    parents = torch.tensor([[-1, 0, 1, 2, 3], [-1, -1, -2, 3, 0], [-1, 1, 1, 7, 2], [0, 0, 0, 0, 0]], dtype=torch.int32, device=cuda)
    check(x, p, u)
    check(x, p, u, None, parents)


def test_siblings_twice_and_all_of_the_mass(cuda):
    """A token tried twice, and rejected siblings that hold all of p: drawn from p itself."""
    p = torch.zeros((2, 5, 10), device=cuda)
    p[:, :, 2], p[:, :, 5] = 0.5, 0.5
    x = torch.tensor([[2, 2, 5, 5]] * 2, device=cuda)
    parents = torch.full((2, 4), -1, dtype=torch.int32, device=cuda)
    check(x, p, torch.tensor([[0.9, 0.0, 1.0, 0.0, 0.7], [0.9, 0.0, 0.9999, 0.5, 0.1]], device=cuda), None, parents)


def test_equal_draft_and_target(cuda):
    """max(p - q, 0) without any weight behind a rejection (u = 1): drawn from p."""
    x, p, u, _, _ = inputs(cuda, 3, 2, 5000, "f32", SEED + 5, False, False)
    u[:, 0] = 1.0
    check(x, p, u, p[:, :2].clone())


def test_not_finite(cuda):
    """Negative, NaN and infinite probabilities count as nothing."""
    x, p, u, q, _ = inputs(cuda, 6, 3, 5000, "f32", SEED + 6, True, False)
    p[0, 0, 7], p[1, :, 100:4000], p[2, 0], p[3, 1, 4999] = float("nan"), float("inf"), -1.0, float("inf")
    p[4] = float("nan")
    q[0, 0, :50], q[5, 1] = float("nan"), float("inf")
    check(x, p, u, q)
    check(x, p, u)


def test_more_than_one_pass_over_the_runs(cuda):
    """Over 64 runs of the vocabulary."""
    x, p, u, q, _ = inputs(cuda, 2, 1, 300000, "bf16", SEED + 7, True, False)
    p, q = (torch.cat((t, t * 0.5), -1) for t in (p, q))
    check(x, p, u, q)
    u[:, 1] = 0.99
    check(x, p, torch.where(u > 1, u, u * 0 + 0.99), q)
