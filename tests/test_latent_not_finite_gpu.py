"""GPU: NaN and infinities that the rows of latent attention attend, feature by feature, against
64 bits (the tolerances of finite features are those of test_latent_gpu.py)."""

import numpy as np
import pytest
import torch

from oracle import step as O
from tests.conftest import SEED
from tests.test_latent_gpu import close, keep_of, randn

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def close_features(out, lse, ref, n_keys, v_top):
    """Features that are not finite equal, the others and the logsumexp within the tolerance."""
    want, wl, size, reach = (x.copy() for x in ref)
    got = out.double().cpu().numpy().reshape(want.shape)
    odd = ~np.isfinite(want) & np.isfinite(wl)[:, None]
    assert np.array_equal(got[odd], want[odd], equal_nan=True)
    assert np.isfinite(got[~odd & np.isfinite(wl)[:, None]]).all()
    got[odd] = want[odd] = size[odd] = 0.0
    close(torch.from_numpy(got), lse, (want, wl, size, reach), n_keys, v_top)


def prompt(dev, T, ctx, counts, D, put, H=2, seed=0):
    """Runs B prompts before and after `put` changes their values; checks both and returns them."""
    import torch_spyre_amd as tsa

    B, L = len(ctx), max(c + n for c, n in zip(ctx, counts))
    kv, kr = randn((B, L, H, 2 * D), dev, SEED + seed, 0.5), randn((B, L, 64), dev, SEED + seed + 1, 0.5)
    q = randn((B, T, H, D + 64), dev, SEED + seed + 2)
    k, v = kv[..., :D], kv[..., D:]
    lens, new = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (ctx, counts))
    results = []
    for change in (None, put):
        if change:
            change(k, v)
        out, lse = tsa.latent_attention(q[..., :D], q[..., D:], k, kr, v, lens, new, return_lse=True)
        Q, K, V, R = (x.double().cpu().numpy() for x in (q, k, v, kr))
        for b in range(B):
            n = ctx[b] + counts[b]
            for h in range(H):
                with np.errstate(invalid="ignore"):
                    ref = O.attend(Q[b, :, h], np.concatenate((K[b, :n, h], R[b, :n]), -1), V[b, :n, h],
                                   keep_of(T, 1, ctx[b], counts[b]), (D + 64) ** -0.5)
                close_features(out[b, :, h], lse[b, :, h], ref, n, 8.0)
        results.append((out, lse))
    return results


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("T,at", [(300, 200), (300, 255), (300, 256), (300, 63), (100, 64), (33, 0), (1, 0)])
def test_one_feature_of_a_value(cuda, D, bad, T, at):
    """Only that feature of the rows that attend it, in the row block of the value and behind it; no logsumexp."""
    def put(k, v):
        v[0, at, 1, 5] = bad

    clean, got = prompt(cuda, T, [0, 70], [T, T], D, put, seed=T)
    assert torch.equal(got[1], clean[1])
    keep = torch.ones(got[0].shape, dtype=torch.bool, device=cuda)
    keep[0, at:, 1, 5] = False
    assert torch.equal(got[0][keep], clean[0][keep]) and not got[0][~keep].isfinite().any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,ctx", [(290, 0), (150, 37), (40, 100), (3, 5)])
def test_many_values(cuda, D, T, ctx):
    """Several in a tile, in both its halves, some of both signs in one feature, all features of a token."""
    def put(k, v):
        for i, (t, f, x) in enumerate([(0, 0, INF), (1, D - 1, NAN), (2, 3, INF), (2, 40, -INF), (17, 3, -INF), (18, 33, NAN),
                                       (31, 40, -INF), (63, 63, INF), (64, 8, INF), (130, 9, NAN), (261, 60, -INF)]):
            if ctx + t < v.shape[1]:
                v[0, ctx + t, i % 2, f] = x
        if T > 140:
            v[0, ctx + 139, 0] = NAN
            v[0, ctx + 140, 1] = INF

    prompt(cuda, T, [ctx], [T], D, put, seed=T + 1)


@pytest.mark.parametrize("D", [64, 128])
def test_values_behind_a_split(cuda, D):
    """Few rows of many keys, in parts that a second kernel joins."""
    def put(k, v):
        v[0, 6000, 0, 7] = INF   # the first query's own
        v[0, 6002, 1, 9] = NAN
        v[0, 100, 1, 11] = -INF

    prompt(cuda, 5, [6000], [3], D, put, seed=9)


@pytest.mark.parametrize("D", [64, 128])
def test_values_that_keys_weigh_nothing(cuda, D):
    """A key at infinity with a score of -infinity weighs 0: its value's infinities are NaN in the rows that attend it,
    and nothing else of it reaches them."""
    import torch_spyre_amd as tsa

    T, at = 200, 150
    kv, kr, q = randn((1, T, 1, 2 * D), cuda, SEED, 0.5), randn((1, T, 64), cuda, SEED + 1, 0.5), randn((1, T, 1, D + 64), cuda, SEED + 2)
    k, v, ctx = kv[..., :D], kv[..., D:], torch.zeros(1, dtype=torch.int32, device=cuda)
    q[..., 2] = -q[..., 2].abs() - 0.1
    k[0, at, 0, 2] = INF
    keep = keep_of(T, 1, 0, T) & (np.arange(T) != at)
    ref = O.attend(*(torch.cat(x, -1)[0].double().cpu().numpy().reshape(T, -1) for x in ((q,), (k[:, :, 0].nan_to_num(posinf=0), kr), (v,))),
                   keep, (D + 64) ** -0.5)
    v[0, at, 0, 5], v[0, at, 0, 6] = INF, -INF
    out, lse = tsa.latent_attention(q[..., :D], q[..., D:], k, kr, v, ctx, return_lse=True)
    assert out[0, at:, 0, 5:7].isnan().all()
    out[0, at:, 0, 5:7] = torch.from_numpy(ref[0][at:, 5:7]).to(out)
    close(out[0, :, 0], lse[0, :, 0], ref, T, 8.0)


@pytest.mark.parametrize("rank", [256, 512])
@pytest.mark.parametrize("H", [16, 33, 64])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("where", ["latent", "last latent", "rotated"])
def test_own_token_of_a_decode_step(cuda, rank, H, bad, where):
    """It makes the sequence NaN with and without a mask, whatever the score's sign; sequences that have no new token,
    and those beside it, do not notice."""
    import torch_spyre_amd as tsa

    ctx, counts = [0, 63, 64, 100, 2000, 70, 31], [1, 1, 1, 1, 1, 0, 1]
    B, W = len(ctx), 33
    cache = randn((B * W, (rank + 64) // 64, 64, 64), cuda, SEED + H)
    table = torch.randperm(B * W, generator=torch.Generator().manual_seed(SEED)).view(B, W).to(torch.int32).to(cuda)
    q, qr = randn((B, 1, H, rank), cuda, SEED + 1, 0.5), randn((B, 1, H, 64), cuda, SEED + 2)
    lens, new = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (ctx, counts))
    call = lambda mask: tsa.paged_latent_attention(q, qr, cache, table, lens, 0.07, mask, new, max_context_len=2000, return_lse=True)  # noqa: E731
    clean = call(None)
    stick, feature = {"latent": (1, 7), "last latent": (rank // 64 - 1, 63), "rotated": (rank // 64, 13)}[where]
    for b in range(B - 1):  # the last one stays as it is
        cache[table[b, ctx[b] // 64], stick, ctx[b] % 64, feature] = bad
    for mask in (None, torch.ones((1, 1), dtype=torch.bool, device=cuda)):
        out, lse = call(mask)
        assert out[:5].isnan().all() and lse[:5].isnan().all()
        assert torch.equal(out[5:], clean[0][5:]) and torch.equal(lse[5:], clean[1][5:])


RUNS = [(400, [(0, 32)]), (400, [(0, 64)]), (400, [(0, 150)]), (400, [(32, 64)]), (90, [(0, 90)]), (3000, [(0, 600), (900, 1700)])]


@pytest.mark.parametrize("rank", [256, 512])
@pytest.mark.parametrize("T,H", [(1, 16), (1, 64), (3, 8), (7, 32)])
@pytest.mark.parametrize("ctx,runs", RUNS)
def test_runs_that_score_minus_infinity(cuda, rank, T, H, ctx, runs):
    """Runs of tokens whose keys hold infinities (and whose values do not) weigh nothing, wherever a run begins."""
    import torch_spyre_amd as tsa

    W = (ctx + T + 63) // 64
    cache = randn((W, rank // 64 + 1, 64, 64), cuda, SEED + 1)
    table = torch.randperm(W, generator=torch.Generator().manual_seed(SEED)).view(1, W).to(torch.int32).to(cuda)
    q, qr = randn((1, T, H, rank), cuda, SEED + 2, 0.5), randn((1, T, H, 64), cuda, SEED + 3)
    qr[..., 0] = qr[..., 0].abs() + 0.125
    rows = cache[table[0].long()].double().cpu().numpy().transpose(0, 2, 1, 3).reshape(W * 64, -1)[:ctx + T]
    keep = keep_of(T, H, ctx, T)
    for first, end in runs:
        keep[:, first:end] = False
        for t in range(first, end):
            cache[table[0, t // 64], rank // 64, t % 64, 0] = -INF
    out, lse = tsa.paged_latent_attention(q, qr, cache, table, torch.tensor([ctx], dtype=torch.int32, device=cuda), 0.07,
                                          max_context_len=ctx, return_lse=True)
    ref = O.attend(torch.cat((q, qr), -1).double().cpu().numpy().reshape(T * H, -1), rows, rows[:, :rank], keep, 0.07)
    close(out, lse, ref, ctx + T, np.abs(rows).max())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,ctx,runs", [(300, 0, [(0, 40)]), (300, 0, [(64, 128)]), (300, 0, [(100, 290)]), (70, 60, [(0, 125)]),
                                        (2, 3000, [(0, 600), (900, 1700)])])
def test_prompt_runs_that_score_minus_infinity(cuda, D, T, ctx, runs):
    """The same of prompts; rows that attend nothing else are zeros."""
    import torch_spyre_amd as tsa

    n = ctx + T
    kv, kr, q = randn((1, n, 1, 2 * D), cuda, SEED), randn((1, n, 64), cuda, SEED + 1), randn((1, T, 1, D + 64), cuda, SEED + 2)
    q[..., 1] = q[..., 1].abs() + 0.125
    K = torch.cat((kv[:, :, 0, :D], kr), -1)[0].double().cpu().numpy()
    keep = keep_of(T, 1, ctx, T)
    for first, end in runs:
        keep[:, first:end] = False
        kv[0, first:end, 0, 1] = -INF
    out, lse = tsa.latent_attention(q[..., :D], q[..., D:], kv[..., :D], kr, kv[..., D:], torch.tensor([ctx], dtype=torch.int32, device=cuda),
                                    return_lse=True)
    ref = O.attend(q[0, :, 0].double().cpu().numpy(), K, kv[0, :, 0, D:].double().cpu().numpy(), keep, (D + 64) ** -0.5)
    close(out[0, :, 0], lse[0, :, 0], ref, n, 8.0)
