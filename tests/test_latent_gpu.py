"""GPU: the paged latent cache and both forms of its attention, against 64 bits.

Tolerances: out rounds to fp16 (half a step: 2^-11 of it, 2^-25 below the normal
range), the weights round to fp16 before the second product (2^-11 of sum w |v|, and
2^-32 of |v| a key for weights far below the largest), sums and exponentials are fp32
(2^-20 of sum w |v| covers 2^4 roundings of partial sums), and scores are sums of fp32
products in steps of 16 or 32: at most 48 roundings of 2^-23 (an MFMA may truncate) of
sum |q| |k| scale, delta, which moves a weight by 2 delta of itself.  The logsumexp is off
by delta, 2^-20 for its sum and 2^-22 of itself."""

import math

import numpy as np
import pytest
import torch

from oracle import step as O
from tests.conftest import SEED

pytestmark = pytest.mark.gpu


def randn(shape, dev, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).half()


def table_of(B, W, pool, dev, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pool, generator=g)[:B * W].view(B, W).to(torch.int32).to(dev)


def rows_of(cache):
    """Logical rows [pages, 64, rank + 64] in 64 bits."""
    c = cache.double().cpu().numpy()
    return c.transpose(0, 2, 1, 3).reshape(c.shape[0], 64, -1)


def close(out, lse, ref, n_keys, v_top):
    want, wl, size, reach = ref
    delta = 48 * 2.0 ** -23 * reach
    got, gl = out.double().cpu().numpy().reshape(want.shape), lse.double().cpu().numpy().reshape(wl.shape)
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (2.0 ** -11 + 2.0 ** -20 + 2 * delta)[:, None] * size + 2.0 ** -32 * n_keys * v_top
    nan = np.isnan(wl)
    assert np.array_equal(np.isnan(gl), nan)
    assert np.isnan(got[nan]).all()
    assert np.array_equal(np.isneginf(gl), np.isneginf(wl)), "rows that attend nothing"
    assert not got[np.isneginf(wl)].any()
    err = np.abs(got - want)[~nan]
    assert (err <= tol[~nan]).all(), f"off by {np.max(err - tol[~nan]):.3e} more than {np.max(tol[~nan]):.3e}"
    fine = np.isfinite(wl)
    assert (np.abs(gl - wl)[fine] <= (delta + 2.0 ** -20 + 2.0 ** -22 * np.abs(wl))[fine]).all()


def keep_of(T, H, ctx, n, mask=None):
    """[T H, ctx + n]"""
    k = np.zeros((T, ctx + n), dtype=bool)
    m = np.tril(np.ones((T, T), dtype=bool)) if mask is None else np.asarray(mask)
    k[:n, :ctx], k[:n, ctx:] = True, m[:n, :n]
    return np.repeat(k, H, 0)


def check_paged(out, lse, q, qr, cache, table, ctx, counts, scale, mask=None):
    rank = q.shape[-1]
    rows, T, H = rows_of(cache), q.shape[1], q.shape[2]
    Q = np.concatenate((q.double().cpu().numpy(), qr.double().cpu().numpy()), -1)
    for b in range(q.shape[0]):
        total = ctx[b] + counts[b]
        k = rows[table[b, :max(1, -(-total // 64))].cpu().numpy()].reshape(-1, rank + 64)[:total]
        m = None if mask is None else mask[b if mask.shape[0] > 1 else 0]
        ref = O.attend(Q[b].reshape(T * H, -1), k, k[:, :rank], keep_of(T, H, ctx[b], counts[b], m), scale)
        close(out[b], lse[b], ref, total, np.abs(k).max() if total else 0.0)


def paged(dev, B, T, H, rank, ctx, counts=None, mask=None, seed=0, scale=0.07, change=None, **kw):
    import torch_spyre_amd as tsa

    n = [T] * B if counts is None else counts
    W = max(1, max(-(-(c + x) // 64) for c, x in zip(ctx, n)))
    cache = randn((B * W + 3, (rank + 64) // 64, 64, 64), dev, SEED + seed)
    table = table_of(B, W, B * W + 3, dev, SEED + seed + 1)
    q, qr = randn((B, T, H, rank), dev, SEED + seed + 2, 0.5), randn((B, T, H, 64), dev, SEED + seed + 3)
    if change:
        change(cache, table, q, qr)
    lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
    dl = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev)
    out, lse = tsa.paged_latent_attention(q, qr, cache, table, lens, scale, mask, dl, max_context_len=max(ctx), return_lse=True, **kw)
    check_paged(out, lse, q, qr, cache, table, ctx, n, scale, None if mask is None else mask.view(-1, T, T).cpu().numpy())
    return out, lse


# ---------------------------------------------------------------- the cache --

@pytest.mark.parametrize("rank", [256, 512])
@pytest.mark.parametrize("n", [1, 7, 64, 513])
def test_append(cuda, rank, n):
    import torch_spyre_amd as tsa

    P = -(-n // 64) + 2
    packed = randn((n, rank + 64 + 8), cuda, SEED + n)  # one projection's output
    latent, rope = packed[:, :rank], packed[:, rank:rank + 64]
    slots = torch.randperm(P * 64, generator=torch.Generator().manual_seed(SEED))[:n].to(cuda)
    slots[0] = -1
    if n > 6:
        slots[3], slots[5] = P * 64, 2**40
    cache = randn((P, (rank + 64) // 64, 64, 64), cuda, SEED + 1)
    want = rows_of(cache).reshape(P * 64, -1)
    for s, row in zip(slots.tolist(), packed[:, :rank + 64].double().cpu().numpy()):
        if 0 <= s < P * 64:
            want[s] = row
    tsa.latent_append(latent, rope, cache, slots)
    assert np.array_equal(rows_of(cache).reshape(P * 64, -1), want)


def test_append_shapes(cuda):
    """[B, T, ...] rows, strides and alignments that are copied first, no rows."""
    import torch_spyre_amd as tsa

    B, T, rank = 3, 5, 256
    slots = torch.arange(B * T, device=cuda).view(B, T) * 3
    for latent in (randn((B, T, rank), cuda, SEED), randn((B, T, rank + 1), cuda, SEED)[..., 1:], randn((T, B, rank), cuda, SEED).transpose(0, 1),
                   randn((B, T, 2 * rank), cuda, SEED)[..., ::2]):
        cache = torch.zeros((2, 5, 64, 64), dtype=torch.float16, device=cuda)
        rope = randn((B, T, 64), cuda, SEED + 1)
        tsa.latent_append(latent, rope, cache, slots)
        got = rows_of(cache).reshape(128, -1)
        assert np.array_equal(got[slots.flatten().cpu().numpy(), :rank].reshape(B, T, rank), latent.double().cpu().numpy())
        assert np.array_equal(got[slots.flatten().cpu().numpy(), rank:].reshape(B, T, 64), rope.double().cpu().numpy())
        assert np.count_nonzero(got) == np.count_nonzero(got[slots.flatten().cpu().numpy()])
    tsa.latent_append(latent[:, :0], rope[:, :0], cache, slots[:, :0])
    tsa.latent_append(latent, rope, cache[:0], slots)


@pytest.mark.parametrize("rank", [256, 512])
def test_read(cuda, rank):
    import torch_spyre_amd as tsa

    B, W, L = 3, 3, 150
    cache = tsa.LatentKVCache(B * W, rank, device=cuda)
    cache.pages.copy_(randn(cache.pages.shape, cuda, SEED))
    table = table_of(B, W, B * W, cuda, SEED + 1)
    table[2, 1] = B * W  # no such page
    lens = torch.tensor([150, 0, 140], dtype=torch.int32, device=cuda)
    rows = rows_of(cache.pages)
    for start in (None, torch.tensor([10, 0, 60], dtype=torch.int32, device=cuda)):
        c, r = cache.read(table, lens, L, start)
        assert c.shape == (B, L, rank) and r.shape == (B, L, 64)
        for b in range(B):
            first = 0 if start is None else int(start[b])
            want = np.zeros((L, rank + 64))
            for i in range(L):
                t = first + i
                if t < int(lens[b]):
                    page = int(table[b, t // 64])
                    want[i] = rows[page, t % 64] if page < B * W else np.nan
            got = np.concatenate((c[b].double().cpu().numpy(), r[b].double().cpu().numpy()), -1)
            assert np.array_equal(got, want, equal_nan=True)
    c, r = cache.read(table, lens, 0)
    assert c.shape == (B, 0, rank) and r.shape == (B, 0, 64)


# ------------------------------------------------------------ over the cache --

@pytest.mark.parametrize("rank", [256, 512])
@pytest.mark.parametrize("H", [1, 16, 20, 32, 33, 64, 128])
@pytest.mark.parametrize("ctx", [[0], [1, 62, 63, 64], [130, 700], [2500]])
def test_decode(cuda, rank, H, ctx):
    paged(cuda, len(ctx), 1, H, rank, ctx, seed=H)


@pytest.mark.parametrize("rank", [256, 512])
@pytest.mark.parametrize("T,H", [(2, 16), (5, 20), (7, 32), (3, 128), (70, 4)])
@pytest.mark.parametrize("kind", ["chain", "tree", "one tree", "ragged"])
def test_drafts(cuda, rank, T, H, kind):
    ctx = [0, 61, 128, 333]
    rng = np.random.default_rng(SEED + T)
    mask = counts = None
    if "tree" in kind:
        m = rng.random((1 if kind == "one tree" else 4, T, T)) < 0.5
        m[:, 1] = False  # a row that attends its context only (or nothing)
        mask = torch.from_numpy(m).to(cuda)
    if kind == "ragged":
        counts = [T, 0, 1, T - 1]
    paged(cuda, 4, T, H, rank, ctx, counts, mask if kind != "one tree" else mask[0], seed=T)


@pytest.mark.parametrize("B,H,ctx", [(64, 16, 900), (40, 64, 300), (9, 128, 3000), (300, 8, 70)])
def test_batches(cuda, B, H, ctx):
    """Ragged batches: sequences whole, in parts, several to a workgroup.  (A few rows of each are checked.)"""
    import torch_spyre_amd as tsa

    rng = np.random.default_rng(SEED + B)
    lens = rng.integers(0, ctx + 1, B)
    lens[0], lens[-1] = ctx, 0
    W = -(-(ctx + 1) // 64)
    rank = 512
    cache = randn((B * W, 9, 64, 64), cuda, SEED + B)
    table = table_of(B, W, B * W, cuda, SEED + 1)
    q, qr = randn((B, 1, H, rank), cuda, SEED + 2, 0.5), randn((B, 1, H, 64), cuda, SEED + 3)
    out, lse = tsa.paged_latent_attention(q, qr, cache, table, torch.tensor(lens, dtype=torch.int32, device=cuda), 0.07,
                                          return_lse=True)
    some = sorted({0, H // 2, H - 1})
    check_paged(out[:, :, some], lse[:, :, some], q[:, :, some], qr[:, :, some], cache, table, lens.tolist(), [1] * B, 0.07)


@pytest.mark.parametrize("counts", [[1, 7, 0, 3], [0, 0, 0, 7], [7, 7, 7, 7]])
@pytest.mark.parametrize("rank", [256, 512])
def test_rows_of_uneven_drafts_and_parts(cuda, rank, counts):
    """Row blocks without rows between others that several ranges share."""
    paged(cuda, 4, 7, 33, rank, [4000, 130, 700, 1], counts=counts, seed=70)


def test_one_token_operands(cuda):
    import torch_spyre_amd as tsa

    cache, table = randn((4, 9, 64, 64), cuda, SEED), torch.tensor([[2, 0]], dtype=torch.int32, device=cuda)
    q, qr = randn((1, 16, 512), cuda, SEED + 1), randn((1, 16, 64), cuda, SEED + 2)
    ctx = torch.tensor([70], dtype=torch.int32, device=cuda)
    a = tsa.paged_latent_attention(q, qr, cache, table, ctx, 0.05)
    b, lse = tsa.paged_latent_attention(q[:, None], qr[:, None], cache, table, ctx, 0.05, return_lse=True)
    assert a.shape == q.shape and torch.equal(a, b[:, 0]) and lse.shape == (1, 1, 16)


def test_strides(cuda):
    """q as a product batched over heads leaves it, views of wider rows, copies of odd ones."""
    import torch_spyre_amd as tsa

    B, T, H, rank = 2, 3, 5, 256
    cache, table = randn((6, 5, 64, 64), cuda, SEED), table_of(B, 3, 6, cuda, SEED)
    ctx = torch.tensor([100, 5], dtype=torch.int32, device=cuda)
    q, qr = randn((H, B, T, rank), cuda, SEED + 1).permute(1, 2, 0, 3), randn((B, T, H, 192), cuda, SEED + 2)[..., 128:]
    want = tsa.paged_latent_attention(q.contiguous(), qr.contiguous(), cache, table, ctx, 0.1)
    odd = torch.zeros((B, T, H, rank + 3), dtype=torch.float16, device=cuda)
    odd[..., 3:] = q
    wide = torch.zeros((B, 8), dtype=torch.int32, device=cuda)
    wide[:, 2:5] = table
    for x in (q, odd[..., 3:]):
        assert torch.equal(tsa.paged_latent_attention(x, qr, cache, wide[:, 2:5], ctx, 0.1), want)


def test_large_scores(cuda):
    """Scores of hundreds: one key takes all; the reference moves page after page."""
    paged(cuda, 1, 2, 32, 512, [900], seed=5, scale=0.2, change=lambda c, t, q, qr: q.mul_(40))


def test_rising_scores(cuda):
    """Later pages with larger scores: the reference moves many times."""
    def change(cache, table, q, qr):
        for p, page in enumerate(table[0].tolist()):
            cache[page] *= 0.02 * (p + 1)

    for H in (16, 64):
        paged(cuda, 1, 1, H, 512, [1500], seed=6, scale=1.0, change=change)


@pytest.mark.parametrize("rank", [256, 512])
@pytest.mark.parametrize("H", [16, 64])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_not_attended_is_not_reached(cuda, rank, H, bad):
    """NaN and infinities in drafts that a row does not attend, and behind the last token, do not reach it."""
    import torch_spyre_amd as tsa

    ctx, T = [60, 5], 6
    m = np.tril(np.ones((T, T), dtype=bool))
    m[:, 2] = False
    m[4, 2] = True  # only row 4 attends draft 2
    mask = torch.from_numpy(m).to(cuda)
    cache, table = randn((5, rank // 64 + 1, 64, 64), cuda, SEED), torch.tensor([[3, 1], [0, 4]], dtype=torch.int32, device=cuda)
    q, qr = randn((2, T, H, rank), cuda, SEED + 1, 0.5), randn((2, T, H, 64), cuda, SEED + 2)
    lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    clean = tsa.paged_latent_attention(q, qr, cache, table, lens, 0.07, mask, return_lse=True)
    for b in range(2):
        t = ctx[b] + 2
        cache[table[b, t // 64], 1, t % 64, 5] = bad
        t = ctx[b] + T
        cache[table[b, t // 64], :, t % 64:] = bad
    cache[2] = bad
    out, lse = tsa.paged_latent_attention(q, qr, cache, table, lens, 0.07, mask, return_lse=True)
    rows = [0, 1, 2, 3, 5]
    assert torch.equal(out[:, rows], clean[0][:, rows]) and torch.equal(lse[:, rows], clean[1][:, rows])
    assert out[:, 4].isnan().all() and lse[:, 4].isnan().all()


def test_nan_in_the_context_reaches_every_row(cuda):
    import torch_spyre_amd as tsa

    cache, table = randn((4, 9, 64, 64), cuda, SEED), torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device=cuda)
    cache[2, 8, 10, 3] = float("nan")
    q, qr = randn((2, 2, 20, 512), cuda, SEED + 1), randn((2, 2, 20, 64), cuda, SEED + 2)
    out, lse = tsa.paged_latent_attention(q, qr, cache, table, torch.tensor([100, 100], dtype=torch.int32, device=cuda), 0.05,
                                          return_lse=True)
    assert out[0].isnan().all() and lse[0].isnan().all() and out[1].isfinite().all() and lse[1].isfinite().all()


def test_bad_pages_and_long_contexts_are_nan(cuda):
    import torch_spyre_amd as tsa

    cache = randn((4, 9, 64, 64), cuda, SEED)
    table = torch.tensor([[2, 0], [1, 4], [3, -1], [0, 1], [1, 2]], dtype=torch.int32, device=cuda)
    ctx = torch.tensor([100, 100, 64, 64, 110], dtype=torch.int32, device=cuda)
    counts = torch.tensor([1, 1, 1, 0, 1], dtype=torch.int32, device=cuda)
    q, qr = randn((5, 1, 16, 512), cuda, SEED + 1), randn((5, 1, 16, 64), cuda, SEED + 2)
    out, lse = tsa.paged_latent_attention(q, qr, cache, table, ctx, 0.05, draft_lens=counts, max_context_len=100, return_lse=True)
    assert out[0].isfinite().all() and out[1].isnan().all() and out[2].isnan().all() and lse[1:3].isnan().all()
    assert not out[3].any() and (lse[3] == -math.inf).all()
    assert out[4].isnan().all()


def test_query_not_finite(cuda):
    """A query with a NaN makes its own row NaN, no other."""
    import torch_spyre_amd as tsa

    cache, table = randn((4, 9, 64, 64), cuda, SEED), torch.tensor([[2, 0]], dtype=torch.int32, device=cuda)
    q, qr = randn((1, 1, 33, 512), cuda, SEED + 1), randn((1, 1, 33, 64), cuda, SEED + 2)
    ctx = torch.tensor([100], dtype=torch.int32, device=cuda)
    clean = tsa.paged_latent_attention(q, qr, cache, table, ctx, 0.05)
    q[0, 0, 7, 300] = float("nan")
    out = tsa.paged_latent_attention(q, qr, cache, table, ctx, 0.05)
    keep = [h for h in range(33) if h != 7]
    assert out[0, 0, 7].isnan().all() and torch.equal(out[0, 0, keep], clean[0, 0, keep])


# ------------------------------------------------------------------ expanded --

def expanded(dev, B, T, H, D, ctx, counts=None, keys=None, seed=0, change=None):
    import torch_spyre_amd as tsa

    n = [T] * B if counts is None else counts
    L = max(c + x for c, x in zip(ctx, n)) if keys is None else keys
    kv = randn((B, L, H, 2 * D), dev, SEED + seed)
    k, v, kr = kv[..., :D], kv[..., D:], randn((B, L, 64), dev, SEED + seed + 1)
    q = randn((B, T, H, D + 64), dev, SEED + seed + 2)
    if change:
        change(k, v, kr, q)
    lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
    nl = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev)
    out, lse = tsa.latent_attention(q[..., :D], q[..., D:], k, kr, v, lens, nl, return_lse=True)
    Q, K, V, R = (x.double().cpu().numpy() for x in (q, k, v, kr))
    for b in range(B):
        total = ctx[b] + n[b]
        keep = keep_of(T, 1, ctx[b], n[b])
        for h in sorted({0, H // 2, H - 1}):
            ref = O.attend(Q[b, :, h], np.concatenate((K[b, :total, h], R[b, :total]), -1), V[b, :total, h], keep, (D + 64) ** -0.5)
            close(out[b, :, h], lse[b, :, h], ref, total, np.abs(V[b]).max() if total else 0.0)
    return out, lse


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 2, 31, 64, 65, 127, 300])
@pytest.mark.parametrize("ctx", [[0], [1, 64], [63, 500]])
def test_prompts(cuda, D, T, ctx):
    expanded(cuda, len(ctx), T, 3, D, ctx, seed=T)


@pytest.mark.parametrize("D", [64, 128])
def test_ragged_prompts(cuda, D):
    expanded(cuda, 5, 270, 9, D, [0, 100, 0, 64, 7], [270, 0, 1, 129, 64], seed=3)


@pytest.mark.parametrize("D", [64, 128])
def test_few_rows_of_many_keys(cuda, D):
    """Split over the keys, one split of the short sequence is empty."""
    expanded(cuda, 2, 2, 2, D, [6000, 3], counts=[2, 1], seed=60)
    expanded(cuda, 1, 1, 1, D, [9000], seed=61)


def test_many_heads(cuda):
    expanded(cuda, 2, 40, 64, 128, [30, 200], seed=4)


def test_long_chunk(cuda):
    expanded(cuda, 1, 600, 2, 128, [3000], seed=5)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_not_attended_keys_are_not_reached(cuda, D, bad):
    """Keys and values from a position on that some rows attend; rows before it do not notice."""
    import torch_spyre_amd as tsa

    B, T, H = 2, 300, 2
    kv, kr, q = randn((B, T + 80, H, 2 * D), cuda, SEED), randn((B, T + 80, 64), cuda, SEED + 1), randn((B, T, H, D + 64), cuda, SEED + 2)
    ctx = torch.tensor([0, 70], dtype=torch.int32, device=cuda)
    call = lambda: tsa.latent_attention(q[..., :D], q[..., D:], kv[..., :D], kr, kv[..., D:], ctx, return_lse=True)  # noqa: E731
    clean = call()
    kv[0, T:], kr[0, T:] = bad, bad     # behind the last key
    kv[1, T + 70:], kr[1, T + 70:] = bad, bad
    for a, b in zip(call(), clean):
        assert torch.equal(a, b)
    for x, key in ((kv[0, 200, 1, 3:4], True), (kv[0, 200, 1, D + 5:D + 6], False)):  # a key's, a value's feature
        old = x.clone()
        x.fill_(bad)
        out, lse = call()
        assert torch.equal(out[0, :200], clean[0][0, :200]) and torch.equal(out[1], clean[0][1]) and torch.equal(out[0, :, 0], clean[0][0, :, 0])
        # A key at infinity has a score of q x inf: where that is -inf its weight is exp(-inf) = 0, so
        # the row is what it is without the key; +inf and NaN make it NaN, as a value does.
        reached = torch.full((T - 200,), True, device=cuda)
        if key and not math.isnan(bad):
            reached = (q[0, 200:, 1, 3] > 0) == (bad > 0)
        assert (out[0, 200:, 1].isfinite().all(-1) == ~reached).all()
        if key:
            assert (lse[0, 200:, 1].isfinite() == ~reached).all()
            K = torch.cat((kv[0, :T, 1, :D], kr[0, :T]), -1).double().cpu().numpy()
            keep = keep_of(T, 1, 0, T) & (np.arange(T) != 200)
            rows = [200 + r for r in torch.nonzero(~reached).flatten().tolist()]
            ref = O.attend(q[0, rows, 1].double().cpu().numpy(), K, kv[0, :T, 1, D:].double().cpu().numpy(), keep[rows], (D + 64) ** -0.5)
            close(out[0, rows, 1], lse[0, rows, 1], ref, T, float(kv[0, :T, 1, D:].abs().max()))
        x.copy_(old)


def test_too_few_keys_are_nan(cuda):
    import torch_spyre_amd as tsa

    k, kr, q = randn((3, 50, 2, 64), cuda, SEED), randn((3, 50, 64), cuda, SEED + 1), randn((3, 20, 2, 128), cuda, SEED + 2)
    out, lse = tsa.latent_attention(q[..., :64], q[..., 64:], k, kr, k, torch.tensor([30, 31, 60], dtype=torch.int32, device=cuda),
                                    return_lse=True)
    assert out[0].isfinite().all() and out[1:].isnan().all() and lse[1:].isnan().all()
    none = tsa.latent_attention(q[..., :64], q[..., 64:], k[:, :0], kr[:, :0], k[:, :0], torch.zeros(3, dtype=torch.int32, device=cuda),
                                torch.zeros(3, dtype=torch.int32, device=cuda))
    assert none.shape == (3, 20, 2, 64) and not none.any()


@pytest.mark.parametrize("H", [16, 33])
def test_one_token_that_its_mask_leaves_out(cuda, H):
    """A decode step's own token, masked, holds NaN: the row attends its context alone."""
    import torch_spyre_amd as tsa

    cache, table = randn((6, 5, 64, 64), cuda, SEED + 80), torch.tensor([[2, 0], [4, 1]], dtype=torch.int32, device=cuda)
    ctx = torch.tensor([70, 0], dtype=torch.int32, device=cuda)
    cache[0, :, 70 - 64] = float("nan")
    cache[4, :, 0] = float("inf")
    q, qr = randn((2, 1, H, 256), cuda, SEED + 81), randn((2, 1, H, 64), cuda, SEED + 82)
    mask = torch.zeros((1, 1), dtype=torch.bool, device=cuda)
    out, lse = tsa.paged_latent_attention(q, qr, cache, table, ctx, 0.05, mask, max_context_len=70, return_lse=True)
    clean = cache.clone()
    clean[0, :, 70 - 64] = clean[4, :, 0] = 0
    check_paged(out, lse, q, qr, clean, table, [70, 0], [1, 1], 0.05, mask.view(1, 1, 1).cpu().numpy())
