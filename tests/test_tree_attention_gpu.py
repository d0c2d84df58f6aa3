"""GPU: attention of drafted tokens over the paged cache (fp16 and 8-bit), and
decode over the 8-bit cache, against the fp64 definition on the values that the
cache holds."""

import math

import numpy as np
import pytest
import torch

from oracle import attention as OA
from oracle import serving as OS
from tests.conftest import SEED
from tests.test_quantized_gpu import DTYPE, numbers, table_of

pytestmark = pytest.mark.gpu


def make_cache(kind, pool, Hkv, D, dev, seed, spread=0.5):
    """A full pool of random pages; V rows of uneven sizes."""
    import torch_spyre_amd as tsa

    g = torch.Generator(device=dev).manual_seed(seed)
    k = torch.randn((pool, Hkv, 64, D), generator=g, device=dev).half()
    v = torch.randn((pool, Hkv, 64, D), generator=g, device=dev)
    v = (v * torch.exp(spread * torch.randn((pool, Hkv, 64, 1), generator=g, device=dev))).clamp(-60000, 60000).half()
    if kind == "f16":
        return tsa.PagedKVCache.from_pages(k, v)
    cache = tsa.QuantizedKVCache(pool, Hkv, D, DTYPE[kind], device=dev)
    table = torch.arange(pool, dtype=torch.int32, device=dev)[:, None]
    slots = torch.arange(64, dtype=torch.int32, device=dev).expand(pool, 64)
    cache.append(k.transpose(1, 2), v.transpose(1, 2), table, slots)
    return cache


def logical(cache, kind):
    """fp64 pages [P, H, 64, D] of what the cache stands for."""
    if kind == "f16":
        k, v = OA.pages_to_logical(cache.k.cpu().numpy(), cache.v.cpu().numpy(), cache.num_pages, cache.Hkv, cache.D)
        return k.astype(np.float64), v.astype(np.float64)
    k, v, ks, vs = numbers(cache)
    with np.errstate(invalid="ignore"):
        return k * ks[..., None].astype(np.float64), v * vs[..., None].astype(np.float64)


def scales(cache, kind):
    return {} if kind == "f16" else {"k_scale": cache.k_scale, "v_scale": cache.v_scale}


def tree(B, T, seed):
    """A random tree for each sequence: token i and its ancestors."""
    r = np.random.default_rng(seed)
    m = np.zeros((B, T, T), dtype=bool)
    for b in range(B):
        for i in range(T):
            p = int(r.integers(-1, i)) if i else -1
            if p >= 0:
                m[b, i] = m[b, p]
            m[b, i, i] = True
    return m


def check(out, lse, q, kl, vl, table, ctx, counts, mask, scale=None, draft_keys=True):
    """A row's error against fp64: its weights round to fp16 (2^-11 each, as does
    the output, so 2^-10 of the weighted mean of |v|, `size`), or below fp16's
    normal range by 2^-25 of the largest weight's |v|, n times; scores are off by
    (D + 4) 2^-24 of scale * sum |q k|, which also moves lse, and sums over n
    keys by n 2^-24."""
    B, T, Hq, D = q.shape
    q64 = q.double().cpu().numpy()
    o64, l64 = out.double().cpu().numpy(), lse.double().cpu().numpy()
    s = abs(1 / math.sqrt(D) if scale is None else scale)
    for b in range(B):
        n = counts[b]
        total = ctx[b] + (n if draft_keys else 0)
        k, v = OS.gather(kl, table[b], total), OS.gather(vl, table[b], total)
        if draft_keys:
            keep = OS.tree_keep(ctx[b], n, T, None if mask is None else mask[b] if mask.ndim == 3 else mask)
        else:
            keep = np.zeros((T, total), dtype=bool)
            keep[:n] = True
        ref, rl, size = OS.attend(q64[b], k, v, keep, scale)
        assert np.array_equal(np.isfinite(rl), np.isfinite(l64[b])), "rows that attend nothing"
        if total == 0:
            assert not o64[b].any()
            continue
        fin = np.isfinite(k).all() and np.isfinite(v).all()
        kk, vv = (np.where(np.isfinite(x), x, 0) for x in (k, v))
        g = Hq // k.shape[0]
        ds = (D + 4) * 2.0 ** -24 * s * (np.abs(q64[b]).reshape(T, -1, g, D).transpose(1, 0, 2, 3).reshape(k.shape[0], -1, D)
                                        @ np.abs(kk).transpose(0, 2, 1)).max()
        tol = size * (2.0 ** -10 + total * 2.0 ** -24 + 2 * ds + 2.0 ** -18) + total * 2.0 ** -25 * np.abs(vv).max() + 2.0 ** -24
        if not fin:
            assert np.array_equal(np.isnan(ref), np.isnan(o64[b]))
        ok = np.isfinite(ref)
        with np.errstate(invalid="ignore"):
            err, errl = np.abs(o64[b] - ref), np.abs(l64[b] - rl)
        assert (err[ok] <= tol[ok]).all(), f"b {b}: worst {np.nanmax(err[ok] / tol[ok]):.2f} of the tolerance"
        okl = np.isfinite(rl)
        assert (errl[okl] <= (ds + total * 2.0 ** -24 + 2.0 ** -20 * (4 + np.abs(rl)))[okl]).all()
        assert not o64[b][~np.isfinite(rl) & ~np.isnan(rl)].any()


def run(cuda, kind, ctx, T, Hq, Hkv, D, counts=None, mask="tree", scale=None, seed=0, spread=0.5, poke=None, shared=False):
    import torch_spyre_amd as tsa

    B = len(ctx)
    n = counts if counts is not None else [T] * B
    W = max((c + m + 63) // 64 for c, m in zip(ctx, n)) or 1
    cache = make_cache(kind, B * W + 1, Hkv, D, cuda, SEED + seed, spread)
    table = table_of(B, W, B * W + 1, cuda, SEED + seed + 1)
    m = None if mask is None else tree(B, T, SEED + seed + 2) if isinstance(mask, str) else mask
    if shared:
        m = m[0]
    if poke is not None:
        poke(cache, table, m)
    q = torch.randn((B, T, Hq, D), generator=torch.Generator(device=cuda).manual_seed(SEED + seed + 3), device=cuda).half()
    out, lse = tsa.paged_tree_attention(
        q, cache.k, cache.v, table, torch.tensor(ctx, dtype=torch.int32, device=cuda),
        None if m is None else torch.from_numpy(m).to(cuda),
        draft_lens=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=cuda), scale=scale,
        max_context_len=max(ctx), return_lse=True, **scales(cache, kind))
    assert out.shape == q.shape and out.is_contiguous() and lse.shape == (B, T, Hq)
    kl, vl = logical(cache, kind)
    check(out, lse, q, kl, vl, table.cpu().numpy(), ctx, n, m, scale)
    return out


KINDS = ["f16", "e4m3", "int8"]
CASES = [  # contexts, T, Hq, Hkv, D, counts
    ([0], 1, 1, 1, 64, None),
    ([1], 1, 4, 1, 128, None),
    ([0, 5, 63], 7, 8, 2, 64, None),
    ([64, 65, 31, 32], 5, 8, 8, 128, [5, 0, 1, 3]),
    ([100, 0, 127], 33, 4, 4, 64, [33, 2, 20]),
    ([300, 1000, 0], 16, 16, 2, 128, None),
    ([2500], 3, 32, 8, 128, None),
    ([700, 90], 65, 12, 2, 128, [65, 40]),
    ([190], 70, 40, 8, 64, None),
    ([1500, 20], 64, 64, 8, 128, None),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_tree(cuda, kind, case):
    ctx, T, Hq, Hkv, D, counts = CASES[case]
    run(cuda, kind, ctx, T, Hq, Hkv, D, counts, seed=10 * case)


@pytest.mark.parametrize("kind", KINDS)
def test_chain_shared_mask_and_scale(cuda, kind):
    run(cuda, kind, [130, 3], 9, 8, 2, 128, mask=None, seed=200)
    run(cuda, kind, [130, 3], 9, 8, 2, 64, [9, 4], shared=True, seed=210)
    run(cuda, kind, [130, 3], 9, 8, 2, 128, scale=-0.3, seed=220)
    run(cuda, kind, [130, 3], 9, 8, 2, 64, scale=0.0, seed=230)


@pytest.mark.parametrize("kind", KINDS)
def test_masks_that_leave_nothing(cuda, kind):
    """No context and a mask with empty rows: zeros and -inf; rows that attend
    a later token only; any pattern is taken as it is."""
    r = np.random.default_rng(SEED)
    m = r.random((3, 40, 40)) < 0.2
    m[0, 5] = m[1] = False
    m[2, 0] = np.arange(40) == 39
    run(cuda, kind, [0, 0, 0], 40, 4, 2, 64, mask=m, seed=300)
    run(cuda, kind, [0, 70, 33], 40, 4, 2, 128, [40, 40, 11], mask=m, seed=310)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [6, 40])
def test_not_finite_where_not_attended(cuda, kind, T):
    """NaN and infinities in slots behind the drafts and in drafted tokens:
    only rows that attend them notice, and only in the features concerned."""
    ctx, Hkv, D = [75, 20], 2, 64

    def poke(cache, table, m):
        for b, c in enumerate(ctx):
            for at, (value, heads) in {c + 1: (float("nan"), slice(0, 1)), c + T - 1: (float("inf"), slice(1, 2)),
                                       c + T: (float("nan"), slice(None)), c + T + 5: (float("inf"), slice(None))}.items():
                if at // 64 >= table.shape[1]:
                    continue
                p, t = int(table[b, at // 64]), at % 64
                if kind == "f16":
                    cache.v[p, heads, 7, t] = value
                    cache.k[p, heads, 0, t, 3 if at >= c + T else 5] = value if at >= c + T else 1.0
                else:
                    cache.v_scale[p, heads, t] = value
                    if kind == "e4m3":
                        cache.v.view(torch.uint8)[p, heads, t // 16, :, t % 16] = 0x7f
                    if at >= c + T:
                        cache.k_scale[p, heads, t] = value

    run(cuda, kind, ctx, T, 4, Hkv, D, seed=400, poke=poke)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_uneven_scales(cuda, kind):
    """V rows whose sizes differ by 2^20 and more: each row's result is exact
    relative to what it attends."""
    run(cuda, kind, [400], 5, 8, 2, 128, spread=4.0, seed=500)
    run(cuda, kind, [400], 5, 8, 2, 64, spread=4.0, seed=510)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("ctx,Hq,Hkv,D", [
    ([1], 8, 8, 64), ([700], 32, 8, 128), ([0, 1, 64, 65, 4000], 16, 2, 64), ([4096] * 4, 32, 8, 128), ([9000, 33], 64, 8, 128)])
def test_decode(cuda, kind, ctx, Hq, Hkv, D):
    import torch_spyre_amd as tsa

    B, W = len(ctx), (max(ctx) + 63) // 64
    cache = make_cache(kind, B * W + 1, Hkv, D, cuda, SEED + 600)
    table = table_of(B, W, B * W + 1, cuda, SEED + 601)
    q = torch.randn((B, Hq, D), generator=torch.Generator(device=cuda).manual_seed(SEED + 602), device=cuda).half()
    lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    out, lse = tsa.paged_decode_attention(q, cache.k, cache.v, table, lens, return_lse=True, **scales(cache, kind))
    kl, vl = logical(cache, kind)
    check(out[:, None], lse[:, None], q[:, None], kl, vl, table.cpu().numpy(), ctx, [1] * B, None, draft_keys=False)
    again = tsa.paged_decode_attention(q, cache.k, cache.v, table, lens, max_context_len=max(ctx), **scales(cache, kind))
    assert torch.equal(out, again)


def test_f16_agrees_with_decode(cuda):
    """One drafted token over fp16 pages is a decode step over the context and
    itself: both round as `check` says, against the same exact values."""
    import torch_spyre_amd as tsa

    ctx = [64, 1000, 0]
    cache = make_cache("f16", 60, 8, 128, cuda, SEED + 700)
    table = table_of(3, 17, 60, cuda, SEED + 701)
    q = torch.randn((3, 1, 32, 128), generator=torch.Generator(device=cuda).manual_seed(SEED + 702), device=cuda).half()
    lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    out, lse = tsa.paged_tree_attention(q, cache.k, cache.v, table, lens, return_lse=True)
    ref, rl = tsa.paged_decode_attention(q[:, 0].contiguous(), cache.k, cache.v, table, lens + 1, return_lse=True)
    kl, vl = logical(cache, "f16")
    for o, l in ((out, lse), (ref[:, None], rl[:, None])):
        check(o, l, q, kl, vl, table.cpu().numpy(), ctx, [1] * 3, None)


def test_bad_pages_and_contexts(cuda):
    """A page outside the pool, tokens past the table and a context above
    max_context_len give NaN for that sequence, never a fault; the others are as ever."""
    import torch_spyre_amd as tsa

    for kind in KINDS:
        cache = make_cache(kind, 20, 2, 64, cuda, SEED + 800)
        table = table_of(4, 4, 20, cuda, SEED + 801)
        q = torch.randn((4, 5, 4, 64), generator=torch.Generator(device=cuda).manual_seed(SEED + 802), device=cuda).half()
        lens = torch.tensor([100, 100, 100, 100], dtype=torch.int32, device=cuda)
        good = tsa.paged_tree_attention(q, cache.k, cache.v, table, lens, max_context_len=256, **scales(cache, kind))
        assert torch.isfinite(good).all()
        wrong = table.clone()
        wrong[1, 1] = 20
        wrong[2, 0] = -5
        far = lens.clone()
        far[3] = 254  # drafts past the table's 256 tokens
        out = tsa.paged_tree_attention(q, cache.k, cache.v, wrong, far, max_context_len=256, **scales(cache, kind))
        assert torch.equal(out[0], good[0]) and torch.isnan(out[1:]).all()
        out = tsa.paged_tree_attention(q, cache.k, cache.v, table, far, max_context_len=100, **scales(cache, kind))
        assert torch.equal(out[:3], good[:3]) and torch.isnan(out[3]).all()
        neg = lens.clone()
        neg[0] = -3
        out = tsa.paged_tree_attention(q, cache.k, cache.v, table, neg, max_context_len=100, **scales(cache, kind))
        assert torch.equal(out[1:], good[1:]) and torch.isfinite(out).all()


def test_strided_operands(cuda):
    """q as a slice of a packed projection, a transposed mask, a table cut from a wider one."""
    import torch_spyre_amd as tsa

    cache = make_cache("e4m3", 20, 2, 128, cuda, SEED + 900)
    big = table_of(2, 9, 20, cuda, SEED + 901)
    packed = torch.randn((2, 12, 12, 128), generator=torch.Generator(device=cuda).manual_seed(SEED + 902), device=cuda).half()
    q = packed[:, :, 2:10]
    m = torch.from_numpy(tree(2, 12, SEED + 903)).to(cuda)
    lens = torch.tensor([300, 17], dtype=torch.int32, device=cuda)
    args = dict(max_context_len=300, **scales(cache, "e4m3"))
    want = tsa.paged_tree_attention(q.contiguous(), cache.k, cache.v, big[:, :6].contiguous(), lens, m, **args)
    mt = m.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(tsa.paged_tree_attention(q, cache.k, cache.v, big[:, :6], lens, mt, **args), want)
    odd = torch.empty(q.numel() + 1, dtype=torch.float16, device=cuda)[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(tsa.paged_tree_attention(odd, cache.k, cache.v, big[:, :6], lens, m, **args), want)
    assert torch.equal(tsa.paged_tree_attention(q, cache.k, cache.v, big[:, :6], lens, m[:1].expand(2, 12, 12), **args)[0], want[0])


@pytest.mark.parametrize("kind", ["f16", "int8"])
def test_streams_and_graphs(cuda, kind):
    """Two streams at once, and two captured calls replayed between each other
    and eager ones: every result is the eager call's."""
    import torch_spyre_amd as tsa

    ctx = [2500, 100]
    cache = make_cache(kind, 90, 2, 128, cuda, SEED + 1000)
    table = table_of(2, 40, 90, cuda, SEED + 1001)
    lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    q = [torch.randn((2, 9, 8, 128), generator=torch.Generator(device=cuda).manual_seed(SEED + 1002 + i), device=cuda).half()
         for i in range(2)]

    def call(i):
        return tsa.paged_tree_attention(q[i], cache.k, cache.v, table, lens, max_context_len=2500, **scales(cache, kind))

    want = [call(0), call(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(i))
        graphs.append(g)
    for step in range(4):
        q[0].add_(0.125)
        lens.sub_(37)
        for g in graphs:
            g.replay()
        eager = [call(0), call(1)]
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], eager[i]) for i in range(2)), step


def test_refusals(cuda):
    import torch_spyre_amd as tsa

    f16, e4m3 = make_cache("f16", 4, 2, 64, cuda, SEED + 1100), make_cache("e4m3", 4, 2, 64, cuda, SEED + 1101)
    table = torch.arange(4, dtype=torch.int32, device=cuda).view(2, 2)
    lens = torch.tensor([10, 20], dtype=torch.int32, device=cuda)
    q = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device=cuda)
    m = torch.ones((3, 3), dtype=torch.bool, device=cuda)
    good = dict(q=q, k_cache=f16.k, v_cache=f16.v, block_table=table, context_lens=lens, tree_mask=m)
    eight = good | dict(k_cache=e4m3.k, v_cache=e4m3.v, **scales(e4m3, "e4m3"))
    for base, change in [
        (good, dict(q=q.float())), (good, dict(q=q[0])), (good, dict(q=q[..., :32])), (good, dict(q=q[:, :, :3])),
        (good, dict(k_cache=f16.k.float())), (good, dict(v_cache=f16.v[:3])), (good, dict(k_cache=e4m3.k, v_cache=e4m3.v)),
        (good, dict(k_scale=e4m3.k_scale)), (good, dict(block_table=table.long())), (good, dict(block_table=table[:1])),
        (good, dict(context_lens=lens.long())), (good, dict(context_lens=lens[:1])), (good, dict(context_lens=lens.cpu())),
        (good, dict(tree_mask=m.float())), (good, dict(tree_mask=m[:2])), (good, dict(tree_mask=m.expand(3, 3, 3))),
        (good, dict(tree_mask=m.cpu())), (good, dict(draft_lens=lens.long())), (good, dict(max_context_len=129)),
        (good, dict(k_cache=f16.k.cpu())), (eight, dict(v_scale=None)), (eight, dict(k_scale=e4m3.k_scale[:2])),
        (eight, dict(v_cache=e4m3.v.view(torch.int8))), (eight, dict(k_cache=f16.k)),
    ]:
        with pytest.raises((ValueError, TypeError)):
            tsa.paged_tree_attention(**(base | change))
    with pytest.raises(ValueError):
        tsa.paged_decode_attention(q[:, 0], e4m3.k, e4m3.v, table, lens, k_scale=e4m3.k_scale)
    with pytest.raises(ValueError):
        tsa.paged_decode_attention(q[:, 0], e4m3.k, e4m3.v, table, lens, out=q[:, 0], **scales(e4m3, "e4m3"))
    assert tsa.paged_tree_attention(q[:0], f16.k, f16.v, table[:0], lens[:0]).shape == (0, 3, 4, 64)
    assert tsa.paged_tree_attention(q[:, :0], f16.k, f16.v, table, lens).shape == (2, 0, 4, 64)
