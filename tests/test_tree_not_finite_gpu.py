"""GPU: NaN and infinities in the cache under every kernel of drafted-token
attention: in tokens that rows do not attend they reach nothing, in those that
rows do attend (drafted, or in whole pages of the context) they give what the
definition gives."""

import numpy as np
import pytest
import torch

from oracle import serving as OS
from tests.conftest import SEED
from tests.test_quantized_gpu import table_of
from tests.test_tree_attention_gpu import KINDS, check, logical, make_cache, scales, tree

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")

# Rows to a KV head, g = 2: 12, 40, 80, 200 (16, 64, 128, 512 at most to a kernel).
TOKENS = [6, 20, 40, 100]


def attend(cuda, kind, T, D, ctx, poke, counts=None, seed=0):
    """Random pages with `poke`(cache, table, tokens of b) applied, checked
    against the definition; infinities have to be those of the definition too."""
    import torch_spyre_amd as tsa

    B, Hq, Hkv = len(ctx), 4, 2
    n = counts if counts is not None else [T] * B
    W = (max(ctx) + T + 70) // 64 + 1
    cache = make_cache(kind, B * W + 1, Hkv, D, cuda, SEED + seed)
    table = table_of(B, W, B * W + 1, cuda, SEED + seed + 1)
    m = tree(B, T, SEED + seed + 2)
    poke(cache, lambda b, t: (int(table[b, t // 64]), t % 64), m)
    q = torch.randn((B, T, Hq, D), generator=torch.Generator(device=cuda).manual_seed(SEED + seed + 3), device=cuda).half()
    out, lse = tsa.paged_tree_attention(
        q, cache.k, cache.v, table, torch.tensor(ctx, dtype=torch.int32, device=cuda), torch.from_numpy(m).to(cuda),
        draft_lens=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=cuda),
        max_context_len=max(ctx), return_lse=True, **scales(cache, kind))
    kl, vl = logical(cache, kind)
    rows = table.cpu().numpy()
    check(out, lse, q, kl, vl, rows, ctx, n, m)
    o = out.double().cpu().numpy()
    for b in range(B):
        with np.errstate(all="ignore"):
            ref, _, _ = OS.attend(q[b].double().cpu().numpy(), OS.gather(kl, rows[b], ctx[b] + n[b]),
                                  OS.gather(vl, rows[b], ctx[b] + n[b]), OS.tree_keep(ctx[b], n[b], T, m[b]))
        assert np.array_equal(np.isinf(ref), np.isinf(o[b])) and np.array_equal(ref[np.isinf(ref)], o[b][np.isinf(ref)])
    return out


def poke_v(cache, kind, at, value, heads=slice(None), feature=7):
    """V of a token: one feature (fp16), the codes (e4m3, NaN only) or the scale."""
    p, t = at
    if kind == "f16":
        cache.v[p, heads, feature, t] = value
    elif kind == "e4m3" and value != value:
        cache.v.view(torch.uint8)[p, heads, t // 16, feature, t % 16] = 0x7f
    else:
        cache.v_scale[p, heads, t] = value


def poke_k(cache, kind, at, value, heads=slice(None)):
    p, t = at
    if kind == "f16":
        cache.k[p, heads, 0, t, 5] = value
    elif kind == "e4m3" and value != value:
        cache.k.view(torch.uint8)[p, heads, 0, t, 5] = 0x7f
    else:
        cache.k_scale[p, heads, t] = value


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", TOKENS)
def test_drafted_tokens_that_some_rows_attend(cuda, kind, D, T):
    """K and V of drafted tokens that only their descendants attend, and
    everything behind the drafts."""
    ctx = [75, 20, 128]

    def poke(cache, at, m):
        for b, c in enumerate(ctx):
            first = next(j for j in range(1, T) if not m[b, T - 1, j])  # not attended by the last row
            last = max(j for j in range(T) if not m[b, T - 1, j])
            poke_v(cache, kind, at(b, c + first), NAN, slice(0, 1))
            poke_v(cache, kind, at(b, c + last), INF, slice(1, 2))
            poke_k(cache, kind, at(b, c + last), NAN, slice(0, 1))
            poke_k(cache, kind, at(b, c + first), INF if kind == "f16" else NAN, slice(1, 2))
            for t in range(c + T, c + T + 70, 3):
                poke_v(cache, kind, at(b, t), NAN if t % 2 else INF)
                poke_k(cache, kind, at(b, t), INF if t % 2 else NAN)
                if kind != "f16":
                    cache.v_scale[at(b, t)[0], :, at(b, t)[1]] = INF if t % 2 else NAN

    out = attend(cuda, kind, T, D, ctx, poke, seed=100)
    assert torch.isfinite(out[:, T - 1]).all() and not torch.isfinite(out).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", TOKENS)
def test_rows_behind_the_drafts(cuda, kind, D, T):
    """Rows and tokens from a sequence's draft count on: zeros, whatever the
    slots hold; one sequence has no drafts and NaN in all of its context."""
    ctx, counts = [100, 64, 200], [T - 1, 0, 1]

    def poke(cache, at, m):
        for b, (c, n) in enumerate(zip(ctx, counts)):
            for t in range(0 if n == 0 else c + n, c + T + 5):
                poke_v(cache, kind, at(b, t), NAN)
                poke_k(cache, kind, at(b, t), NAN)

    out = attend(cuda, kind, T, D, ctx, poke, counts, seed=200)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("value", [NAN, INF])
def test_values_in_whole_pages_of_the_context(cuda, kind, D, T, value):
    """V of tokens that every row attends, in the first, an inner and the last
    whole page: NaN and infinities in the features concerned, no others."""
    ctx = [640, 333]

    def poke(cache, at, m):
        for t in (3, 200, 639):
            poke_v(cache, kind, at(0, t), value, slice(0, 1), feature=t % D)
        poke_v(cache, kind, at(1, 130), value, slice(1, 2), feature=11)
        if kind != "f16" and value == INF:  # its codes without a zero: infinities, not NaN
            p, t = at(1, 130)
            cache.v.view(torch.uint8)[p, 1, t // 16, :, t % 16] = 3
            cache.v.view(torch.uint8)[p, 1, t // 16, 9, t % 16] = 0x83

    out = attend(cuda, kind, T, D, ctx, poke, seed=300)
    assert torch.isfinite(out[0, :, 2:]).all() and torch.isfinite(out[1, :, :2]).all()
    if kind == "f16":
        assert int((~torch.isfinite(out[1])).any(0).sum()) == 2  # one feature of two heads


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", TOKENS)
def test_keys_in_whole_pages_of_the_context(cuda, kind, D, T):
    """A NaN key that every row attends makes the rows of its KV head NaN."""
    def poke(cache, at, m):
        poke_k(cache, kind, at(0, 70), NAN, slice(0, 1))

    out = attend(cuda, kind, T, D, [500, 500], poke, seed=400)
    assert torch.isnan(out[0, :, :2]).all() and torch.isfinite(out[0, :, 2:]).all() and torch.isfinite(out[1]).all()
