"""GPU: attention over the 8-bit cache, and of drafted tokens, where the tokens
with the largest weights add little or nothing to the result: V rows of zeros
(stored with scale 1 whatever the others' are), and of one feature, in every
kernel of it."""

import math

import numpy as np
import pytest
import torch

from oracle import serving as OS
from tests.conftest import SEED
from tests.test_quantized_gpu import table_of
from tests.test_tree_attention_gpu import logical, make_cache, scales

pytestmark = pytest.mark.gpu

# Rows to a KV head: 12 and 16; 40 and 64; 100 and 120; 160 and 300.
SHAPES = [(3, 8, 2, 128), (4, 4, 1, 64), (10, 8, 2, 128), (16, 4, 1, 64), (25, 8, 2, 128), (30, 4, 1, 64),
          (40, 8, 2, 128), (150, 2, 1, 64)]


def put(cache, kind, table, token, k, v):
    """Token `token` of the table's one sequence; k, v [Hkv, D]."""
    if kind == "f16":
        p, t = int(table[0, token // 64]), token % 64
        Hkv, D = k.shape
        cache.k[p, :, :, t] = k.view(Hkv, D // 64, 64)
        cache.v[p, :, :, t] = v
    else:
        cache.append(k[None], v[None], table, torch.tensor([token], dtype=torch.int32, device=k.device))


def check_small(out, lse, q, kl, vl, table, ctx, T, draft_keys=True, headroom=1.0, f16=False):
    """Each row within half a step (2^-11) of its rounding to fp16 and of each
    weight's, and sums, scores and exponentials in fp32 as elsewhere.  Weights
    below fp16's normal range are off by 2^-25 of a unit that is at most
    1 / headroom of the largest weight times V row (rows of zeros count nothing
    there; fp16 pages: of the largest weight, times the largest V).  lse is a sum of up to two numbers below 2^7 and of its logarithm."""
    D = q.shape[-1]
    total = ctx + (T if draft_keys else 0)
    q64, o64, l64 = (x.double().cpu().numpy() for x in (q, out, lse))
    k, v = OS.gather(kl, table[0], total), OS.gather(vl, table[0], total)
    g = q.shape[1] // k.shape[0]
    amax = np.abs(v).max(-1)
    for i in range(T):
        n = ctx + i + 1 if draft_keys else total
        for h in range(q.shape[1]):
            kk, vv = k[h // g, :n], v[h // g, :n]
            score = kk @ q64[i, h] / math.sqrt(D)
            l = np.logaddexp.reduce(score)
            p = np.exp(score - l)
            ref, size = p @ vv, p @ np.abs(vv)
            ds = (D + 4) * 2.0 ** -24 / math.sqrt(D) * (np.abs(kk) @ np.abs(q64[i, h])).max()
            tol = (size * (2 * 2.0 ** -11 + n * 2.0 ** -24 + 2 * ds + 2.0 ** -18)
                   + n * 2.0 ** -25 / headroom * (p.max() * amax[h // g, :n].max() if f16 else (p * amax[h // g, :n]).max())
                   + 2.0 ** -25)
            err = np.abs(o64[i, h] - ref)
            assert (err <= tol).all(), f"row {i} head {h}: worst {(err / tol).max():.1f} of the tolerance, " \
                                       f"result {np.abs(ref).max():.2e}, off by {err.max():.2e}"
            assert abs(l64[i, h] - l) <= ds + n * 2.0 ** -24 + 2.0 ** -17 + 2.0 ** -20 * abs(l)


def queries(T, Hq, D, dev, seed):
    q = torch.randn((1, T, Hq, D), generator=torch.Generator(device=dev).manual_seed(seed), device=dev).half()
    q[..., 0] = 4.0
    return q


def key(Hkv, D, score, dev):
    """A key that every query scores by `score` (as near as fp16 has it)."""
    k = torch.zeros((Hkv, D), dtype=torch.float16, device=dev)
    k[:, 0] = score * math.sqrt(D) / 4
    return k


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("score", [7.0, 11.0, 14.0])
def test_value_rows_of_zeros(cuda, kind, shape, score):
    """Tokens whose V is zero, attended with about 0.7, 0.99 and 0.9995 of a
    row: the first one, one inside (negative zeros), two in one page, one in a
    page of its own, the last of the context, a drafted one."""
    import torch_spyre_amd as tsa

    T, Hq, Hkv, D = shape
    ctx = 2050
    W = (ctx + T + 63) // 64
    cache = make_cache(kind, W, Hkv, D, cuda, SEED + 1)
    table = table_of(1, W, W, cuda, SEED + 2)
    codes = cache.v.view(torch.uint8 if kind == "e4m3" else torch.int8)
    codes.copy_(codes & 0x7f if kind == "e4m3" else codes.abs())  # the others add up, to numbers that fp16 holds
    zero = torch.zeros((Hkv, D), dtype=torch.float16, device=cuda)
    for token in (0, 700, 1025, 1026, 1990, ctx - 1, ctx):
        put(cache, kind, table, token, key(Hkv, D, score, cuda), -zero if token == 700 else zero)
    p, t = int(table[0, 1026 // 64]), 1026 % 64
    assert cache.v_scale[p, 0, t] == 1 and not cache.v[p, :, t // 16, :, t % 16].float().any()
    q = queries(T, Hq, D, cuda, SEED + 3)
    lens = torch.tensor([ctx], dtype=torch.int32, device=cuda)
    kl, vl = logical(cache, kind)
    out, lse = tsa.paged_tree_attention(q, cache.k, cache.v, table, lens, max_context_len=ctx, return_lse=True,
                                        **scales(cache, kind))
    check_small(out[0], lse[0], q[0], kl, vl, table.cpu().numpy(), ctx, T)
    out, lse = tsa.paged_decode_attention(q[:, 0], cache.k, cache.v, table, lens, max_context_len=ctx, return_lse=True,
                                          **scales(cache, kind))
    check_small(out, lse, q[0, :1], kl, vl, table.cpu().numpy(), ctx, 1, draft_keys=False)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("shape", SHAPES[::2])
def test_values_all_zero_or_all_of_scale_one(cuda, kind, shape):
    """A cache whose V is zero gives zeros and the same logsumexp; rows whose
    largest value is the type's (scale 1 as well) are not taken for zeros."""
    import torch_spyre_amd as tsa

    T, Hq, Hkv, D = shape
    ctx = 300
    W = (ctx + T + 63) // 64
    cache = make_cache(kind, W, Hkv, D, cuda, SEED + 4)
    table = table_of(1, W, W, cuda, SEED + 5)
    q = queries(T, Hq, D, cuda, SEED + 6)
    lens = torch.tensor([ctx], dtype=torch.int32, device=cuda)
    top = OS.TOP[kind]
    for token in range(0, ctx + T, 3):
        v = torch.zeros((Hkv, D), dtype=torch.float16, device=cuda)
        v[:, (token * 7) % D] = -top if token % 2 else top
        put(cache, kind, table, token, key(Hkv, D, 0.5, cuda), v)
    kl, vl = logical(cache, kind)
    args = dict(max_context_len=ctx, return_lse=True, **scales(cache, kind))
    out, lse = tsa.paged_tree_attention(q, cache.k, cache.v, table, lens, **args)
    check_small(out[0], lse[0], q[0], kl, vl, table.cpu().numpy(), ctx, T)
    cache.v.view(torch.uint8).zero_()
    cache.v_scale.fill_(1.0)
    nothing, same = tsa.paged_tree_attention(q, cache.k, cache.v, table, lens, **args)
    assert not nothing.any()
    check_small(nothing[0], same[0], q[0], kl, np.zeros_like(vl), table.cpu().numpy(), ctx, T)


@pytest.mark.parametrize("kind", ["f16", "e4m3", "int8"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("ctx,token", [(120, 0), (120, 119), (190, 64), (2050, 1000)])
def test_small_weights_beside_one_that_takes_all(cuda, kind, shape, ctx, token):
    """One token takes nearly all of every row and has V in one feature only
    (fp16: none); what the others add to the rest, with weights of 2^-27 each,
    is there.  The reference of the weights is 2^7 below the largest."""
    import torch_spyre_amd as tsa

    T, Hq, Hkv, D = shape
    W = (ctx + T + 63) // 64
    cache = make_cache(kind, W, Hkv, D, cuda, SEED + 7)
    table = table_of(1, W, W, cuda, SEED + 8)
    if kind == "f16":
        cache.v.abs_().mul_(64)  # results that fp16 holds
    else:
        cache.v_scale.mul_(64)
        codes = cache.v.view(torch.uint8 if kind == "e4m3" else torch.int8)
        codes.copy_(codes & 0x7f if kind == "e4m3" else codes.abs())
    v = torch.zeros((Hkv, D), dtype=torch.float16, device=cuda)
    v[:, D - 1] = 0.0 if kind == "f16" else 128.0
    put(cache, kind, table, token, key(Hkv, D, 18.8, cuda), v)
    q = queries(T, Hq, D, cuda, SEED + 9)
    q[..., 1:] *= 0.0625
    lens = torch.tensor([ctx], dtype=torch.int32, device=cuda)
    kl, vl = logical(cache, kind)
    out, lse = tsa.paged_tree_attention(q, cache.k, cache.v, table, lens, max_context_len=ctx, return_lse=True,
                                        **scales(cache, kind))
    check_small(out[0], lse[0], q[0], kl, vl, table.cpu().numpy(), ctx, T, headroom=2.0 ** 7, f16=kind == "f16")
    assert (out[..., :D - 1] > 0).all()
