"""GPU: how drafted-token attention shares its pages out -- many sequences,
parts that several workgroups join, sequences of no tokens between long ones,
captured and concurrent calls -- and the 8-bit cache at the ends of its slots."""

import numpy as np
import pytest
import torch

from oracle import serving as OS
from tests.conftest import SEED
from tests.test_quantized_gpu import DTYPE, _randn, numbers, table_of
from tests.test_tree_attention_gpu import check, logical, make_cache, run, scales

pytestmark = pytest.mark.gpu


def lengths(B, low, high, seed):
    """Uneven lengths, some of them 0, one of them `high`."""
    r = np.random.default_rng(SEED + seed)
    n = np.exp(r.uniform(np.log(low), np.log(high), B)).astype(int)
    n[r.random(B) < 0.15] = 0
    n[B // 2] = high
    return [int(x) for x in n]


@pytest.mark.parametrize("kind", ["f16", "int8"])
@pytest.mark.parametrize("B,low,high,T,Hq,Hkv,D", [
    (70, 1, 700, 1, 4, 2, 64),      # more sequences than a wavefront has lanes
    (300, 1, 200, 2, 2, 1, 64),     # more than a wavefront reads at once
    (66, 30, 300, 2, 8, 8, 128),    # half workgroups
    (5, 1, 20000, 2, 4, 1, 64),     # hundreds of parts of few rows
    (5, 1, 9000, 12, 4, 1, 128),    # of up to 64 rows
    (4, 1, 6000, 30, 4, 1, 64),     # of up to 128 rows
    (3, 1, 4000, 50, 8, 1, 128),    # of two row blocks
])
def test_uneven_batches(cuda, kind, B, low, high, T, Hq, Hkv, D):
    r = np.random.default_rng(SEED + B + T)
    counts = [int(x) for x in r.integers(0, T + 1, B)]
    counts[B // 2] = T
    run(cuda, kind, lengths(B, low, high, B + T), T, Hq, Hkv, D, counts, mask=None, seed=1200 + B)


@pytest.mark.parametrize("T", [1, 20, 40])
def test_equal_shares(cuda, T):
    """256 (sequence, KV head)s of nearly one length: none is cut."""
    run(cuda, "e4m3", [200 + (3 * b) % 50 for b in range(32)], T, 8 if T > 1 else 16, 8, 64, mask=None, seed=1300 + T)


def test_many_sequences_decode(cuda):
    """A decode step of more than 64 sequences x 8 KV heads."""
    import torch_spyre_amd as tsa

    ctx = lengths(68, 1, 600, 7)
    W = 10
    cache = make_cache("e4m3", 68 * W, 8, 128, cuda, SEED + 1400)
    table = table_of(68, W, 68 * W, cuda, SEED + 1401)
    q = _randn((68, 16, 128), cuda, SEED + 1402)
    out, lse = tsa.paged_decode_attention(q, cache.k, cache.v, table, torch.tensor(ctx, dtype=torch.int32, device=cuda),
                                          max_context_len=600, return_lse=True, **scales(cache, "e4m3"))
    kl, vl = logical(cache, "e4m3")
    check(out[:, None], lse[:, None], q[:, None], kl, vl, table.cpu().numpy(), ctx, [1] * 68, None, draft_keys=False)


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("T", [2, 20, 40])
def test_joined_parts_in_streams_and_graphs(cuda, kind, T):
    """Parts of few, 80 and 160 rows: two streams at once, and two captured
    calls replayed between each other and eager ones, over changing lengths."""
    import torch_spyre_amd as tsa

    cache = make_cache(kind, 130, 1, 128, cuda, SEED + 1500)
    table = table_of(2, 65, 130, cuda, SEED + 1501)
    lens = torch.tensor([4000, 900], dtype=torch.int32, device=cuda)
    q = [_randn((2, T, 4, 128), cuda, SEED + 1502 + i) for i in range(2)]

    def call(i):
        return tsa.paged_tree_attention(q[i], cache.k, cache.v, table, lens, max_context_len=4000, return_lse=True,
                                        **scales(cache, kind))

    def same(x, y):
        return torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])

    want = [call(0), call(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(same(x, want[i]) for i in range(2) for x in got[i])
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(call(i))
        graphs.append(g)
    for step in range(4):
        q[0].add_(0.125)
        lens.copy_(torch.tensor([4000 - 700 * step, 90 + 800 * step], dtype=torch.int32))
        for i, g in enumerate(graphs):
            g.replay()
            eager = call(i)
            torch.cuda.synchronize()
            assert same(outs[i], eager), (step, i)


def test_slots_at_the_end_of_their_type(cuda):
    """The largest slot, past any table, takes nothing from its neighbours."""
    import torch_spyre_amd as tsa

    T, W = 20, 2
    cache = tsa.QuantizedKVCache(W, 2, 64, DTYPE["int8"], device=cuda)
    table = torch.arange(W, dtype=torch.int32, device=cuda)[None]
    slots = torch.arange(T, dtype=torch.int32)[None] + 30
    slots[0, 0], slots[0, -1] = -1, 2**31 - 1
    k, v = _randn((1, T, 2, 64), cuda, SEED + 1600), _randn((1, T, 2, 64), cuda, SEED + 1601)
    cache.append(k, v, table, slots.to(cuda))
    kn, vn, ks, vs = numbers(cache)
    for x, n, s in ((k, kn, ks), (v, vn, vs)):
        c, sc = OS.quantise(x.cpu().numpy(), "int8")
        assert np.array_equal(n[0, :, 31:49], c[0, 1:19].transpose(1, 0, 2)) and np.array_equal(s[0, :, 31:49], sc[0, 1:19].T)
        assert not n[0, :, 49:].any() and not n[0, :, :31].any() and not n[1].any() and (s[1] == 1).all()


def test_scales_anywhere(cuda):
    """Scales that are contiguous, but not on a 16-byte boundary."""
    import torch_spyre_amd as tsa

    caches = [tsa.QuantizedKVCache(3, 2, 128, DTYPE["e4m3"], device=cuda) for _ in range(2)]
    for i, name in enumerate(("k_scale", "v_scale")):
        setattr(caches[1], name, torch.ones(3 * 2 * 64 + 4, device=cuda)[i + 1:][:3 * 2 * 64].view(3, 2, 64))
    k, v = _randn((1, 150, 2, 128), cuda, SEED + 1700), _randn((1, 150, 2, 128), cuda, SEED + 1701)
    table = torch.arange(3, dtype=torch.int32, device=cuda)[None]
    for c in caches:
        c.append(k, v, table, torch.arange(150, dtype=torch.int32, device=cuda)[None] + 2)
    for x, y in zip(caches[0].tensors, caches[1].tensors):
        assert torch.equal(x.float(), y.float())


def test_rotary_training_step_in_a_graph(cuda):
    """Forward and gradient captured together, replayed between eager ones."""
    import torch_spyre_amd as tsa

    f, amp = tsa.rotary_frequencies(64, scaling="yarn", factor=4.0, device=cuda)
    pos = torch.arange(37, device=cuda)
    q, k, gq, gk = (_randn((2, h, 37, 128), cuda, SEED + 1800 + i) for i, h in enumerate((8, 2, 8, 2)))

    def step():
        a, b = q.detach().requires_grad_(), k.detach().requires_grad_()
        yq, yk = tsa.rotary_embedding(a, b, pos, f, amplitude=amp)
        return (yq.detach(), yk.detach()) + torch.autograd.grad((yq, yk), (a, b), (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        pos.add_(1000)
        q.add_(0.25)
        gk.mul_(-1)
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, step()):
            assert torch.equal(x, y), i


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
@pytest.mark.parametrize("mask", [None, "tree"])
def test_drafts_longer_than_pages(cuda, kind, mask):
    """Drafted tokens over several pages, in ten row blocks."""
    run(cuda, kind, [37, 0, 500], 200, 12, 1, 128, [200, 130, 1], mask=mask, seed=1900)


@pytest.mark.parametrize("kind", ["f16", "int8"])
@pytest.mark.parametrize("Hq,Hkv", [(20, 1), (64, 1), (71, 1), (140, 1), (300, 1), (17, 17)])
def test_many_heads_to_a_kv_head(cuda, kind, Hq, Hkv):
    """One drafted token, but as many rows as any."""
    run(cuda, kind, [700, 64, 0], 1, Hq, Hkv, 64, [1, 1, 0], mask=None, seed=2000)
