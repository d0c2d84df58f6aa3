"""GPU: the 8-bit paged cache -- codes and scales bit for bit, reading back,
the rotation on the way in -- against the definition."""

import numpy as np
import pytest
import torch

from oracle import serving as OS
from tests.conftest import SEED

pytestmark = pytest.mark.gpu
DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _randn(shape, dev, seed):
    return torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).half()


def table_of(B, W, pool, dev, seed):
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed))[:B * W]
    return order.view(B, W).to(torch.int32).to(dev)


def numbers(cache):
    """The codes as the numbers they are, logical pages [P, H, 64, D], and the scales."""
    k, v = OS.pages8_to_logical(cache.k.float().cpu().numpy(), cache.v.float().cpu().numpy())
    return k, v, cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy()


CASES = [  # B, T, Hkv, D, first slot of each sequence
    (1, 1, 1, 64, [0]), (5, 1, 8, 128, [63, 64, 0, 17, 100]), (2, 16, 2, 128, [0, 16]), (2, 16, 2, 64, [48, 5]),
    (3, 50, 3, 64, [0, 33, 7]), (3, 50, 3, 128, [64, 1, 15]), (2, 200, 8, 128, [11, 32]), (1, 129, 5, 64, [63]),
]


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("B,T,Hkv,D,first", CASES)
def test_append_and_read(cuda, codes, B, T, Hkv, D, first):
    """fp16 rows are quantised to the definition's very codes and scales; the
    rest of the cache stays as it was; tokens read back as code * scale."""
    import torch_spyre_amd as tsa

    W = (max(first) + T + 63) // 64 + 1
    cache = tsa.QuantizedKVCache(B * W + 3, Hkv, D, DTYPE[codes], device=cuda)
    cache.k.view(torch.uint8).random_(0, 100)
    cache.v.view(torch.uint8).random_(0, 100)
    table = table_of(B, W, B * W + 3, cuda, SEED)
    k, v = _randn((B, T, Hkv, D), cuda, SEED + 1), _randn((B, T, Hkv, D), cuda, SEED + 2)
    k[:, 0] *= 1000  # rows of other sizes
    v[-1, -1] = 0
    v[0, 0, 0, 3:] = 0
    slots = torch.tensor(first, dtype=torch.int32, device=cuda)[:, None] + torch.arange(T, dtype=torch.int32, device=cuda)
    kn, vn, ksn, vsn = (x.copy() for x in numbers(cache))
    if T == 1:
        cache.append(k[:, 0], v[:, 0], table, slots[:, 0].contiguous())
    else:
        cache.append(k, v, table, slots)
    for x, into, scales in ((k, kn, ksn), (v, vn, vsn)):
        c, s = OS.quantise(x.cpu().numpy(), codes)
        for b in range(B):
            for t in range(T):
                p = first[b] + t
                into[int(table[b, p // 64]), :, p % 64] = c[b, t]
                scales[int(table[b, p // 64]), :, p % 64] = s[b, t]
    for got, want in zip(numbers(cache), (kn, vn, ksn, vsn)):
        assert np.array_equal(got, want)
    lens = slots[:, -1] + 1
    for start, length in ((None, max(first) + T + 2), (torch.tensor(first, dtype=torch.int32, device=cuda), T),
                          (torch.tensor([max(0, f - 3) for f in first], dtype=torch.int32, device=cuda), T + 70)):
        rk, rv = cache.read(table, lens.contiguous(), length, start)
        for got, c, s in ((rk, kn, ksn), (rv, vn, vsn)):
            want = np.zeros((B, Hkv, length, D), dtype=np.float16)
            for b in range(B):
                s0 = 0 if start is None else int(start[b])
                n = min(length, first[b] + T - s0)
                if n > 0:
                    cc = OS.gather(c, table[b].cpu().numpy(), first[b] + T)[:, s0:s0 + n].astype(np.float32)
                    want[b, :, :n] = (cc * OS.gather(s, table[b].cpu().numpy(), first[b] + T)[:, s0:s0 + n, None]).astype(np.float16)
            assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_scattered_slots(cuda, codes):
    """Slots in any order, left and right padding (-1), dropped slots and pages:
    each token lands at its own slot and nothing else is written."""
    import torch_spyre_amd as tsa

    B, T, Hkv, D, W = 4, 40, 3, 128, 3
    cache = tsa.QuantizedKVCache(B * W, Hkv, D, DTYPE[codes], device=cuda)
    table = table_of(B, W, B * W, cuda, SEED + 3)
    table[3, 1] = B * W      # no such page
    table[3, 2] = -1
    k, v = _randn((B, T, Hkv, D), cuda, SEED + 4), _randn((B, T, Hkv, D), cuda, SEED + 5)
    slots = torch.empty((B, T), dtype=torch.int32)
    slots[0] = torch.randperm(64 * W, generator=torch.Generator().manual_seed(SEED))[:T]
    slots[1] = torch.arange(T) - 7            # left padding: -7 .. -1
    slots[1, :7] = -1
    slots[2] = torch.arange(T) + 64 * W - 20  # past the table from token 20 on
    slots[3] = torch.arange(T) + 50           # into a page that is not there
    cache.append(k, v, table, slots.to(cuda))
    kn, vn, ksn, vsn = numbers(cache)
    wk, wv = np.zeros_like(kn), np.zeros_like(vn)
    wks, wvs = np.ones_like(ksn), np.ones_like(vsn)
    for x, into, scales in ((k, wk, wks), (v, wv, wvs)):
        c, s = OS.quantise(x.cpu().numpy(), codes)
        for b in range(B):
            for t in range(T):
                p = int(slots[b, t])
                if 0 <= p < 64 * W and 0 <= int(table[b, p // 64]) < B * W:
                    into[int(table[b, p // 64]), :, p % 64] = c[b, t]
                    scales[int(table[b, p // 64]), :, p % 64] = s[b, t]
    for got, want in ((kn, wk), (vn, wv), (ksn, wks), (vsn, wvs)):
        assert np.array_equal(got, want)
    rk, _ = cache.read(table, torch.full((B,), 64 * W, dtype=torch.int32, device=cuda), 64 * W)
    bad = torch.isnan(rk).any(-1).any(1)
    assert not bad[:3].any() and not bad[3, :64].any() and bad[3, 64:].all()
    _, far = cache.read(table, torch.full((B,), 64 * W + 9, dtype=torch.int32, device=cuda), 64 * W + 20)
    assert torch.isnan(far[0, :, 64 * W:64 * W + 9]).all() and not far[:, :, 64 * W + 9:].any()


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_not_finite(cuda, codes):
    """A row that holds a NaN or an infinity reads back as NaN, its neighbours as ever."""
    import torch_spyre_amd as tsa

    cache = tsa.QuantizedKVCache(1, 2, 64, DTYPE[codes], device=cuda)
    table = torch.zeros((1, 1), dtype=torch.int32, device=cuda)
    x = _randn((1, 20, 2, 64), cuda, SEED + 6)
    x[0, 3, 0, 5], x[0, 9, 1, 0], x[0, 16, 1, 63] = float("nan"), float("inf"), float("-inf")
    x[0, 18, 0] = 65504.0
    cache.append(x, x, table, torch.arange(20, dtype=torch.int32, device=cuda)[None])
    for y in cache.read(table, torch.full((1,), 20, dtype=torch.int32, device=cuda), 20):
        nan = torch.isnan(y[0]).cpu()
        want = torch.zeros((2, 20, 64), dtype=torch.bool)
        want[0, 3] = want[1, 9] = want[1, 16] = True
        assert torch.equal(nan, want)
        assert (y[0, 0, 18] == 65504).all()


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,R,interleaved,amplitude", [
    (3, 1, 8, 2, 128, 128, False, 1.0), (2, 37, 6, 3, 64, 64, True, 1.0), (2, 20, 5, 5, 64, 16, False, 1.3),
    (1, 100, 4, 1, 128, 32, True, 1.0)])
def test_rotary_append(cuda, codes, B, T, Hq, Hkv, D, R, interleaved, amplitude):
    """q as spyre::rotary rotates it; K rotated and quantised without a rounding
    between: every stored value is within half a step of its code (2^-4 of the
    value for e4m3, and half the smallest subnormal, 2^-10 of a scale; half a
    scale for int8) plus the rotation's 8 x 2^-24 of the pair, of the exact
    rotation; V is untouched by it."""
    import torch_spyre_amd as tsa

    cache = tsa.QuantizedKVCache(B * 3, Hkv, D, DTYPE[codes], device=cuda)
    table = table_of(B, 3, B * 3, cuda, SEED + 7)
    packed = _randn((B, T, Hq + 2 * Hkv, D), cuda, SEED + 8)
    q, k, v = packed[:, :, :Hq], packed[:, :, Hq:Hq + Hkv], packed[:, :, Hq + Hkv:]
    slots = (torch.arange(T, device=cuda, dtype=torch.int32) + 11).expand(B, T)
    pos = torch.randint(0, 1 << 17, (B, T), device=cuda, dtype=torch.int64)
    f, _ = tsa.rotary_frequencies(R, device=cuda)
    if T == 1:
        out = cache.rotary_append(q[:, 0], k[:, 0], v[:, 0], table, slots[:, 0].contiguous(), pos[:, 0], f, amplitude, interleaved)
        out = out.unsqueeze(1)
    else:
        out = cache.rotary_append(q, k, v, table, slots, pos, f, amplitude, interleaved)
    assert torch.equal(out, tsa.rotary_embedding(q.transpose(1, 2), None, pos, f, amplitude, interleaved).transpose(1, 2))
    other = tsa.QuantizedKVCache(B * 3, Hkv, D, DTYPE[codes], device=cuda)
    other.append(k, v, table, slots)
    assert torch.equal(other.v.view(torch.uint8), cache.v.view(torch.uint8)) and torch.equal(other.v_scale, cache.v_scale)
    kn, _, ks, _ = numbers(cache)
    x = k.double().cpu().numpy().transpose(0, 2, 1, 3)
    exact = OS.rotate(x, pos.cpu().numpy()[:, None], f.cpu().numpy(), amplitude, interleaved)
    for b in range(B):
        row = table[b].cpu().numpy()
        scale = OS.gather(ks, row, 11 + T)[:, 11:, None].astype(np.float64)
        got = OS.gather(kn, row, 11 + T)[:, 11:] * scale
        fuzz = 8 * 2.0 ** -24 * 2 * amplitude * np.abs(x[b]).max(-1, keepdims=True)
        half = 0.5 * scale if codes == "int8" else 2.0 ** -4 * np.abs(exact[b]) + 2.0 ** -10 * scale
        assert (np.abs(got - exact[b]) <= half * (1 + 2.0 ** -20) + fuzz).all()


def test_streams_and_graph(cuda):
    """Appends and reads follow the current stream; captured ones follow their
    inputs through replays."""
    import torch_spyre_amd as tsa

    cache = tsa.QuantizedKVCache(4, 2, 128, device=cuda)
    table = torch.arange(4, dtype=torch.int32, device=cuda).view(2, 2)
    k, v = _randn((2, 1, 2, 128), cuda, SEED + 9), _randn((2, 1, 2, 128), cuda, SEED + 10)
    slots = torch.zeros((2, 1), dtype=torch.int32, device=cuda)
    lens = torch.zeros((2,), dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append(k, v, table, slots)
        a, _ = cache.read(table, lens + 1, 3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a[:, :, 0], cache.read(table, lens + 1, 1)[0][:, :, 0]) and not a[:, :, 1:].any()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.append(k, v, table, slots)
        rk, rv = cache.read(table, lens, 100)
    for n in (1, 64, 99):
        slots.fill_(n - 1)
        lens.fill_(n)
        k.add_(0.25)
        g.replay()
        torch.cuda.synchronize()
        ek, ev = cache.read(table, lens, 100)
        assert torch.equal(rk, ek) and torch.equal(rv, ev) and rk[:, :, n - 1].any()


def test_empty_and_refusals(cuda):
    import torch_spyre_amd as tsa

    cache = tsa.QuantizedKVCache(4, 2, 128, device=cuda)
    table = torch.arange(4, dtype=torch.int32, device=cuda).view(2, 2)
    k = _randn((2, 3, 2, 128), cuda, SEED + 11)
    slots = torch.zeros((2, 3), dtype=torch.int32, device=cuda) + torch.arange(3, dtype=torch.int32, device=cuda)
    lens = torch.full((2,), 3, dtype=torch.int32, device=cuda)
    f, _ = tsa.rotary_frequencies(128, device=cuda)
    cache.append(k[:0], k[:0], table[:0], slots[:0])
    cache.append(k[:, :0], k[:, :0], table, slots[:, :0])
    assert not cache.k.view(torch.uint8).any()
    assert cache.read(table, lens, 0)[0].shape == (2, 2, 0, 128)
    assert cache.read(table[:0], lens[:0], 5)[0].shape == (0, 2, 5, 128)
    good = dict(k_new=k, v_new=k, k_cache=cache.k, v_cache=cache.v, k_scale=cache.k_scale, v_scale=cache.v_scale,
                block_table=table, slots=slots)
    for change in (dict(k_new=k.float()), dict(v_new=k[:, :2]), dict(k_new=k[..., :64], v_new=k[..., :64]),
                   dict(k_new=k[:, :, :1], v_new=k[:, :, :1]), dict(v_new=k.cpu()), dict(k_cache=cache.k.view(torch.uint8)),
                   dict(v_cache=cache.v.view(torch.int8)), dict(v_cache=cache.k), dict(k_cache=cache.k.transpose(2, 3)),
                   dict(k_scale=cache.k_scale.half()), dict(v_scale=cache.v_scale[:3]), dict(k_scale=cache.k_scale.cpu()),
                   dict(block_table=table.long()), dict(block_table=table[:1]), dict(block_table=table.cpu()),
                   dict(slots=slots.long()), dict(slots=slots[:, :2]), dict(slots=slots.cpu())):
        with pytest.raises((ValueError, TypeError)):
            tsa.kv_append_quantized(**(good | change))
    rot = good | dict(q=k, positions=slots, frequencies=f)
    for change in (dict(q=k[:, :2]), dict(q=k.float()), dict(positions=slots.float()), dict(frequencies=f.float()),
                   dict(frequencies=f[:4]), dict(positions=slots[:, :2])):
        with pytest.raises((ValueError, TypeError)):
            tsa.rotary_kv_append_quantized(**(rot | change))
    for change in (dict(lens=lens.long()), dict(lens=lens[:1]), dict(length=-1), dict(start=lens.long()), dict(start=lens.cpu())):
        args = dict(lens=lens, length=3, start=None) | change
        with pytest.raises((ValueError, TypeError)):
            tsa.kv_read_quantized(*cache.tensors, table, **args)
    with pytest.raises(ValueError):
        tsa.QuantizedKVCache(1, 1, 96, device=cuda)
    with pytest.raises(ValueError):
        tsa.QuantizedKVCache(1, 1, 64, torch.float16, device=cuda)
