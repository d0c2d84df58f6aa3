"""GPU: caches, rows and results whose offsets pass 32 bits: what lies there is,
bit for bit, what a small call gives."""

import pytest
import torch

from tests.conftest import SEED
from tests.test_quantized_gpu import DTYPE, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def freed():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", ["f16", "int8"])
def test_far_pages(cuda, kind):
    """Appending to, reading and attending pages more than 4 GiB into the cache."""
    import torch_spyre_amd as tsa

    Hkv, D, W, ctx = 8, 128, 4, 130
    caches, tables = [], []
    for P in (2 * W, (70000 if kind != "f16" else 36000)):
        caches.append(tsa.PagedKVCache(P, Hkv, D, device=cuda) if kind == "f16" else
                      tsa.QuantizedKVCache(P, Hkv, D, DTYPE[kind], device=cuda))
        order = torch.tensor([[3, 0, 6, 1], [2, 7, 5, 4]], dtype=torch.int32, device=cuda)
        tables.append(order + (P - 2 * W))
    assert caches[1].k.numel() * caches[1].k.element_size() > 2**32
    k, v = _randn((2, ctx + 40, Hkv, D), cuda, SEED + 1900), _randn((2, ctx + 40, Hkv, D), cuda, SEED + 1901)
    slots = torch.arange(ctx + 40, dtype=torch.int32, device=cuda).expand(2, -1).contiguous()
    lens = torch.full((2,), ctx, dtype=torch.int32, device=cuda)
    results = []
    for c, t in zip(caches, tables):
        out = []
        if kind == "f16":
            for i in range(ctx + 40):
                tsa.kv_append(k[:, i].contiguous(), v[:, i].contiguous(), c.k, c.v, t, slots[:, i].contiguous())
            args = {}
        else:
            c.append(k, v, t, slots)
            out += c.read(t, torch.full_like(lens, ctx + 40), 200)
            args = dict(k_scale=c.k_scale, v_scale=c.v_scale)
            out.append(tsa.paged_decode_attention(_randn((2, 16, D), cuda, SEED + 1902), c.k, c.v, t, lens,
                                                  max_context_len=ctx, **args))
        for T in (1, 10, 25, 40):  # every kernel
            out.append(tsa.paged_tree_attention(_randn((2, T, 32, D), cuda, SEED + 1903), c.k, c.v, t, lens,
                                                max_context_len=ctx, **args))
        results.append(out)
    assert all(torch.equal(a, b) and torch.isfinite(a).all() and a.abs().sum() > 0 for a, b in zip(*results))


def test_far_rows_read(cuda):
    """The last rows of a result of more than 2^31 numbers."""
    import torch_spyre_amd as tsa

    Hkv, D, L = 8, 128, 2_200_000
    cache = tsa.QuantizedKVCache(3, Hkv, D, DTYPE["e4m3"], device=cuda)
    cache.append(_randn((1, 192, Hkv, D), cuda, SEED + 1910), _randn((1, 192, Hkv, D), cuda, SEED + 1911),
                 torch.arange(3, dtype=torch.int32, device=cuda)[None], torch.arange(192, dtype=torch.int32, device=cuda)[None])
    table = (torch.arange(-(-L // 64), device=cuda) % 3).to(torch.int32)[None]
    k, v = cache.read(table, torch.tensor([L - 5], dtype=torch.int32, device=cuda), L)
    first = (L // 64 - 2) * 64
    sk, sv = cache.read(table[:, first // 64:].contiguous(), torch.tensor([L - 5 - first], dtype=torch.int32, device=cuda), L - first)
    assert k.numel() > 2**31
    for big, small in ((k, sk), (v, sv)):
        assert torch.equal(big[:, :, first:], small) and small[:, :, :-5].abs().sum() > 0 and not small[:, :, -5:].any()


def test_far_rows_rotated(cuda):
    import torch_spyre_amd as tsa

    S, H, D = 8_500_000, 2, 128
    f, _ = tsa.rotary_frequencies(D, device=cuda)
    q = torch.zeros((1, S, H, D), dtype=torch.float16, device=cuda)
    assert q.numel() > 2**31
    tail = _randn((1, 9, H, D), cuda, SEED + 1920)
    q[:, -9:] = tail
    pos = torch.arange(S, dtype=torch.int32, device=cuda)
    y = tsa.rotary_embedding(q.transpose(1, 2), None, pos, f)
    assert torch.equal(y[:, :, -9:], tsa.rotary_embedding(tail.transpose(1, 2), None, pos[-9:], f))
    assert not y[:, :, :4096].any()
