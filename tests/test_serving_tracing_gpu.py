"""GPU: the rotary, 8-bit cache and drafted-token ops through the dispatcher's
own checks (schema, autograd registration, fake kernels, traced form), and a
serving step of them compiled as one graph."""

import pytest
import torch

from tests.conftest import SEED
from tests.test_quantized_gpu import _randn, table_of

pytestmark = pytest.mark.gpu


def cases(dev):
    import torch_spyre_amd as tsa

    B, T, Hq, Hkv, D = 2, 5, 4, 2, 64
    cache = tsa.QuantizedKVCache(8, Hkv, D, torch.int8, device=dev)  # (compared elementwise: int8 has equality)
    f16 = tsa.PagedKVCache(8, Hkv, D, device=dev)
    table = table_of(B, 4, 8, dev, SEED)
    q, k, v = (_randn((B, T, h, D), dev, SEED + 1 + h) for h in (Hq, Hkv, Hkv))
    pos = torch.arange(T, dtype=torch.int32, device=dev).expand(B, T).contiguous() + 100
    lens = torch.tensor([100, 64], dtype=torch.int32, device=dev)
    f, _ = tsa.rotary_frequencies(D, device=dev)
    long = torch.arange(105, dtype=torch.int32, device=dev).expand(B, 105).contiguous()
    cache.append(_randn((B, 105, Hkv, D), dev, SEED + 9), _randn((B, 105, Hkv, D), dev, SEED + 10), table, long)
    f16.k.normal_()
    f16.v.normal_()
    mask = torch.ones((T, T), dtype=torch.bool, device=dev).tril()
    ops = torch.ops.spyre
    qh, kh = q.transpose(1, 2), k.transpose(1, 2)
    grads = [x.detach().clone().requires_grad_() for x in (qh, kh)]
    return {
        "rotary": (ops.rotary, (qh, kh, pos, f, 1.1, True)),
        "rotary, q alone": (ops.rotary, (qh, None, pos[0], f)),
        "rotary, gradients": (ops.rotary, (*grads, pos, f)),
        "kv_quant_append": (ops.kv_quant_append, (k, v, *cache.tensors, table, pos)),
        "rotary_kv_quant_append": (ops.rotary_kv_quant_append, (q, k, v, *cache.tensors, table, pos, pos, f)),
        "kv_quant_read": (ops.kv_quant_read, (*cache.tensors, table, lens, 20, lens - 15)),
        "quant_paged_decode_attention": (ops.quant_paged_decode_attention,
                                         (q[:, 0].contiguous(), *cache.tensors, table, lens, None, 100)),
        "paged_tree_attention": (ops.paged_tree_attention,
                                 (q, f16.k, f16.v, table, lens, mask, None, None, None, None, 100)),
        "paged_tree_attention, 8-bit": (ops.paged_tree_attention,
                                        (q, cache.k, cache.v, table, lens, None, lens // 25, cache.k_scale,
                                         cache.v_scale, 0.1, 100)),
    }


NAMES = ["rotary", "rotary, q alone", "rotary, gradients", "kv_quant_append", "rotary_kv_quant_append", "kv_quant_read",
         "quant_paged_decode_attention", "paged_tree_attention", "paged_tree_attention, 8-bit"]


@pytest.mark.parametrize("name", NAMES)
def test_opcheck(cuda, name):
    op, args = cases(cuda)[name]
    torch.library.opcheck(op, args)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_compiled_step(cuda, dtype):
    """torch.compile(fullgraph=True) of a step: q and k rotated, K and V
    quantised into the cache, a tree of drafts and a decode step attended, the
    new tokens read back.  Equal to the eager step bit for bit, caches too."""
    import torch_spyre_amd as tsa

    B, T, Hq, Hkv, D = 3, 6, 8, 2, 128
    f, amp = tsa.rotary_frequencies(D, scaling="llama3", factor=8.0, device=cuda)
    table = table_of(B, 5, 15, cuda, SEED + 20)
    ctx = torch.tensor([200, 3, 127], dtype=torch.int32, device=cuda)
    packed = _randn((B, T, Hq + 2 * Hkv, D), cuda, SEED + 21)
    past = [_randn((B, 200, Hkv, D), cuda, SEED + 22 + i) for i in range(2)]

    def step(x, k, v, ks, vs):
        q, kn, vn = x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]
        slots = ctx[:, None] + torch.arange(T, dtype=torch.int32, device=x.device)
        q = torch.ops.spyre.rotary_kv_quant_append(q, kn, vn, k, v, ks, vs, table, slots, slots, f, amp)
        out, lse = torch.ops.spyre.paged_tree_attention(q, k, v, table, ctx, None, None, ks, vs, None, 200)
        one, _ = torch.ops.spyre.quant_paged_decode_attention(q[:, 0], k, v, ks, vs, table, ctx + 1, None, 201)
        rk, rv = torch.ops.spyre.kv_quant_read(k, v, ks, vs, table, ctx + T, T, ctx)
        return q, out, lse, one, rk, rv

    results = []
    for fn in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
        cache = tsa.QuantizedKVCache(15, Hkv, D, dtype, device=cuda)
        cache.append(*past, table, torch.arange(200, dtype=torch.int32, device=cuda).expand(B, 200))
        out = fn(packed, *cache.tensors)
        results.append([x.clone() for x in out] + [cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale])
    for x, y in zip(*results):
        assert torch.equal(x, y)
