"""GPU: the serving operators together, as a step of a server uses them: a
prompt in two chunks through the 8-bit cache and SDPA, a tree of drafted tokens
behind it, the accepted ones kept, a decode step after them."""

import math

import numpy as np
import pytest
import torch

from oracle import serving as OS
from tests.conftest import SEED
from tests.test_quantized_gpu import DTYPE, table_of
from tests.test_tree_attention_gpu import check, logical, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_prompt_drafts_decode(cuda, kind):
    import torch_spyre_amd as tsa

    B, Hq, Hkv, D, T = 2, 8, 2, 128, 13
    prompt, chunk = [150, 97], 70  # the first `chunk` tokens, then the rest
    cache = tsa.QuantizedKVCache(B * 4 + 2, Hkv, D, DTYPE[kind], device=cuda)
    table = table_of(B, 4, B * 4 + 2, cuda, SEED)
    freq, amp = tsa.rotary_frequencies(D, scaling="yarn", factor=4.0, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(SEED + 1)
    i32 = dict(dtype=torch.int32, device=cuda)

    def new(n):
        x = torch.randn((B, n, Hq + 2 * Hkv, D), generator=g, device=cuda).half()
        return x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]

    # the prompts, right-padded to the longer one in the second chunk
    done = torch.zeros((B,), **i32)
    for n in (chunk, max(prompt) - chunk):
        q, k, v = new(n)
        t = done[:, None] + torch.arange(n, **i32)
        slots = torch.where(t < torch.tensor(prompt, **i32)[:, None], t, torch.full_like(t, -1))
        q = cache.rotary_append(q, k, v, table, slots, t, freq, amp)
        lens = torch.minimum(done + n, torch.tensor(prompt, **i32))
        length = int(lens.max())
        dk, dv = cache.read(table, lens, length)
        at = torch.arange(length, device=cuda)
        mask = (at <= t[:, :, None]) & (at < lens[:, None, None])
        out = tsa.scaled_dot_product_attention(q.transpose(1, 2), dk, dv, attn_mask=mask[:, None], enable_gqa=True)
        kl, vl = logical(cache, kind)
        for b in range(B):
            real = int((slots[b] >= 0).sum())
            keys, values = (OS.gather(x, table[b].cpu().numpy(), int(lens[b])) for x in (kl, vl))
            keep = mask[b, :real, :int(lens[b])].cpu().numpy()
            ref, _, _ = OS.attend(q[b, :real].double().cpu().numpy(), keys, values, keep)
            # dense K / V add one rounding of each value (2^-11) to the operator's own 1e-2 relative
            err = np.abs(out[b, :, :real].transpose(0, 1).double().cpu().numpy() - ref)
            assert (err <= 2e-3 + 1e-2 * np.abs(ref)).all()
        done = done + n
    ctx = torch.tensor(prompt, **i32)

    # a tree of drafts behind each prompt, at the positions of their depths
    m = tree(B, T, SEED + 2)
    depth = torch.from_numpy(m.sum(-1).astype(np.int32) - 1).to(cuda)
    q, k, v = new(T)
    slots = ctx[:, None] + torch.arange(T, **i32)
    q = cache.rotary_append(q, k, v, table, slots, ctx[:, None] + depth, freq, amp)
    args = dict(k_scale=cache.k_scale, v_scale=cache.v_scale)
    out, lse = tsa.paged_tree_attention(q, cache.k, cache.v, table, ctx, torch.from_numpy(m).to(cuda),
                                        max_context_len=max(prompt), return_lse=True, **args)
    kl, vl = logical(cache, kind)
    check(out, lse, q, kl, vl, table.cpu().numpy(), prompt, [T] * B, m)

    # the deepest path of each is accepted: its tokens move to the front, the
    # rest are forgotten; a row quantised again has the same codes
    before = cache.read(table, ctx + T, T, ctx)
    keep = torch.full((B, T), -1, **i32)
    n = []
    for b in range(B):
        leaf = int(m[b].sum(-1).argmax())
        path = np.flatnonzero(m[b, leaf])
        keep[b, torch.from_numpy(path).to(cuda)] = ctx[b] + torch.arange(len(path), **i32)
        n.append(len(path))
    cache.rotary_append(q, k, v, table, keep, ctx[:, None] + depth, freq, amp)
    after = cache.read(table, ctx + T, T, ctx)
    for b in range(B):
        path = torch.from_numpy(np.flatnonzero(m[b, int(m[b].sum(-1).argmax())])).to(cuda)
        for x, y in zip(before, after):
            assert torch.equal(y[b, :, :n[b]], x[b][:, path])
    ctx = ctx + torch.tensor(n, **i32)

    # a decode step
    q, k, v = (x[:, 0] for x in new(1))
    q = cache.rotary_append(q, k, v, table, ctx, ctx, freq, amp)
    out, lse = tsa.paged_decode_attention(q, cache.k, cache.v, table, ctx + 1, return_lse=True, **args)
    kl, vl = logical(cache, kind)
    lens = [int(x) + 1 for x in ctx]
    check(out[:, None], lse[:, None], q[:, None], kl, vl, table.cpu().numpy(), lens, [1] * B, None, draft_keys=False)
    assert math.isfinite(float(lse.sum()))


def test_f16_cache_with_drafts(cuda):
    """The fp16 cache: tokens appended one by one by kv_append, then attended as a line of drafts."""
    import torch_spyre_amd as tsa

    B, Hq, Hkv, D, T = 3, 8, 4, 64, 5
    ctx = [0, 61, 64]
    g = torch.Generator(device=cuda).manual_seed(SEED + 3)
    cache = tsa.PagedKVCache(10, Hkv, D, device=cuda)
    table = table_of(B, 2, 10, cuda, SEED + 4)
    for t in range(max(ctx) + T):
        k, v = (torch.randn((B, Hkv, D), generator=g, device=cuda).half() for _ in range(2))
        pos = torch.tensor([t if t < c + T else -1 for c in ctx], dtype=torch.int32, device=cuda)
        tsa.kv_append(k, v, cache.k, cache.v, table, pos)
    q = torch.randn((B, T, Hq, D), generator=g, device=cuda).half()
    f, a = tsa.rotary_frequencies(D, device=cuda)
    lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    pos = lens[:, None] + torch.arange(T, dtype=torch.int32, device=cuda)
    q = tsa.rotary_embedding(q.transpose(1, 2), None, pos, f, a).transpose(1, 2)
    out, lse = tsa.paged_tree_attention(q, cache.k, cache.v, table, lens, return_lse=True)
    kl, vl = logical(cache, "f16")
    check(out, lse, q, kl, vl, table.cpu().numpy(), ctx, [T] * B, None)
