"""GPU: page plans with the fp16 and the 8-bit cache and rotary positions: three steps of ragged
sequences whose pages come and go, against tables and positions built on the host."""

import pytest
import torch

from tests.conftest import SEED
from tests.test_quantized_gpu import DTYPE
from tests.test_tree_attention_gpu import check, logical

pytestmark = pytest.mark.gpu

B, Hq, Hkv, D, T = 4, 8, 2, 128, 70


def steps(dev):
    """Cached tokens before each step and its new ones; what a sequence keeps behind it."""
    return [([0, 0, 0, 0], [70, 5, 64, 0], [70, 0, 64, 0]), ([70, 0, 64, 0], [1, 70, 70, 3], [0, 70, 100, 3]),
            ([0, 70, 100, 3], [60, 59, 29, 70], [60, 129, 129, 73])]


class Host:
    """The same pages handed out by hand."""

    def __init__(self, pages, W):
        self.free, self.rows, self.W = list(range(pages)), [[] for _ in range(B)], W

    def plan(self, ctx, n):
        for b in range(B):
            while len(self.rows[b]) < min(-(-(ctx[b] + n[b]) // 64), self.W) and self.free:
                self.rows[b].append(self.free.pop(0))

    def release(self, kept):
        for b in range(B):
            while len(self.rows[b]) > -(-kept[b] // 64):
                at = -(-kept[b] // 64)
                self.free.append(self.rows[b].pop(at))

    def table(self, dev):
        return torch.tensor([r + [-1] * (self.W - len(r)) for r in self.rows], dtype=torch.int32, device=dev)


def draw(dev, g):
    x = torch.randn((B, T, Hq + 2 * Hkv, D), generator=g, device=dev).half()
    return x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]


@pytest.mark.parametrize("pages", [12, 3])  # 3: the ring runs out, some tokens have no page
@pytest.mark.parametrize("kind", ["e4m3", "int8", "f16"])
def test_planned_steps(cuda, kind, pages):
    import torch_spyre_amd as tsa

    new_cache = lambda: (tsa.PagedKVCache(pages, Hkv, D, device=cuda) if kind == "f16"  # noqa: E731
                         else tsa.QuantizedKVCache(pages, Hkv, D, DTYPE[kind], device=cuda))
    pool, host, cache, other = tsa.PagePool(pages, B, 4, device=cuda), Host(pages, 4), new_cache(), new_cache()
    freq, amp = tsa.rotary_frequencies(D, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(SEED)
    short = False
    for ctx, n, kept in steps(cuda):
        lens, new = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (ctx, n))
        plan = pool.plan(lens, new, length=T)
        host.plan(ctx, n)
        table = host.table(cuda)
        assert plan.held.tolist() == [len(r) for r in host.rows]
        places = torch.where(plan.slots < 0, -1, plan.positions)  # of tokens that have a page
        want = torch.tensor([[ctx[b] + t if t < n[b] and (ctx[b] + t) // 64 < len(host.rows[b]) else -1 for t in range(T)]
                             for b in range(B)], dtype=torch.int32, device=cuda)
        assert torch.equal(places, want)
        short |= any(want[b, :n[b]].min() < 0 for b in range(B) if n[b])
        q, k, v = draw(cuda, g)
        at = torch.tensor([[ctx[b] + t for t in range(T)] for b in range(B)], device=cuda)
        live = want >= 0
        if kind == "f16":
            rq, rk = (x.transpose(1, 2) for x in tsa.rotary_embedding(q.transpose(1, 2), k.transpose(1, 2), plan.positions, freq, amp))
            hq, hk = (x.transpose(1, 2) for x in tsa.rotary_embedding(q.transpose(1, 2), k.transpose(1, 2), at, freq, amp))
            assert torch.equal(rq[live], hq[live]) and torch.equal(rk[live], hk[live])
            for t in range(max(n)):
                tsa.kv_append(rk[:, t].contiguous(), v[:, t].contiguous(), cache.k, cache.v, pool.block_table, places[:, t].contiguous())
                tsa.kv_append(hk[:, t].contiguous(), v[:, t].contiguous(), other.k, other.v, table, want[:, t].contiguous())
            args = {}
        else:
            rq = cache.rotary_append(q, k, v, pool.block_table, places, plan.positions, freq, amp)
            hq = other.rotary_append(q, k, v, table, want, at, freq, amp)
            assert torch.equal(rq[live], hq[live])
            args = dict(k_scale=cache.k_scale, v_scale=cache.v_scale)
            assert torch.equal(cache.k_scale, other.k_scale) and torch.equal(cache.v_scale, other.v_scale)
        assert torch.equal(cache.k.view(torch.uint8), other.k.view(torch.uint8))
        assert torch.equal(cache.v.view(torch.uint8), other.v.view(torch.uint8))
        got = [min(n[b], max(64 * len(host.rows[b]) - ctx[b], 0)) for b in range(B)]  # tokens that have a page
        kept = [min(kept[b], ctx[b] + got[b]) for b in range(B)]
        here = [min(ctx[b], 64 * len(host.rows[b])) for b in range(B)]
        out, lse = tsa.paged_tree_attention(rq, cache.k, cache.v, pool.block_table, torch.tensor(here, dtype=torch.int32, device=cuda),
                                            None, torch.tensor(got, dtype=torch.int32, device=cuda), max_context_len=128,
                                            return_lse=True, **args)
        kl, vl = logical(cache, kind)
        check(out, lse, rq, kl, vl, table.clamp(min=0).cpu().numpy(), here, got, None)
        if pages == 3:
            break  # what a sequence without its pages would cache next is the program's to say
        pool.release(torch.tensor(kept, dtype=torch.int32, device=cuda))
        host.release(kept)
        assert pool.held.tolist() == [len(r) for r in host.rows]
    assert short == (pages == 3)
