"""GPU: speculative serving steps with a latent cache, all operators together: pages
planned, rows appended, drafts attended and verified, pages given back; prompts through
the cache and the expanded form.  Each result against the oracle on the same inputs (the
tolerances are those of the single operators), and the whole step captured and replayed."""

import numpy as np
import pytest
import torch

from oracle import step as O
from tests.conftest import SEED
from tests.test_latent_gpu import check_paged, close, keep_of, randn

pytestmark = pytest.mark.gpu

B, H, RANK, D, V, K = 5, 6, 256, 64, 97, 4  # K drafted tokens behind each sequence's last
SCALE = (D + 64) ** -0.5
T = K + 1


class Model:
    """Random weights; what a token's row, query and output are."""

    def __init__(self, dev):
        self.latent, self.rope = randn((V, RANK), dev, SEED + 1), randn((V, 64), dev, SEED + 2)
        self.q, self.q_rope = randn((V, H, RANK), dev, SEED + 3, 0.3), randn((V, H, 64), dev, SEED + 4)
        self.head = randn((H * RANK, V), dev, SEED + 5, 0.1).float()
        self.draft = torch.randint(0, V, (V,), generator=torch.Generator(device=dev).manual_seed(SEED + 6), device=dev)

    def probs(self, out):
        return torch.softmax(out.flatten(2).float() @ self.head, -1)

    def line(self, last):  # the last token and its K drafts
        x = [last]
        for _ in range(K):
            x.append(self.draft[x[-1]])
        return torch.stack(x, 1)


class State:
    def __init__(self, dev, pages=24):
        import torch_spyre_amd as tsa

        self.pool = tsa.PagePool(pages, B, 8, device=dev)
        self.cache = tsa.LatentKVCache(pages, RANK, device=dev)
        self.ctx = torch.zeros(B, dtype=torch.int32, device=dev)
        self.last = torch.arange(B, device=dev)
        self.new = torch.full((B,), T, dtype=torch.int32, device=dev)
        self.kept = torch.zeros((B, T), dtype=torch.int64, device=dev)


def step(m, s, u, watch=None):
    """Every sequence gets its last token and K drafts; those that are kept stay."""
    import torch_spyre_amd as tsa

    x = m.line(s.last)
    plan = s.pool.plan(s.ctx, s.new, length=T)
    s.cache.append(m.latent[x], m.rope[x], plan.slots)
    out, lse = s.cache.attend(m.q[x], m.q_rope[x], s.pool.block_table, s.ctx, SCALE, max_context_len=8 * 64 - T, return_lse=True)
    p = m.probs(out)
    tokens, kept, path = tsa.verify_drafts(x[:, 1:], p, u)
    if watch:
        watch(x, plan, out, lse, p, tokens, kept, path)
    s.ctx.add_(kept + 1)
    s.last.copy_(tokens.gather(1, kept.long().unsqueeze(1)).squeeze(1))
    s.kept.copy_(tokens)
    s.pool.release(s.ctx)


def uniforms(dev, steps):
    return torch.rand((steps, B, T), generator=torch.Generator(device=dev).manual_seed(SEED + 9), device=dev) * torch.tensor(
        [0.02] * K + [1.0], device=dev)


def test_steps_against_the_oracle(cuda):
    import torch_spyre_amd as tsa

    m, s, history = Model(cuda), State(cuda), [[] for _ in range(B)]
    counts = set()
    for u in uniforms(cuda, 40):
        ints = lambda t: t.cpu().numpy()  # noqa: E731
        before = [ints(t) for t in (s.pool.block_table, s.pool.held, s.ctx, s.new, s.pool.free_pages, s.pool.cursor)]

        def watch(x, plan, out, lse, p, tokens, kept, path):
            want = O.plan_pages(*before, length=T)
            for got, ref in zip((s.pool.block_table, plan.positions, plan.slots, plan.held, plan.cursor), want):
                assert np.array_equal(ints(got), ref)
            assert (plan.slots >= 0).all()
            ctx = before[2].tolist()
            check_paged(out, lse, m.q[x], m.q_rope[x], s.cache.pages, s.pool.block_table, ctx, [T] * B, SCALE)
            for b in range(B):
                path_, drawn = O.verify(ints(x)[b, 1:], ints(p.double())[b], ints(u.double())[b])
                assert path[b].tolist() == path_ + [-1] * (K - len(path_)) and int(kept[b]) == len(path_)
                row = [int(x[b, 1 + i]) for i in path_] + [drawn]
                assert tokens[b].tolist() == row + [-1] * (T - len(row))
                history[b] += [int(x[b, 0])] + row[:-1]
                counts.add(len(path_))

        step(m, s, u, watch)
        assert s.ctx.tolist() == [len(h) for h in history]
        # Pages of rejected tokens are back: those that rows hold and those that are free are all there are.
        table, held, free, (taken, returned) = ints(s.pool.block_table), ints(s.pool.held), ints(s.pool.free_pages), ints(s.pool.cursor)
        assert held.tolist() == [-(-len(h) // 64) for h in history]
        assert sorted([int(table[b, i]) for b in range(B) for i in range(held[b])]
                      + [int(free[c % len(free)]) for c in range(taken, returned)]) == list(range(len(free)))
    assert len(counts) > 2, "some drafts are kept, some are not"
    # What is cached is what was kept, and both forms of the attention agree on it.
    longest = max(len(h) for h in history)
    latent, rope = s.cache.read(s.pool.block_table, s.ctx, longest)
    for b, h in enumerate(history):
        x = torch.tensor(h, device=cuda)
        assert torch.equal(latent[b, :len(h)], m.latent[x]) and torch.equal(rope[b, :len(h)], m.rope[x])
        assert not latent[b, len(h):].any() and not rope[b, len(h):].any()
    wk = randn((H, D, RANK), cuda, SEED + 20, RANK ** -0.5)
    wv = randn((H, D, RANK), cuda, SEED + 21, RANK ** -0.5)
    k, v = (torch.matmul(latent.view(-1, RANK), w.view(-1, RANK).t()).view(B, longest, H, D) for w in (wk, wv))
    q, qr = randn((B, 1, H, D), cuda, SEED + 22), randn((B, 1, H, 64), cuda, SEED + 23)
    out, lse = tsa.latent_attention(q, qr, k, rope, v, s.ctx - 1, return_lse=True)
    for b, h in enumerate(history):
        n, R = len(h), rope.double().cpu().numpy()
        for hd in range(H):
            keys = np.concatenate((k[b, :n, hd].double().cpu().numpy(), R[b, :n]), -1)
            one = torch.cat((q, qr), -1)[b, :, hd].double().cpu().numpy()
            ref = O.attend(one, keys, v[b, :n, hd].double().cpu().numpy(), keep_of(1, 1, n - 1, 1), SCALE)
            close(out[b, :, hd], lse[b, :, hd], ref, n, float(v.abs().max()))


def eager(m, u):
    s, rows = State(u.device), []
    for x in u:
        step(m, s, x)
        rows.append(s.kept.clone())
    return torch.stack(rows), s


@pytest.mark.parametrize("graphs", [1, 2])
def test_captured_step(cuda, graphs):
    """The captured step, replayed with the program's own eager work between, gives the eager
    run's tokens and cache; two graphs with states of their own take turns."""
    m, u = Model(cuda), uniforms(cuda, 30)
    want, end = eager(m, u)
    runs = []
    for _ in range(graphs):
        s, x = State(cuda), u[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # warm
            step(m, s, x)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(m, s, x)
        fresh = State(cuda)
        for a, b in ((s.pool.block_table, fresh.pool.block_table), (s.pool.held, fresh.pool.held), (s.ctx, fresh.ctx),
                     (s.pool.free_pages, fresh.pool.free_pages), (s.pool.cursor, fresh.pool.cursor), (s.last, fresh.last),
                     (s.cache.pages, fresh.cache.pages)):
            a.copy_(b)
        runs.append((s, x, g))
    for i in range(len(u)):
        for s, x, g in runs:
            x.copy_(u[i])
            g.replay()
        if i % 7 == 3:
            eager(m, u[:2])
            torch.cuda.synchronize()
        for s, _, _ in runs:
            assert torch.equal(s.kept, want[i]), i
    for s, _, _ in runs:
        for a, b in ((s.pool.block_table, end.pool.block_table), (s.ctx, end.ctx), (s.pool.free_pages, end.pool.free_pages),
                     (s.pool.cursor, end.pool.cursor), (s.cache.pages, end.cache.pages)):
            assert torch.equal(a, b)


def test_another_stream(cuda):
    """The step on a stream of its own, behind work that its inputs wait for."""
    m, u = Model(cuda), uniforms(cuda, 6)
    want, _ = eager(m, u)
    a = torch.randn((2048, 2048), device=cuda)
    side, late = torch.cuda.Stream(), torch.zeros_like(u)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            a = a @ a * 1e-2
        late.copy_(u)
        got, _ = eager(m, late)
    side.synchronize()
    assert torch.equal(got, want)


def test_same_call_on_two_streams(cuda):
    """Calls that run at once, each with its own workspace, equal those that run alone."""
    import torch_spyre_amd as tsa

    cache, table = randn((400, 5, 64, 64), cuda, SEED + 30), torch.randperm(400, device=cuda)[:396].view(4, 99).int()
    ctx = torch.tensor([6000, 3000, 77, 6200], dtype=torch.int32, device=cuda)
    q, qr = randn((4, 1, 16, 256), cuda, SEED + 31), randn((4, 1, 16, 64), cuda, SEED + 32)
    kv, kr = randn((2, 5000, 2, 128), cuda, SEED + 33), randn((2, 5000, 64), cuda, SEED + 34)
    few, keys = randn((2, 3, 2, 128), cuda, SEED + 35), torch.tensor([4990, 1234], dtype=torch.int32, device=cuda)
    p, u = torch.softmax(randn((3, 5, 40000), cuda, SEED + 36).float(), -1), torch.rand((3, 5), device=cuda)
    x = torch.randint(0, 40000, (3, 4), device=cuda)
    calls = [lambda: tsa.paged_latent_attention(q, qr, cache, table, ctx, 0.1, max_context_len=6300, return_lse=True),
             lambda: tsa.latent_attention(few[..., :64], few[..., 64:], kv[..., :64], kr, kv[..., 64:], keys, return_lse=True),
             lambda: tsa.verify_drafts(x, p, u)]
    for call in calls:
        want = [t.clone() for t in call()]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for _ in range(10):
            for st in streams:
                with torch.cuda.stream(st):
                    got.append(call())
        torch.cuda.synchronize()
        for g in got:
            assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_captured_calls_of_parts(cuda):
    """Calls whose workspaces hold parts, captured together and replayed over changed lengths."""
    import torch_spyre_amd as tsa

    cache, table = randn((400, 9, 64, 64), cuda, SEED + 40), torch.randperm(400, device=cuda)[:396].view(4, 99).int()
    ctx, counts = torch.zeros(4, dtype=torch.int32, device=cuda), torch.zeros(4, dtype=torch.int32, device=cuda)
    q, qr = randn((4, 3, 40, 512), cuda, SEED + 41, 0.3), randn((4, 3, 40, 64), cuda, SEED + 42)
    kv, kr = randn((4, 6336, 2, 256), cuda, SEED + 43), randn((4, 6336, 64), cuda, SEED + 44)
    few = randn((4, 3, 2, 192), cuda, SEED + 45)

    def run():
        return (*tsa.paged_latent_attention(q, qr, cache, table, ctx, 0.1, None, counts, 6300, True),
                *tsa.latent_attention(few[..., :128], few[..., 128:], kv[..., :128], kr, kv[..., 128:], ctx, counts, return_lse=True))

    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for lens, n in (([6300, 1, 700, 64], [3, 1, 0, 2]), ([0, 0, 0, 0], [1, 0, 0, 3]), ([5, 6000, 6000, 6000], [2, 2, 3, 3]),
                    ([6300] * 4, [3] * 4), ([63, 64, 65, 128], [0] * 4)):
        ctx.copy_(torch.tensor(lens)), counts.copy_(torch.tensor(n))
        g.replay()
        got_now = [t.clone() for t in got]
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got_now, want))
        check_paged(want[0], want[1], q, qr, cache, table, lens, n, 0.1)


def test_far_apart(cuda):
    """Offsets beyond 32 bits: pages behind the first 4 GiB, sequences of keys 4 GiB apart."""
    import torch_spyre_amd as tsa

    pages = (1 << 32) // (9 * 64 * 64 * 2) + 300
    cache = torch.empty((pages, 9, 64, 64), dtype=torch.float16, device=cuda)
    ids = torch.randperm(280, device=cuda).int()[:66] + (pages - 290)
    ids[3] = 0
    table = ids.view(2, 33)
    n = torch.tensor([2050, 1999], dtype=torch.int32, device=cuda)
    latent, rope = randn((2, 2050, 512), cuda, SEED + 50), randn((2, 2050, 64), cuda, SEED + 51)
    t = torch.arange(2050, device=cuda)
    slots = table.long()[:, t // 64] * 64 + t % 64
    tsa.latent_append(latent, rope, cache, slots)
    got = tsa.latent_read(cache, table, n, 2050)
    for b in range(2):
        assert torch.equal(got[0][b, :n[b]], latent[b, :n[b]]) and torch.equal(got[1][b, :n[b]], rope[b, :n[b]])
    q, qr = randn((2, 1, 16, 512), cuda, SEED + 52, 0.3), randn((2, 1, 16, 64), cuda, SEED + 53)
    out, lse = tsa.paged_latent_attention(q, qr, cache, table, n - 1, 0.1, max_context_len=2050, return_lse=True)
    small = torch.cat((cache[:1], cache[pages - 290:]))
    near = torch.where(table == 0, 0, table - (pages - 290) + 1).int()
    want = tsa.paged_latent_attention(q, qr, small, near, n - 1, 0.1, max_context_len=2050, return_lse=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    del cache

    far = (1 << 31) + 4096  # elements
    room = torch.empty(far + 300 * 2 * 128, dtype=torch.float16, device=cuda)
    kv = room.as_strided((2, 300, 2, 128), (far, 256, 128, 1))
    kv.copy_(randn((2, 300, 2, 128), cuda, SEED + 54))
    kr, one = randn((2, 300, 64), cuda, SEED + 55), randn((2, 200, 2, 128), cuda, SEED + 56)
    ctx = torch.tensor([100, 37], dtype=torch.int32, device=cuda)
    args = one[..., :64], one[..., 64:]
    assert torch.equal(tsa.latent_attention(*args, kv[..., :64], kr, kv[..., 64:], ctx),
                       tsa.latent_attention(*args, kv[..., :64].contiguous(), kr, kv[..., 64:].contiguous(), ctx))
    p = room.as_strided((2, 3, 100), (far, 100, 1))
    p.copy_(torch.softmax(randn((2, 3, 100), cuda, SEED + 57).float(), -1))
    x, u = torch.tensor([[3, 50], [99, 0]], device=cuda), torch.rand((2, 3), device=cuda)
    assert all(torch.equal(a, b) for a, b in zip(tsa.verify_drafts(x, p, u), tsa.verify_drafts(x, p.contiguous(), u)))
