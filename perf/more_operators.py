"""A speculative serving step over a latent cache, as cases to time.

* ``pages``   the block table extended from the sequences' lengths, with the position and the
              cache slot of every new token (padded rows or packed ones), and pages given back;
* ``verify``  drafted tokens accepted or replaced by the target's probabilities and given
              random numbers: one line of drafts, with or without the draft's probabilities, or
              a tree of them;
* ``write``   tokens' latent vectors and rotated keys put into their slots of the paged cache,
              and the sequences read back for their keys and values to be expanded;
* ``latent``  attention over that cache, whose keys and values are a token's one latent vector
              with a rotated key beside it (the weights are in q and behind the output):
              decode steps and drafted tokens;
* ``prompt``  the same attention with every head's keys and values expanded, the rotated key
              shared by the heads: whole prompts, and chunks behind cached tokens.

A case holds sizes only; lengths of a batch follow from them by a fixed low-discrepancy
sequence, so that ``work`` needs no seed.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 64
ROPE = 64
GOLDEN = 0.6180339887498949
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _named(name, c):
    return {"name": name, **c} if name else c


def _pages(name, batch, ctx_min, ctx_max, new_min, new_max, packed, keep):
    """keep: of how many of its new tokens a sequence keeps the pages afterwards; -1: of all, nothing is given back."""
    return _named(name, {"kind": "pages", "batch": batch, "ctx_min": ctx_min, "ctx_max": ctx_max, "new_min": new_min,
                         "new_max": new_max, "packed": packed, "keep": keep})


def _verify(name, batch, drafts, ragged, vocab, dtype, drawn, tree):
    """drawn: the draft's own probabilities are given."""
    return _named(name, {"kind": "verify", "batch": batch, "drafts": drafts, "ragged": ragged, "vocab": vocab,
                         "dtype": dtype, "drawn": drawn, "tree": tree})


def _write(name, batch, new_min, new_max, rank):
    return _named(name, {"kind": "write", "batch": batch, "new_min": new_min, "new_max": new_max, "rank": rank})


def _latent(name, batch, tokens, ragged, ctx_min, ctx_max, heads, rank, tree):
    return _named(name, {"kind": "latent", "batch": batch, "tokens": tokens, "ragged": ragged, "ctx_min": ctx_min,
                         "ctx_max": ctx_max, "heads": heads, "rank": rank, "tree": tree})


def _prompt(name, batch, tokens, ragged, ctx_min, ctx_max, heads, head_dim):
    return _named(name, {"kind": "prompt", "batch": batch, "tokens": tokens, "ragged": ragged, "ctx_min": ctx_min,
                         "ctx_max": ctx_max, "heads": heads, "head_dim": head_dim})


def listed():
    return [
        # A speculative step of 64 sequences: pages for 25 drafted tokens each, those of the
        # rejected ones given back.  Latency.
        _pages("pages_drafts", 64, 100, 16000, 25, 25, False, 9),
        # 256 prompts of up to 8192 tokens admitted at once, packed.
        _pages("pages_prompts", 256, 0, 0, 128, 8192, True, -1),
        # One user's line of 7 drafted tokens, with the draft model's probabilities.  Latency.
        _verify("verify_one", 1, 7, False, 32000, "f32", True, False),
        # A batch's lines of up to 5 drafted tokens over a large vocabulary.
        _verify("verify_batch", 64, 5, True, 128000, "f32", True, False),
        # Trees of 25 drafted tokens (the likeliest ones, no probabilities), odd vocabulary.
        _verify("verify_tree", 16, 25, False, 100003, "bf16", False, True),
        # Prompts written to the cache, packed, and read back.
        _write("latent_write", 16, 100, 1500, 512),
        # One user, a short chat so far, 16 heads (a share of a model's).  Latency.
        _latent("latent_one", 1, 1, False, 700, 700, 16, 512, False),
        # The benchmark's step, 32 sequences of 4096 tokens, with many heads.
        _latent("latent_batch", 32, 1, False, 4096, 4096, 128, 512, False),
        # Continuous batching: 64 sequences anywhere between 128 and 16384 tokens, 16 heads.
        _latent("latent_ragged", 64, 1, False, 128, 16384, 16, 512, False),
        # Trees of up to 7 drafted tokens behind their contexts.
        _latent("latent_drafts", 16, 7, True, 500, 6000, 32, 512, True),
        # Chunked prefill: 512 tokens behind 2000 to 8000 cached ones.
        _prompt("prompt_chunk", 4, 512, False, 2000, 8000, 32, 128),
        # Prompts from their first token on, uneven (the largest call).
        _prompt("prompt_whole", 3, 4000, True, 0, 0, 32, 128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["pages", "pages", "verify", "verify", "verify", "write", "latent", "latent", "latent", "prompt", "prompt"])
    if kind == "pages":
        batch = _log_int(rng, 1, 512)
        if rng.random() < 0.5:  # a step of drafts or of single tokens
            new = rng.choice([1, _log_int(rng, 2, 64)])
            lo, hi = sorted(_log_int(rng, 1, 16384) for _ in range(2))
            return _pages(None, batch, lo, hi, rng.randint(0, new), new, rng.random() < 0.3, rng.choice([-1, rng.randint(0, new)]))
        hi = _log_int(rng, 2, min(8192, (1 << 20) // batch))
        ctx = rng.choice([0, _log_int(rng, 1, 8192)])
        return _pages(None, batch, ctx // 3, ctx, hi // 4, hi, rng.random() < 0.7, -1)
    if kind == "verify":
        drafts, vocab = _log_int(rng, 1, 32), _log_int(rng, 500, 160000)
        batch = _log_int(rng, 1, max(1, min(64, (1 << 25) // (drafts * vocab))))
        drawn = rng.random() < 0.5
        return _verify(None, batch, drafts, rng.random() < 0.5, vocab, rng.choice(["f32", "f32", "f16", "bf16"]), drawn,
                       not drawn and rng.random() < 0.6)
    rank = rng.choice([512, 512, 256])
    if kind == "write":
        batch = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, max(1, 16000 // batch))
        return _write(None, batch, hi // 3, hi, rank)
    batch, heads = _log_int(rng, 1, 64), rng.choice([8, 16, 20, 32, 64, 128])
    if kind == "latent":
        tokens = 1 if rng.random() < 0.5 else _log_int(rng, 2, 25)
        # At most the listed batch's products, a quarter of the ragged batch's tokens.
        hi = _log_int(rng, 1, max(1, min(16384, (1 << 24) // (batch * tokens * heads), (1 << 17) // batch)))
        lo = hi if rng.random() < 0.3 else int(hi * rng.uniform(0.0, 0.9))
        return _latent(None, batch, tokens, tokens > 1 and rng.random() < 0.5, lo, hi, heads, rank,
                       tokens > 1 and rng.random() < 0.5)
    tokens = _log_int(rng, 16, 4000)
    # At most a quarter of the listed prompts' products and of the listed chunks' keys.
    batch = max(1, min(batch, (1 << 27) // (tokens * tokens * heads), (1 << 18) // (tokens * heads)))
    hi = min(16384, (1 << 27) // (batch * tokens * heads), (1 << 18) // (batch * heads))
    hi = _log_int(rng, 1, max(1, hi)) if rng.random() < 0.6 else 0
    lo = hi if rng.random() < 0.3 else int(hi * rng.uniform(0.0, 0.9))
    return _prompt(None, batch, tokens, rng.random() < 0.5, lo, hi, heads, rng.choice([128, 128, 64]))


# ---------------------------------------------------------------- sizes --

def _spread(n, lo, hi):
    """n whole numbers between lo and hi, the first of them hi."""
    return [hi] + [lo + int((hi - lo + 1) * ((i * GOLDEN) % 1.0)) for i in range(1, n)]


def _contexts(case):
    return _spread(case["batch"], case["ctx_min"], case["ctx_max"])


def _new(case):
    """New tokens of each sequence."""
    if case["kind"] in ("pages", "write"):
        return _spread(case["batch"] + 1, case["new_min"], case["new_max"])[::-1][:-1]  # another order than the contexts'
    n = case["drafts" if case["kind"] == "verify" else "tokens"]
    return _spread(case["batch"], max(1, n // 3), n) if case["ragged"] else [n] * case["batch"]


def _count(n):
    return -(-n // PAGE)


def work(case):
    B = case["batch"]
    if case["kind"] == "pages":
        ctx, new = _contexts(case), _new(case)
        rows = sum(new) if case["packed"] else B * max(new)
        taken = sum(_count(c + n) - _count(c) for c, n in zip(ctx, new))
        return {"bytes": 12 * rows + 12 * taken + 16 * B, "flops": 2 * rows}
    if case["kind"] == "verify":
        size, V = DTYPES[case["dtype"]].itemsize, case["vocab"]
        rows = 2 if case["drawn"] else 1  # the target's row where the line ends, and the draft's
        return {"bytes": B * (rows * V * size + 16 * case["drafts"]), "flops": 3 * B * V}
    if case["kind"] == "write":
        n, width = sum(_new(case)), case["rank"] + ROPE
        return {"bytes": n * (4 * width + 8) + 2 * (n + B * max(_new(case))) * width, "flops": n * width}
    H, T = case["heads"], case["tokens"]
    counts, ctx = _new(case), _contexts(case)
    tokens = sum(c + n for c, n in zip(ctx, counts))
    if case["kind"] == "latent":
        rank, pairs = case["rank"], sum(n * (c + n) for c, n in zip(ctx, counts))
        mask = B * T * T if case["tree"] else 0
        return {"bytes": 2 * tokens * (rank + ROPE) + B * T * H * (4 * rank + 2 * ROPE + 4) + mask,
                "flops": 2 * pairs * H * (2 * rank + ROPE)}
    D, pairs = case["head_dim"], sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, counts))
    return {"bytes": 2 * tokens * (2 * H * D + ROPE) + B * T * H * (4 * D + 2 * ROPE + 4),
            "flops": 2 * pairs * H * (2 * D + ROPE)}


# --------------------------------------------------------------- inputs --

def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 64 + what) % (1 << 62))


def _randn(shape, seed, what, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=_gen(seed, what))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _shuffled(n, seed, what):
    return torch.randperm(n, generator=_gen(seed, what), device="cuda").to(torch.int32)


def _table(counts, seed):
    """A block table whose pages are anywhere in the pool, and the pool's size."""
    pages = [max(1, _count(c)) for c in counts]
    total, width = sum(pages), max(pages)
    order = _shuffled(total, seed, 40).cpu()
    table = torch.zeros((len(counts), width), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to("cuda"), total


def _prepare_pages(case, s, seed):
    """A pool in use: every sequence holds its context's pages, the ring of free ones has been gone round."""
    B, ctx, new = case["batch"], _contexts(case), _new(case)
    held = [_count(c) for c in ctx]
    need = [_count(c + n) for c, n in zip(ctx, new)]
    spare = 1 + sum(need) // 8
    size = sum(need) + spare
    order = _shuffled(size, seed, 40)
    width = max(need) + 3
    table = torch.full((B, width), -1, dtype=torch.int32)
    ids, at = order.cpu(), 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    taken = size + int(seed) % 1000  # pages taken and returned since the pool was made
    ring = torch.empty_like(order)
    ring[(torch.arange(size - at, device="cuda") + taken) % size] = order[at:]
    ring[(torch.arange(at, device="cuda") + taken + size - at) % size] = order[:at]  # stale: given out
    s["table"], s["ring"] = table.to("cuda"), ring
    s["held"], s["ctx"], s["new"] = _int32(held), _int32(ctx), _int32(new)
    s["cursor"] = torch.tensor([taken, taken + size - at], dtype=torch.int64, device="cuda")
    s["length"], s["total"] = max(new), sum(new)
    if case["keep"] >= 0:
        s["kept"] = _int32([c + min(n, case["keep"]) for c, n in zip(ctx, new)])


def _parents(case, seed):
    """A random tree over each sequence's drafts: the parent of each, -1 the context's last token."""
    r = torch.rand((case["batch"], case["drafts"]), generator=_gen(seed, 12), device="cuda")
    return (r * torch.arange(1, case["drafts"] + 1, device="cuda")).to(torch.int32) - 1


def _prepare_verify(case, s, seed):
    B, T, V, dtype = case["batch"], case["drafts"], case["vocab"], DTYPES[case["dtype"]]
    logits = _randn((B, T + 1, V), seed, 1, torch.float32).mul_(2.5)
    s["target"] = torch.softmax(logits, -1).to(dtype)
    s["uniforms"] = torch.rand((B, T + 1), generator=_gen(seed, 2), device="cuda")
    s["counts"] = _int32(_new(case)) if case["ragged"] else None
    s["parents"] = _parents(case, seed) if case["tree"] else None
    if case["drawn"]:  # a draft model near the target; the tokens are drawn from it
        q = torch.softmax(logits[:, :T] + 0.7 * _randn((B, T, V), seed, 3, torch.float32), -1).to(dtype)
        s["draft"], source = q, q
    else:  # tokens that are likely behind their parents
        rows = s["parents"].long() + 1 if case["tree"] else torch.arange(T, device="cuda").expand(B, T)
        s["draft"], source = None, s["target"].gather(1, rows.unsqueeze(-1).expand(-1, -1, V))
        source = source.float() ** 1.5
    s["tokens"] = torch.multinomial(source.reshape(B * T, V).float(), 1, generator=_gen(seed, 4)).view(B, T)


def _latents(shape, rank, seed, what):
    """Latent vectors and rotated keys as a model's are: features of uneven size."""
    x = _randn((*shape, rank + ROPE), seed, what)
    x *= torch.exp(0.3 * _randn((rank + ROPE,), seed, 30, torch.float32)).half()
    return x


def _prepare_write(case, s, seed):
    new = _new(case)
    table, pool = _table(new, seed)
    rows = _latents((sum(new),), case["rank"], seed, 1)
    s["latent"], s["rope"] = rows[:, :case["rank"]], rows[:, case["rank"]:]  # one projection's output
    s["cache"] = _randn((pool, (case["rank"] + ROPE) // 64, PAGE, 64), seed, 2)
    slots = [table[b, :max(1, _count(n))].long().unsqueeze(1) * PAGE + torch.arange(PAGE, device="cuda")
             for b, n in enumerate(new)]
    s["slots"] = torch.cat([x.flatten()[:n] for x, n in zip(slots, new)])
    s["table"], s["lens"], s["length"] = table, _int32(new), max(new)


def _tree_mask(case, seed):
    """mask[b, i, j]: j is drafted token i or one it descends from."""
    B, T = case["batch"], case["tokens"]
    parents = _parents({**case, "drafts": T}, seed).long().cpu()
    mask = torch.eye(T, dtype=torch.bool).repeat(B, 1, 1)
    rows = torch.arange(B)
    for i in range(1, T):
        mask[:, i] |= mask[rows, parents[:, i].clamp(min=0)] & (parents[:, i] >= 0).unsqueeze(1)
    return mask.to("cuda")


def _prepare_latent(case, s, seed):
    B, T, H, rank = case["batch"], case["tokens"], case["heads"], case["rank"]
    ctx, counts = _contexts(case), _new(case)
    s["table"], pool = _table([c + n for c, n in zip(ctx, counts)], seed)
    rows = _latents((pool, PAGE), rank, seed, 1)  # pages [pool, (rank + ROPE) / 64, 64 tokens, 64]
    s["cache"] = rows.view(pool, PAGE, -1, 64).transpose(1, 2).contiguous()
    # q with the keys' weights in it, as a product batched over the heads leaves it
    s["q"] = _randn((H, B, T, rank), seed, 2).mul_(0.5).permute(1, 2, 0, 3)
    s["q_rope"] = _randn((B, T, H, ROPE), seed, 3)
    s["scale"] = 1.0 / math.sqrt(128 + ROPE)
    s["ctx"], s["max_ctx"] = _int32(ctx), max(ctx)
    s["counts"] = _int32(counts) if case["ragged"] else None
    s["mask"] = _tree_mask(case, seed) if case["tree"] else None


def _prepare_prompt(case, s, seed):
    B, T, H, D = case["batch"], case["tokens"], case["heads"], case["head_dim"]
    ctx, counts = _contexts(case), _new(case)
    n = max(c + k for c, k in zip(ctx, counts))
    kv = _latents((B, n, H), 2 * D - ROPE, seed, 1)  # one projection's output: keys and values of a head
    s["k"], s["v"], s["k_rope"] = kv[..., :D], kv[..., D:], _randn((B, n, ROPE), seed, 2)
    q = _randn((B, T, H, D + ROPE), seed, 3)
    s["q"], s["q_rope"] = q[..., :D], q[..., D:]
    s["ctx"], s["counts"] = _int32(ctx), _int32(counts) if case["ragged"] else None


def prepare(case, seed):
    s = dict(case)
    {"pages": _prepare_pages, "verify": _prepare_verify, "write": _prepare_write, "latent": _prepare_latent,
     "prompt": _prepare_prompt}[case["kind"]](case, s, seed)
    return s


# ------------------------------------------------------- the plain forms --

def _before(x):
    """The sum of what lies before each entry."""
    return x.cumsum(0) - x


def _plain_pages(s):
    table, held, ctx, new = s["table"], s["held"].long(), s["ctx"].long(), s["new"].long()
    ring, taken, returned = s["ring"], s["cursor"][0], s["cursor"][1]
    B, W, F = *table.shape, ring.numel()
    need = (torch.div(ctx + new + PAGE - 1, PAGE, rounding_mode="floor").clamp(max=W) - held).clamp(min=0)
    first = _before(need)
    got = torch.minimum(need, (returned - taken - first).clamp(min=0))
    column = torch.arange(W, device="cuda")
    i = column - held.unsqueeze(1)
    fresh = (i >= 0) & (i < got.unsqueeze(1))
    pages = ring[(taken + first.unsqueeze(1) + i) % F]
    table.copy_(torch.where(fresh, pages, table))
    held2 = held + got
    cursor = torch.stack((taken + got.sum(), returned))
    if s["packed"]:
        starts = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), new.cumsum(0)))
        n = torch.arange(s["total"], device="cuda")
        b = torch.searchsorted(starts[1:], n, right=True)
        at, live = ctx[b] + n - starts[b], None
    else:
        starts = torch.zeros(0, dtype=torch.int64, device="cuda")
        t = torch.arange(s["length"], device="cuda")
        at, live = ctx.unsqueeze(1) + t, t < new.unsqueeze(1)
        b = torch.arange(B, device="cuda").unsqueeze(1).expand_as(at)
    page = torch.div(at, PAGE, rounding_mode="floor")
    there = page < held2[b] if live is None else live & (page < held2[b])
    slots = table[b, page.clamp(max=W - 1)].long() * PAGE + at % PAGE
    nowhere = torch.full_like(at, -1)
    out = {"positions": (at if live is None else torch.where(live, at, nowhere)).to(torch.int32),
           "slots": torch.where(there, slots, nowhere), "starts": starts.to(torch.int32), "table": table}
    if s["keep"] >= 0:
        keep = torch.minimum(held2, torch.div(s["kept"].long() + PAGE - 1, PAGE, rounding_mode="floor"))
        back = held2 - keep
        i = column - keep.unsqueeze(1)
        gone = (i >= 0) & (i < back.unsqueeze(1))
        to = torch.where(gone, (returned + _before(back).unsqueeze(1) + i) % F, F)  # F: nowhere
        ring.copy_(torch.cat((ring, ring[:1])).scatter(0, to.flatten(), table.flatten())[:F])
        held2, cursor = keep, torch.stack((cursor[0], returned + back.sum()))
        out["ring"] = ring
    return {**out, "held": held2.to(torch.int32), "cursor": cursor}


def _plain_verify(s):
    target, draft, tokens = s["target"], s["draft"], s["tokens"]
    B, T = tokens.shape
    V = target.shape[-1]
    counts = s["counts"].long() if s["counts"] is not None else torch.full((B,), T, device="cuda")
    parents = s["parents"].long() if s["parents"] is not None else torch.arange(-1, T - 1, device="cuda").expand(B, T)
    u, rows = s["uniforms"].double(), torch.arange(B, device="cuda")
    at = torch.full((B,), -1, device="cuda")  # the last accepted token
    left = torch.ones(B, dtype=torch.float64, device="cuda")  # of the probability behind it, what its rejected children leave
    refused = torch.zeros((B, T), dtype=torch.bool, device="cuda")
    accepted = torch.zeros(B, dtype=torch.int64, device="cuda")
    path = torch.full((B, T), -1, device="cuda")
    for i in range(T):
        x = tokens[:, i]
        tried = (parents[:, i] == at) & (i < counts)
        p = target[rows, at + 1, x].double()
        p = torch.where((refused & (tokens == x.unsqueeze(1))).any(1), torch.zeros_like(p), p)
        limit = draft[:, i].gather(1, x.unsqueeze(1)).squeeze(1).double() if draft is not None else left
        taken = tried & (u[:, i] * limit < p)
        lost = tried & ~taken
        left = torch.where(taken, torch.ones_like(left), torch.where(lost, left - p, left))
        refused[:, i] = lost
        refused &= ~taken.unsqueeze(1)
        path[rows, accepted.clamp(max=T - 1)] = torch.where(taken, torch.full_like(at, i), path[rows, accepted.clamp(max=T - 1)])
        accepted += taken
        at = torch.where(taken, torch.full_like(at, i), at)
    p = target[rows, at + 1].double()
    if draft is not None:
        q = draft[rows, (at + 1).clamp(max=T - 1)].double()
        w = torch.where(refused.any(1, keepdim=True), (p - q).clamp(min=0), p)
    else:
        gone = torch.zeros((B, V + 1), dtype=torch.bool, device="cuda")
        gone.scatter_(1, torch.where(refused, tokens, torch.full_like(tokens, V)), True)
        w = p.masked_fill(gone[:, :V], 0)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, p)
    sums = w.cumsum(1)
    last = torch.searchsorted(sums, (u[:, T] * sums[:, -1]).unsqueeze(1), right=True).squeeze(1)
    out = torch.full((B, T + 1), -1, device="cuda")
    out[:, :T] = torch.where(path >= 0, tokens.gather(1, path.clamp(min=0)), path)
    out[rows, accepted] = last
    return {"tokens": out, "accepted": accepted.to(torch.int32), "path": path.to(torch.int32)}


def _rows(s):
    """The latent vectors and rotated keys [B, tokens, rank + ROPE] of the table's pages."""
    rows = s["cache"][s["table"].long()].transpose(2, 3)
    return rows.reshape(rows.shape[0], -1, s["rank"] + ROPE)


def _plain_write(s):
    rows = torch.cat((s["latent"], s["rope"]), 1)
    page, token = torch.div(s["slots"], PAGE, rounding_mode="floor"), s["slots"] % PAGE
    s["cache"][page, :, token] = rows.view(rows.shape[0], -1, 64)
    live = torch.arange(s["length"], device="cuda") < s["lens"].unsqueeze(1)
    back = _rows(s)[:, :s["length"]].masked_fill(~live.unsqueeze(2), 0)
    return {"cache": s["cache"], "latent": back[..., :s["rank"]].contiguous(), "rope": back[..., s["rank"]:].contiguous()}


def _plain_latent(s):
    q, qr, rows, rank = s["q"].float(), s["q_rope"].float(), _rows(s).float(), s["rank"]
    B, T, H, _ = q.shape
    c, n = rows[..., :rank].contiguous(), rows.shape[1]
    score = torch.matmul(torch.cat((q, qr), -1).view(B, T * H, -1), rows.transpose(1, 2).contiguous())
    counts = s["counts"] if s["counts"] is not None else torch.full_like(s["ctx"], T)
    j = torch.arange(n, device="cuda") - s["ctx"].unsqueeze(1)  # which new token; negative in the context
    tree = s["mask"]
    if tree is None:
        tree = torch.ones((T, T), dtype=torch.bool, device="cuda").tril().expand(B, T, T)
    seen = tree.gather(2, j.clamp(0, T - 1).unsqueeze(1).expand(-1, T, -1).long())
    keep = (j < 0).unsqueeze(1) | (seen & ((j >= 0) & (j < counts.unsqueeze(1))).unsqueeze(1))
    keep &= (torch.arange(T, device="cuda") < counts.unsqueeze(1)).unsqueeze(2)  # rows of no new token: zeros
    e, total, lse = _weights((score * s["scale"]).view(B, T, H, n).masked_fill(~keep.unsqueeze(2), -math.inf))
    out = torch.matmul(e.view(B, T * H, n), c).view(B, T, H, rank) / total
    return {"out": out.half(), "lse": lse}


def _plain_prompt(s):
    B, T, H, D = s["q"].shape
    n = s["k"].shape[1]
    counts = s["counts"] if s["counts"] is not None else torch.full_like(s["ctx"], T)
    i = torch.arange(T, device="cuda")
    keep = torch.arange(n, device="cuda").view(1, 1, n) <= (s["ctx"].unsqueeze(1) + i).unsqueeze(2)
    keep &= (i < counts.unsqueeze(1)).unsqueeze(2)  # rows of no new token: zeros
    out = torch.empty((B, T, H, D), dtype=torch.float16, device="cuda")
    lse = torch.empty((B, T, H), dtype=torch.float32, device="cuda")
    for h in range(H):
        q = torch.cat((s["q"][:, :, h], s["q_rope"][:, :, h]), -1).float()
        k = torch.cat((s["k"][:, :, h], s["k_rope"]), -1).float()
        score = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(D + ROPE)
        e, total, lse[:, :, h] = _weights(score.masked_fill(~keep, -math.inf))
        out[:, :, h] = (torch.matmul(e, s["v"][:, :, h].float().contiguous()) / total).half()
    return {"out": out, "lse": lse}


def _weights(score):
    """exp(score - its largest), the sum with empty rows' as one, the logsumexp."""
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e, torch.where(total == 0, torch.ones_like(total), total), (top + total.log()).squeeze(-1)


# ---------------------------------------------------- the framework's calls --

def _own_pages(s):
    import torch_spyre_amd as tsa

    size = {"tokens": s["total"]} if s["packed"] else {"length": s["length"]}
    plan = tsa.plan_pages(s["table"], s["held"], s["ctx"], s["new"], s["ring"], s["cursor"], **size)
    out = {"positions": plan.positions, "slots": plan.slots, "starts": plan.starts, "table": s["table"]}
    held, cursor = plan.held, plan.cursor
    if s["keep"] >= 0:
        held, cursor = tsa.release_pages(s["table"], held, s["kept"], s["ring"], cursor)
        out["ring"] = s["ring"]
    return {**out, "held": held, "cursor": cursor}


def _own_verify(s):
    import torch_spyre_amd as tsa

    tokens, accepted, path = tsa.verify_drafts(s["tokens"], s["target"], s["uniforms"], draft_probs=s["draft"],
                                               parents=s["parents"], draft_lens=s["counts"])
    return {"tokens": tokens, "accepted": accepted, "path": path}


def _own_write(s):
    import torch_spyre_amd as tsa

    tsa.latent_append(s["latent"], s["rope"], s["cache"], s["slots"])
    latent, rope = tsa.latent_read(s["cache"], s["table"], s["lens"], s["length"])
    return {"cache": s["cache"], "latent": latent, "rope": rope}


def _own_latent(s):
    import torch_spyre_amd as tsa

    out, lse = tsa.paged_latent_attention(s["q"], s["q_rope"], s["cache"], s["table"], s["ctx"], s["scale"],
                                          tree_mask=s["mask"], draft_lens=s["counts"], max_context_len=s["max_ctx"],
                                          return_lse=True)
    return {"out": out, "lse": lse}


def _own_prompt(s):
    import torch_spyre_amd as tsa

    out, lse = tsa.latent_attention(s["q"], s["q_rope"], s["k"], s["k_rope"], s["v"], s["ctx"], new_lens=s["counts"],
                                    return_lse=True)
    return {"out": out, "lse": lse}


def run(state):
    kind = state["kind"]
    if own:
        return {"pages": _own_pages, "verify": _own_verify, "write": _own_write, "latent": _own_latent,
                "prompt": _own_prompt}[kind](state)
    return {"pages": _plain_pages, "verify": _plain_verify, "write": _plain_write, "latent": _plain_latent,
            "prompt": _plain_prompt}[kind](state)


# --------------------------------------------- the definitions in 64 bits --

def _exact_pages(case, s):
    """Page by page and token by token, in whole numbers of Python."""
    table, held, ring = s["table"].tolist(), s["held"].tolist(), s["ring"].tolist()
    taken, returned = s["cursor"].tolist()
    ctx, new = _contexts(case), _new(case)
    for b in range(case["batch"]):
        while held[b] * PAGE < ctx[b] + new[b] and held[b] < len(table[b]) and taken < returned:
            table[b][held[b]] = ring[taken % len(ring)]
            held[b], taken = held[b] + 1, taken + 1
    positions, slots, starts = [], [], [0]
    for b in range(case["batch"]):
        p = [ctx[b] + t for t in range(new[b])]
        q = [table[b][x // PAGE] * PAGE + x % PAGE if x // PAGE < held[b] else -1 for x in p]
        if not case["packed"]:
            p, q = (x + [-1] * (s["length"] - new[b]) for x in (p, q))
        positions.append(p)
        slots.append(q)
        starts.append(starts[-1] + new[b])
    if case["packed"]:
        positions, slots = ([y for x in z for y in x] for z in (positions, slots))
    else:
        starts = []
    kept = s["kept"].tolist() if case["keep"] >= 0 else []
    for b, n in enumerate(kept):
        keep = min(held[b], _count(n))
        for i in range(keep, held[b]):
            ring[returned % len(ring)] = table[b][i]
            returned += 1
        held[b] = keep
    out = {"positions": _int32(positions), "slots": torch.tensor(slots, dtype=torch.int64, device="cuda"),
           "starts": _int32(starts), "table": _int32(table)}
    if kept:
        out["ring"] = _int32(ring)
    return {**out, "held": _int32(held), "cursor": torch.tensor([taken, returned], dtype=torch.int64, device="cuda")}


def _exact_verify(case, s):
    """One sequence after the other, as the rule is stated."""
    B, T = case["batch"], case["drafts"]
    tokens, u, counts = s["tokens"].tolist(), s["uniforms"].double().tolist(), _new(case)
    parents = s["parents"].tolist() if case["tree"] else [list(range(-1, T - 1))] * B
    result = {"tokens": [], "accepted": [], "path": []}
    for b in range(B):
        path, node, tried, left = [], -1, [], 1.0
        probs = s["target"][b].double()
        for i in range(counts[b]):
            if parents[b][i] != node:
                continue
            x = tokens[b][i]
            p = 0.0 if x in [tokens[b][k] for k in tried] else float(probs[node + 1, x])
            limit = float(s["draft"][b, i, x].double()) if case["drawn"] else left
            if u[b][i] * limit < p:
                path, node, tried, left = path + [i], i, [], 1.0
            else:
                tried, left = tried + [i], left - p
        w = probs[node + 1].clone()
        if case["drawn"] and tried:
            w = torch.relu(w - s["draft"][b, tried[0]].double())
        elif tried:
            w[[tokens[b][k] for k in tried]] = 0
        if float(w.sum()) <= 0:
            w = probs[node + 1]
        w = w.cpu()
        above = torch.nonzero(torch.cumsum(w, 0) > u[b][T] * float(w.sum()))
        chosen = [tokens[b][i] for i in path] + [int(above[0])]
        result["tokens"].append(chosen + [-1] * (T + 1 - len(chosen)))
        result["accepted"].append(len(path))
        result["path"].append(path + [-1] * (T - len(path)))
    return {"tokens": torch.tensor(result["tokens"], device="cuda"), "accepted": _int32(result["accepted"]),
            "path": _int32(result["path"])}


def _sequence(case, s, b, n):
    """Sequence b's first n rows of the cache, in 64 bits."""
    pages = s["cache"][s["table"][b, :max(1, _count(n))].long()]
    return torch.cat(list(pages.double().unbind(1)), -1).flatten(0, 1)[:n]


def _exact_write(case, s):
    rank, new = case["rank"], _new(case)
    flat = s["cache"].permute(0, 2, 1, 3).reshape(-1, rank + ROPE)  # a row for each slot
    flat[s["slots"], :rank] = s["latent"]
    flat[s["slots"], rank:] = s["rope"]
    s["cache"] = flat.view(-1, PAGE, (rank + ROPE) // 64, 64).permute(0, 2, 1, 3)
    back = torch.zeros((case["batch"], max(new), rank + ROPE), dtype=torch.float64, device="cuda")
    for b, n in enumerate(new):
        back[b, :n] = _sequence(case, s, b, n)
    return {"cache": s["cache"].double(), "latent": back[..., :rank], "rope": back[..., rank:]}


def _attended(q, k, v, scale, keep, out, lse):
    score = (q @ k.t().contiguous() * scale).masked_fill(~keep, -math.inf)
    lse.copy_(torch.logsumexp(score, 1))
    out.copy_(torch.softmax(score, 1) @ v)


def _exact_attention(case, s):
    """One head of one sequence after the other."""
    B, T, H = case["batch"], case["tokens"], case["heads"]
    ctx, counts = _contexts(case), _new(case)
    latent = case["kind"] == "latent"
    D = case["rank"] if latent else case["head_dim"]
    out = torch.zeros((B, T, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, T, H), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, total = counts[b], ctx[b] + counts[b]
        keep = torch.ones((n, total), dtype=torch.bool, device="cuda").tril(ctx[b])
        if latent and case["tree"]:
            keep[:, ctx[b]:] = s["mask"][b, :n, :n]
        q = torch.cat((s["q"][b, :n], s["q_rope"][b, :n]), -1).double()
        if latent:  # all heads have the same keys
            k = _sequence(case, s, b, total)
            o, l = out[b, :n].flatten(0, 1), lse[b, :n].flatten()
            _attended(q.flatten(0, 1), k, k[:, :D].contiguous(), s["scale"], keep.repeat_interleave(H, 0), o, l)
            continue
        for h in range(H):
            k = torch.cat((s["k"][b, :total, h], s["k_rope"][b, :total]), 1).double()
            _attended(q[:, h].contiguous(), k, s["v"][b, :total, h].double().contiguous(), (D + ROPE) ** -0.5, keep, out[b, :n, h],
                      lse[b, :n, h])
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("latent", "prompt"):
        return _exact_attention(case, s)
    return {"pages": _exact_pages, "verify": _exact_verify, "write": _exact_write}[case["kind"]](case, s)
