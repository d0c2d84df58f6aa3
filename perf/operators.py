"""The serving operators around the paged cache, as cases to time.

* ``rotary``  positions rotated into q and k (half and interleaved pairs, part of the head,
              frequencies scaled for long contexts), with the gradients where ``grad``;
* ``write``   a step's or a prompt's K and V quantised into the 8-bit paged cache (with the
              rotation of q and k in the same call where ``rotate``) and tokens read back;
* ``decode``  one query token a sequence over the 8-bit paged cache;
* ``tree``    the drafted tokens of a speculative step, a tree of them for each sequence, over
              the paged cache (fp16 or 8-bit) that holds them behind their context.

A case holds sizes only; contexts and draft counts of a batch follow from them by a fixed
low-discrepancy sequence, so that ``work`` needs no seed.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 64
GOLDEN = 0.6180339887498949
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}
# (q heads, KV heads, head_dim) of this repository's benchmark and tests.
HEADS = [(32, 8, 128), (64, 8, 128), (16, 16, 64), (32, 32, 128), (8, 8, 64)]


def _rotary(name, batch, length, heads, part, interleaved, scaling, dtype, first, grad):
    c = {"kind": "rotary", "batch": batch, "length": length, "q_heads": heads[0], "kv_heads": heads[1],
         "head_dim": heads[2], "part": part, "interleaved": interleaved, "scaling": scaling, "dtype": dtype,
         "first": first, "grad": grad}
    return {"name": name, **c} if name else c


def _write(name, batch, new, ctx_min, ctx_max, heads, codes, rotate, read_all):
    c = {"kind": "write", "batch": batch, "new": new, "ctx_min": ctx_min, "ctx_max": ctx_max, "q_heads": heads[0],
         "kv_heads": heads[1], "head_dim": heads[2], "codes": codes, "rotate": rotate, "read_all": read_all}
    return {"name": name, **c} if name else c


def _decode(name, batch, ctx_min, ctx_max, heads, codes):
    c = {"kind": "decode", "batch": batch, "ctx_min": ctx_min, "ctx_max": ctx_max, "q_heads": heads[0],
         "kv_heads": heads[1], "head_dim": heads[2], "codes": codes}
    return {"name": name, **c} if name else c


def _tree(name, batch, drafts, ragged, ctx_min, ctx_max, heads, codes, mask):
    c = {"kind": "tree", "batch": batch, "drafts": drafts, "ragged": ragged, "ctx_min": ctx_min, "ctx_max": ctx_max,
         "q_heads": heads[0], "kv_heads": heads[1], "head_dim": heads[2], "codes": codes, "mask": mask}
    return {"name": name, **c} if name else c


def listed():
    return [
        # The decode step of 32 sequences: one token each, anywhere in their contexts.  Latency.
        _rotary("rotary_step", 32, 1, (32, 8, 128), 1.0, False, "llama3", "f16", 4000, False),
        # A long prompt of one sequence (the largest rotation).
        _rotary("rotary_prompt", 1, 8192, (64, 8, 128), 1.0, False, "yarn", "f16", 0, False),
        # Fine-tuning: a quarter of the head rotated in interleaved pairs, gradients of q and k.
        _rotary("rotary_train", 4, 1021, (16, 16, 64), 0.25, True, "none", "bf16", 0, True),
        # The decode step again: q and k rotated, K and V quantised into their slots, read back.
        _write("write_step", 32, 1, 100, 4000, (32, 8, 128), "e4m3", True, False),
        # Prompts of 2500 tokens written to an empty int8 cache, read back for dense attention.
        _write("write_prompt", 3, 2500, 0, 0, (32, 32, 128), "int8", False, True),
        # Chunked prefill: 512 tokens behind 1000 to 8000 cached ones, all of them read back.
        _write("write_chunk", 8, 512, 1000, 8000, (32, 8, 128), "e4m3", True, True),
        # One user, a short chat so far.  Latency.
        _decode("decode_one", 1, 700, 700, (32, 8, 128), "int8"),
        # The benchmark's step, 32 sequences of 4096 tokens, over an 8-bit cache.
        _decode("decode_batch", 32, 4096, 4096, (32, 8, 128), "e4m3"),
        # Continuous batching: 64 sequences anywhere between 128 and 16384 tokens.
        _decode("decode_ragged", 64, 128, 16384, (32, 8, 128), "e4m3"),
        # One user's draft of 7 tokens over fp16 pages, multi-head, head_dim 64.  Latency.
        _tree("tree_one", 1, 7, False, 900, 900, (16, 16, 64), "none", "tree"),
        # A batch's drafts of up to 25 tokens, uneven, over an 8-bit cache.
        _tree("tree_batch", 16, 25, True, 500, 6000, (32, 8, 128), "e4m3", "tree"),
        # Wide trees of 64 tokens, 8 q heads to a KV head, fp16 pages (the largest call).
        _tree("tree_wide", 16, 64, False, 8000, 8192, (64, 8, 128), "none", "tree"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "write", "write", "decode", "decode", "decode", "tree", "tree", "tree"])
    heads = rng.choice(HEADS)
    row = heads[1] * heads[2]
    if kind == "rotary":
        n = _log_int(rng, 1, 8192)
        batch = _log_int(rng, 1, max(1, min(64, (1 << 26) // (n * (heads[0] + heads[1]) * heads[2]))))
        return _rotary(None, batch, n, heads, rng.choice([1.0, 1.0, 0.5, 0.25]), rng.random() < 0.5,
                       rng.choice(["none", "linear", "ntk", "yarn", "llama3"]), rng.choice(["f16", "f16", "bf16", "f32"]),
                       _log_int(rng, 1, 200000), rng.random() < 0.3)
    codes = rng.choice(["e4m3", "e4m3", "int8"])
    if kind == "write":
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        batch = _log_int(rng, 1, max(1, min(64, (1 << 24) // (new * row))))
        hi = _log_int(rng, 1, max(1, min(16384, (1 << 26) // (batch * row)))) if rng.random() < 0.7 else 0
        lo = int(hi * rng.uniform(0.1, 1.0))
        return _write(None, batch, new, lo, hi, heads, codes, rng.random() < 0.6, new > 1 or rng.random() < 0.3)
    if kind == "decode":
        batch = _log_int(rng, 1, 64)
        hi = _log_int(rng, 64, min(32768, (1 << 29) // (batch * row)))
        lo = hi if rng.random() < 0.3 else max(1, int(hi * rng.uniform(0.02, 0.9)))
        return _decode(None, batch, lo, hi, heads, codes)
    drafts = _log_int(rng, 2, 100)
    batch = _log_int(rng, 1, 32)
    # At most a quarter of the widest listed tree's products.
    hi = _log_int(rng, 64, max(64, min(16384, (1 << 27) // (batch * drafts * heads[0]), (1 << 28) // (batch * row))))
    lo = hi if rng.random() < 0.3 else int(hi * rng.uniform(0.0, 0.9))
    return _tree(None, batch, drafts, rng.random() < 0.5, lo, hi, heads, rng.choice(["none", "none", "e4m3", "int8"]),
                 rng.choice(["tree", "tree", "chain"]))


# ---------------------------------------------------------------- sizes --

def _spread(n, lo, hi):
    """n whole numbers between lo and hi, the first of them hi."""
    return [hi] + [lo + int((hi - lo + 1) * ((i * GOLDEN) % 1.0)) for i in range(1, n)]


def _contexts(case):
    return _spread(case["batch"], case["ctx_min"], case["ctx_max"])


def _draft_counts(case):
    """Drafted tokens of each sequence."""
    n = case["drafts"]
    return _spread(case["batch"], max(1, n // 3), n) if case["ragged"] else [n] * case["batch"]


def work(case):
    B, Hq, Hkv, D = case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "rotary":
        n = B * case["length"] * (Hq + Hkv) * D
        size = DTYPES[case["dtype"]].itemsize
        passes = 2 if case["grad"] else 1  # the cotangents in, the gradients out
        return {"bytes": passes * 2 * n * size, "flops": passes * 3 * n * case["part"]}
    if case["kind"] == "write":
        rows = B * case["new"] * Hkv * 2
        read = 2 * Hkv * (sum(c + case["new"] for c in _contexts(case)) if case["read_all"] else B * case["new"])
        width = max(_contexts(case)) + case["new"] if case["read_all"] else case["new"]
        q = 2 * B * case["new"] * Hq * D * 2 if case["rotate"] else 0
        return {"bytes": rows * (3 * D + 4) + read * (D + 4) + 2 * B * width * Hkv * D * 2 + q,
                "flops": 4 * rows * D + read * D}
    size = 2 * D if case["codes"] == "none" else D + 4
    if case["kind"] == "decode":
        T = 1
        tokens = [(c, 1) for c in _contexts(case)]
    else:
        T = case["drafts"]
        tokens = [(c + n, n) for c, n in zip(_contexts(case), _draft_counts(case))]
    total, pairs = sum(c for c, _ in tokens), sum(c * n for c, n in tokens)
    mask = B * T * T if case["kind"] == "tree" and case["mask"] == "tree" else 0
    return {"bytes": 2 * total * Hkv * size + B * T * Hq * (4 * D + 4) + mask, "flops": 4 * pairs * Hq * D}


# --------------------------------------------------------------- inputs --

def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 64 + what) % (1 << 62))


def _randn(shape, seed, what, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=_gen(seed, what))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _frequencies(case):
    """Radians per position of each rotated pair (float64) and the factor on the rotated values:
    base 10000 plainly; positions divided by 4 ("linear"); a base raised so that the slowest pair
    turns 4 times slower ("ntk"); a ramp between the two by the turns a pair makes in 8192
    positions ("yarn", with its factor on the values; "llama3", between 1 and 4 turns, base 500000)."""
    rot = int(case["head_dim"] * case["part"])
    i = torch.arange(0, rot, 2, dtype=torch.float64) / rot
    kind, factor = case["scaling"], 4.0
    base = 500000.0 if kind == "llama3" else 10000.0
    if kind == "ntk":
        base = base * factor ** (rot / (rot - 2))
    f = base ** -i
    amplitude = 1.0
    if kind == "linear":
        f = f / factor
    if kind == "yarn":
        bound = [rot * math.log(8192 / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32, 1)]
        low, high = max(math.floor(bound[0]), 0), min(math.ceil(bound[1]), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        amplitude = 0.1 * math.log(factor) + 1.0
    if kind == "llama3":
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f.to("cuda"), amplitude


def _quantise(x, codes):
    """Codes and the scale of each row (the last dimension), in fp32."""
    x = x.float()
    top = x.abs().amax(-1)
    top = torch.where(top > 0, top, torch.full_like(top, TOP[codes]))
    scale = top / TOP[codes]
    y = x * TOP[codes] / top.unsqueeze(-1)  # the product is exact for fp16, so ties stay ties
    return (y.round().to(torch.int8) if codes == "int8" else y.to(torch.float8_e4m3fn)), scale


def _table(counts, seed):
    """A block table whose pages are anywhere in the pool, and the pool's size."""
    pages = [max(1, -(-c // PAGE)) for c in counts]
    total, width = sum(pages), max(pages)
    order = torch.randperm(total, generator=_gen(seed, 40), device="cuda").to(torch.int32).cpu()
    table = torch.zeros((len(counts), width), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to("cuda"), total


# Pages: fp16 K [P, Hkv, D/64, 64, 64], V [P, Hkv, D, 64]; 8-bit K [P, Hkv, D/16, 64, 16],
# V [P, Hkv, 4, D, 16], with the scales of their tokens [P, Hkv, 64].

def _pages(pool, case, seed):
    """A pool of pages holding values as a model's keys and values are."""
    Hkv, D, codes = case["kv_heads"], case["head_dim"], case["codes"]
    k = _randn((pool, Hkv, PAGE, D), seed, 1)
    k *= torch.exp(0.4 * _randn((Hkv, 1, D), seed, 3, torch.float32)).half()
    v = _randn((pool, Hkv, PAGE, D), seed, 2)
    v *= torch.exp(0.4 * _randn((pool, Hkv, PAGE, 1), seed, 4, torch.float32)).half()
    if codes == "none":
        return {"k": k.view(pool, Hkv, PAGE, D // 64, 64).transpose(2, 3).contiguous(),
                "v": v.transpose(2, 3).contiguous()}
    (kc, ks), (vc, vs) = _quantise(k, codes), _quantise(v, codes)
    kc, vc = kc.view(torch.uint8), vc.view(torch.uint8)
    return {"k": kc.view(pool, Hkv, PAGE, D // 16, 16).transpose(2, 3).contiguous().view(CODES[codes]),
            "v": vc.view(pool, Hkv, 4, 16, D).transpose(3, 4).contiguous().view(CODES[codes]),
            "k_scale": ks.contiguous(), "v_scale": vs.contiguous()}


def _tree_mask(case, seed):
    """mask[b, i, j]: j is drafted token i or one it descends from, in a random tree."""
    B, T = case["batch"], case["drafts"]
    r = torch.rand((B, T), generator=torch.Generator().manual_seed(int(seed) % (1 << 62)))
    mask = torch.eye(T, dtype=torch.bool).repeat(B, 1, 1)
    rows = torch.arange(B)
    for i in range(1, T):
        parent = (r[:, i] * (i + 1)).long() - 1  # -1: from the context's last token
        mask[:, i] |= mask[rows, parent.clamp(min=0)] & (parent >= 0).unsqueeze(1)
    return mask.to("cuda")


def prepare(case, seed):
    B, Hq, Hkv, D = case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"]
    s = dict(case)
    if case["kind"] == "rotary":
        n, dtype = case["length"], DTYPES[case["dtype"]]
        s["q"], s["k"] = _randn((B, n, Hq, D), seed, 10, dtype), _randn((B, n, Hkv, D), seed, 11, dtype)
        first = torch.randint(case["first"] // 2, case["first"] + 1, (B, 1), generator=_gen(seed, 12), device="cuda")
        s["positions"] = (first + torch.arange(n, device="cuda")).to(torch.int32)
        s["frequencies"], s["amplitude"] = _frequencies(case)
        if case["grad"]:
            s["dq"], s["dk"] = _randn((B, n, Hq, D), seed, 13, dtype), _randn((B, n, Hkv, D), seed, 14, dtype)
        return s
    ctx = _contexts(case)
    if case["kind"] == "write":
        n = case["new"]
        s["table"], pool = _table([c + n for c in ctx], seed)
        s.update(_pages(pool, case, seed))
        s["k_new"], s["v_new"] = _randn((B, n, Hkv, D), seed, 10), _randn((B, n, Hkv, D), seed, 11)
        lens = _int32(ctx)
        s["positions"] = (lens.unsqueeze(1) + torch.arange(n, device="cuda", dtype=torch.int32)).contiguous()
        s["lens"] = lens + n
        s["start"], s["length"] = (None, max(ctx) + n) if case["read_all"] else (lens, n)
        if case["rotate"]:
            s["q"] = _randn((B, n, Hq, D), seed, 12)
            s["frequencies"], s["amplitude"] = _frequencies({"head_dim": D, "part": 1.0, "scaling": "llama3"})
        return s
    s["max_ctx"] = max(ctx)
    if case["kind"] == "decode":
        s["table"], pool = _table(ctx, seed)
        s["q"] = _randn((B, Hq, D), seed, 10)
    else:
        drafts = _draft_counts(case)
        s["table"], pool = _table([c + d for c, d in zip(ctx, drafts)], seed)
        s["q"] = _randn((B, case["drafts"], Hq, D), seed, 10)
        s["counts"] = _int32(drafts) if case["ragged"] else None
        s["tree"] = _tree_mask(case, seed) if case["mask"] == "tree" else None
    s.update(_pages(pool, case, seed))
    s["ctx"] = _int32(ctx)
    return s


# ------------------------------------------------------- the plain forms --

def _turn(x, cos, sin, interleaved):
    """x [B, n, H, D] with the pairs of its first features rotated; cos / sin [B, n, 1, R/2]."""
    half = cos.shape[-1]
    y = x.float()
    a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if interleaved else (y[..., :half], y[..., half:2 * half])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1)


def _angles(s):
    theta = s["positions"].double().unsqueeze(-1) * s["frequencies"]
    return (theta.cos() * s["amplitude"]).float().unsqueeze(2), (theta.sin() * s["amplitude"]).float().unsqueeze(2)


def _dense(s, table):
    """K and V [B, Hkv, tokens, D] in fp32 of the table's pages."""
    Hkv, D, idx = s["kv_heads"], s["head_dim"], table.long()
    B, W = idx.shape
    if s["codes"] == "none":
        k = s["k"][idx].permute(0, 2, 1, 4, 3, 5).reshape(B, Hkv, W * PAGE, D).float()
        v = s["v"][idx].permute(0, 2, 1, 4, 3).reshape(B, Hkv, W * PAGE, D).float()
        return k, v
    k = s["k"].view(torch.uint8)[idx].permute(0, 2, 1, 4, 3, 5).reshape(B, Hkv, W * PAGE, D)
    v = s["v"].view(torch.uint8)[idx].permute(0, 2, 1, 3, 5, 4).reshape(B, Hkv, W * PAGE, D)
    ks = s["k_scale"][idx].permute(0, 2, 1, 3).reshape(B, Hkv, W * PAGE, 1)
    vs = s["v_scale"][idx].permute(0, 2, 1, 3).reshape(B, Hkv, W * PAGE, 1)
    return k.view(CODES[s["codes"]]).float() * ks, v.view(CODES[s["codes"]]).float() * vs


def _attend(s, q, keep, table):
    """q [B, T, Hq, D] over the table's tokens where keep [B, T, tokens]: out and the logsumexp."""
    B, T, Hq, D = q.shape
    Hkv = s["kv_heads"]
    k, v = _dense(s, table)
    rows = q.float().view(B, T, Hkv, Hq // Hkv, D).transpose(1, 2).reshape(B, Hkv, -1, D)
    score = torch.matmul(rows, k.transpose(-1, -2).contiguous()) / math.sqrt(D)
    score = score.view(B, Hkv, T, Hq // Hkv, -1).masked_fill(~keep[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.view(B, Hkv, -1, k.shape[2]), v).view(B, Hkv, T, Hq // Hkv, D)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + total.log()).squeeze(-1)
    return out.transpose(1, 2).reshape(B, T, Hq, D).half(), lse.transpose(1, 2).reshape(B, T, Hq)


def _plain_rotary(s):
    cos, sin = _angles(s)
    dtype, pairs = DTYPES[s["dtype"]], s["interleaved"]
    out = {"q": _turn(s["q"], cos, sin, pairs).to(dtype), "k": _turn(s["k"], cos, sin, pairs).to(dtype)}
    if s["grad"]:
        out["dq"] = _turn(s["dq"], cos, -sin, pairs).to(dtype)
        out["dk"] = _turn(s["dk"], cos, -sin, pairs).to(dtype)
    return out


def _plain_write(s):
    out, k_new = {}, s["k_new"].float()
    if s["rotate"]:
        cos, sin = _angles(s)
        out["q"], k_new = _turn(s["q"], cos, sin, False).half(), _turn(s["k_new"], cos, sin, False)
    at = s["positions"].long()
    page, slot = s["table"].long().gather(1, at // PAGE), at % PAGE
    D = s["head_dim"]
    (kc, ks), (vc, vs) = _quantise(k_new, s["codes"]), _quantise(s["v_new"], s["codes"])
    kc, vc = kc.view(torch.uint8), vc.view(torch.uint8)
    s["k"].view(torch.uint8)[page, :, :, slot] = kc.view(*kc.shape[:3], D // 16, 16)
    s["v"].view(torch.uint8)[page, :, slot // 16, :, slot % 16] = vc
    s["k_scale"][page, :, slot], s["v_scale"][page, :, slot] = ks, vs
    start = s["start"] if s["start"] is not None else torch.zeros_like(s["lens"])
    t = start.long().unsqueeze(1) + torch.arange(s["length"], device="cuda")
    live = t < s["lens"].unsqueeze(1)
    t = t.clamp(max=s["table"].shape[1] * PAGE - 1)
    page, slot = s["table"].long().gather(1, t // PAGE), t % PAGE
    k = s["k"].view(torch.uint8)[page, :, :, slot].flatten(-2).view(CODES[s["codes"]]).float()
    v = s["v"].view(torch.uint8)[page, :, slot // 16, :, slot % 16].view(CODES[s["codes"]]).float()
    k = k * s["k_scale"][page, :, slot].unsqueeze(-1) * live[..., None, None]
    v = v * s["v_scale"][page, :, slot].unsqueeze(-1) * live[..., None, None]
    out["k"], out["v"] = k.transpose(1, 2).half().contiguous(), v.transpose(1, 2).half().contiguous()
    return out


def _plain_decode(s):
    t = torch.arange(s["table"].shape[1] * PAGE, device="cuda")
    keep = (t < s["ctx"].unsqueeze(1)).unsqueeze(1)
    out, lse = _attend(s, s["q"].unsqueeze(1), keep, s["table"])
    return {"out": out.squeeze(1), "lse": lse.squeeze(1)}


def _plain_tree(s):
    T = s["drafts"]
    t = torch.arange(s["table"].shape[1] * PAGE, device="cuda")
    j = t - s["ctx"].unsqueeze(1)  # [B, tokens]: which drafted token; negative in the context
    counts = s["counts"] if s["counts"] is not None else torch.full_like(s["ctx"], T)
    tree = s["tree"]
    if tree is None:
        tree = torch.ones((T, T), dtype=torch.bool, device="cuda").tril().expand(j.shape[0], T, T)
    seen = tree.gather(2, j.clamp(0, T - 1).unsqueeze(1).expand(-1, T, -1).long())
    keep = (j < 0).unsqueeze(1) | (seen & ((j >= 0) & (j < counts.unsqueeze(1))).unsqueeze(1))
    keep &= (torch.arange(T, device="cuda") < counts.unsqueeze(1)).unsqueeze(2)  # rows of no drafted token: zeros
    out, lse = _attend(s, s["q"], keep, s["table"])
    return {"out": out, "lse": lse}


# ---------------------------------------------------- the framework's calls --

def _own_rotary(s):
    import torch_spyre_amd as tsa

    q, k = s["q"].transpose(1, 2), s["k"].transpose(1, 2)
    if s["grad"]:
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    yq, yk = tsa.rotary_embedding(q, k, s["positions"], s["frequencies"], amplitude=s["amplitude"],
                                  interleaved=s["interleaved"])
    out = {"q": yq.detach().transpose(1, 2), "k": yk.detach().transpose(1, 2)}
    if s["grad"]:
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (s["dq"].transpose(1, 2), s["dk"].transpose(1, 2)))
        out["dq"], out["dk"] = dq.transpose(1, 2), dk.transpose(1, 2)
    return out


def _own_write(s):
    import torch_spyre_amd as tsa

    out = {}
    cache = (s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["rotate"]:
        out["q"] = tsa.rotary_kv_append_quantized(s["q"], s["k_new"], s["v_new"], *cache, s["table"], s["positions"],
                                                  s["positions"], s["frequencies"], amplitude=s["amplitude"])
    else:
        tsa.kv_append_quantized(s["k_new"], s["v_new"], *cache, s["table"], s["positions"])
    out["k"], out["v"] = tsa.kv_read_quantized(*cache, s["table"], s["lens"], s["length"], start=s["start"])
    return out


def _own_decode(s):
    import torch_spyre_amd as tsa

    out, lse = tsa.paged_decode_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], max_context_len=s["max_ctx"],
                                          return_lse=True, k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {"out": out, "lse": lse}


def _own_tree(s):
    import torch_spyre_amd as tsa

    out, lse = tsa.paged_tree_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], s["tree"],
                                        draft_lens=s["counts"], max_context_len=s["max_ctx"], return_lse=True,
                                        k_scale=s.get("k_scale"), v_scale=s.get("v_scale"))
    return {"out": out, "lse": lse}


def run(state):
    kind = state["kind"]
    if own:
        call = {"rotary": _own_rotary, "write": _own_write, "decode": _own_decode, "tree": _own_tree}
        return call[kind](state)
    plain = {"rotary": _plain_rotary, "write": _plain_write, "decode": _plain_decode, "tree": _plain_tree}
    return plain[kind](state)


# --------------------------------------------- the definitions in 64 bits --

def _spun(x, positions, frequencies, amplitude, interleaved, back=False):
    """The pairs as complex numbers, each times amplitude * exp(i * angle)."""
    x = x.double()
    n = 2 * frequencies.numel()
    pairs = x[..., :n].unflatten(-1, (n // 2, 2)) if interleaved else x[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2)
    angle = positions.double()[..., None, None] * frequencies
    z = torch.complex(pairs[..., 0], pairs[..., 1]) * torch.polar(torch.full_like(angle, amplitude), -angle if back else angle)
    z = torch.view_as_real(z)
    z = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., n:]), -1)


def _stored(x, codes):
    """What a row's codes stand for: the nearest of the type's numbers, scaled by the row's largest."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    top = torch.where(top > 0, top, torch.full_like(top, TOP[codes]))
    scale, y = top / TOP[codes], x * TOP[codes] / top
    if codes == "int8":
        return y.round() * scale
    exponent = torch.frexp(y)[1].clamp(min=-5) - 1  # floor(log2|y|), at least -6
    step = torch.exp2((exponent - 3).double())
    return (y / step).round() * step * scale


def _tokens(s, b, n):
    """K and V [Hkv, n, D] of sequence b's first n tokens, in 64 bits."""
    pages = s["table"][b, :max(1, -(-n // PAGE))].long()
    k, v = s["k"], s["v"]
    if s["codes"] == "none":
        k = torch.cat(list(k[pages].double().unbind(2)), -1)  # [pages, Hkv, 64, D]
        v = v[pages].double().mT
    else:
        k, v = (x.view(torch.uint8)[pages].view(CODES[s["codes"]]).double() for x in (k, v))
        k = torch.cat(list(k.unbind(2)), -1) * s["k_scale"][pages].double().unsqueeze(-1)
        v = torch.cat(list(v.unbind(2)), -1).mT * s["v_scale"][pages].double().unsqueeze(-1)
    return (x.transpose(0, 1).flatten(1, 2)[:, :n] for x in (k, v))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        how = (s["positions"], s["frequencies"], s["amplitude"], s["interleaved"])
        out = {"q": _spun(s["q"], *how), "k": _spun(s["k"], *how)}
        if case["grad"]:
            out["dq"], out["dk"] = _spun(s["dq"], *how, back=True), _spun(s["dk"], *how, back=True)
        return out
    B, Hq, Hkv, D = case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "write":
        out, k_new = {}, s["k_new"]
        if case["rotate"]:
            how = (s["positions"], s["frequencies"], s["amplitude"], False)
            out["q"], k_new = _spun(s["q"], *how), _spun(k_new, *how)
        k_new, v_new = _stored(k_new, case["codes"]), _stored(s["v_new"], case["codes"])
        out["k"] = torch.zeros((B, Hkv, s["length"], D), dtype=torch.float64, device="cuda")
        out["v"] = torch.zeros_like(out["k"])
        for b, c in enumerate(_contexts(case)):
            first = 0
            if case["read_all"] and c:
                out["k"][b, :, :c], out["v"][b, :, :c] = _tokens(s, b, c)
                first = c
            out["k"][b, :, first:first + case["new"]] = k_new[b].transpose(0, 1)
            out["v"][b, :, first:first + case["new"]] = v_new[b].transpose(0, 1)
        return out
    decode = case["kind"] == "decode"
    T = 1 if decode else case["drafts"]
    q = s["q"].double().view(B, T, Hkv, Hq // Hkv, D)
    out = torch.zeros((B, T, Hq, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.float64, device="cuda")
    counts = [0] * B if decode else _draft_counts(case)
    for b, c in enumerate(_contexts(case)):
        n = 1 if decode else counts[b]
        if c + counts[b] == 0:
            continue
        k, v = _tokens(s, b, c + counts[b])
        score = torch.matmul(q[b, :n].permute(1, 0, 2, 3).reshape(Hkv, -1, D), k.mT.contiguous()) * D ** -0.5
        score = score.view(Hkv, n, -1, c + counts[b])
        if not decode:
            tree = s["tree"][b, :n, :n] if s["tree"] is not None else torch.ones((n, n), device="cuda").tril().bool()
            score[..., c:].masked_fill_(~tree[None, :, None, :], -math.inf)
        l = torch.logsumexp(score, -1)
        p = torch.exp(score - l.unsqueeze(-1)).flatten(1, 2)
        out[b, :n] = torch.matmul(p, v.contiguous()).view(Hkv, n, -1, D).transpose(0, 1).reshape(n, Hq, D)
        lse[b, :n] = l.transpose(0, 1).reshape(n, Hq)
    return {"out": out[:, 0], "lse": lse[:, 0]} if decode else {"out": out, "lse": lse}
