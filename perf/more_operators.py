"""Measured operators of a paged cache whose keys and values are held in 4 bits.

Kinds (key "kind" of a case)
    rope       norm, rotation and the quantised cache write (ops.rope_store_kv4)
    store      the quantised cache write of rows as they are (ops.store_kv4)
    load       rows of the cache read back (ops.load_kv4)
    attention  attention over the cache (ops.paged_attention_kv4)

A cache is uint8 [pages, key heads, page * (hd / 2 + 4)]: of a page and head first the codes of its tokens (two channels a byte, the even one in the low
half), then their scales and minima (bf16 pairs).  A row x of a head is held as codes floor((x - min) / scale + 1/2), scale = bf16((max - min) / 15).

Head counts and sizes are those of ssd_b200.synth.SHAPES (64 heads over 8 of 128, 32 over 8 of 64 or 128, 16 over 8 of 128) and odd groups; pages of 256
tokens are the framework's default, smaller ones are what other deployments use.  Lengths follow from the case, values from the seed."""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # the seven rows that one user's step verifies, 70B heads, one row of padding
        {"name": "rope_verify_7", "kind": "rope", "rows": 7, "pad": 1, "heads": 64, "kv_heads": 8, "dim": 128, "rot": 128, "page": 256, "norm": False},
        # seven rows for each of 64 users, heads of 16 over 8 with norms
        {"name": "rope_verify_b64", "kind": "rope", "rows": 448, "pad": 0, "heads": 16, "kv_heads": 8, "dim": 128, "rot": 128, "page": 256, "norm": True},
        # prompts of 16000 tokens in one pass
        {"name": "rope_prompts", "kind": "rope", "rows": 16000, "pad": 0, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "page": 256, "norm": False},
        # 300 rows of a model without rotation, an odd number of heads
        {"name": "store_300", "kind": "store", "rows": 300, "pad": 3, "kv_heads": 5, "dim": 128, "page": 16},
        # a prefill worker's cache taken over: 32003 tokens
        {"name": "store_handover", "kind": "store", "rows": 32003, "pad": 0, "kv_heads": 8, "dim": 128, "page": 256},
        # a short prefix read back for a prompt that goes on from it, heads of 64
        {"name": "load_prefix", "kind": "load", "rows": 1000, "kv_heads": 8, "dim": 64, "page": 64},
        # four contexts read back to be handed to an unquantised cache
        {"name": "load_contexts", "kind": "load", "rows": 64004, "kv_heads": 8, "dim": 128, "page": 256},
        # one token of one user with a short context
        {"name": "attention_short", "kind": "attention", "batch": 1, "ctx": 500, "q_len": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 256},
        # one token of one user with a long one
        {"name": "attention_one", "kind": "attention", "batch": 1, "ctx": 32000, "q_len": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 256},
        # one token for each of 48 users, 70B heads
        {"name": "attention_b48", "kind": "attention", "batch": 48, "ctx": 16000, "q_len": 1, "heads": 64, "kv_heads": 8, "dim": 128, "page": 256},
        # eight users, seven rows each (a step that verifies), 70B heads
        {"name": "attention_verify_b8", "kind": "attention", "batch": 8, "ctx": 16000, "q_len": 7, "heads": 64, "kv_heads": 8, "dim": 128, "page": 256},
        # a chunk of a prompt over what came before it
        {"name": "attention_chunk", "kind": "attention", "batch": 1, "ctx": 8000, "q_len": 512, "heads": 32, "kv_heads": 8, "dim": 64, "page": 64},
    ]


#: heads, heads of keys and values, size of a head
HEADS = [(64, 8, 128), (32, 8, 128), (32, 8, 64), (16, 8, 128), (4, 2, 64), (40, 8, 128), (6, 2, 64), (5, 1, 128), (8, 8, 128), (20, 4, 64)]
ROPE_HEADS = [(64, 8, 128), (32, 8, 128), (16, 8, 128), (4, 2, 64), (40, 8, 128), (6, 2, 64), (5, 1, 128), (12, 4, 64)]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))))

    kind = rng.choice(["rope", "store", "load", "attention", "attention"])
    page = rng.choice([16, 64, 80, 128, 256, 256])
    if kind == "rope":
        H, KV, dim = rng.choice(ROPE_HEADS)
        return {"kind": kind, "rows": log(1, 8000), "pad": rng.choice([0, 0, 1, 5]), "heads": H, "kv_heads": KV, "dim": dim, "rot": rng.choice([dim, dim, dim // 2]), "page": page,
                "norm": rng.random() < 0.5}
    KV, dim = rng.choice([1, 2, 4, 5, 8, 8]), rng.choice([64, 128])
    if kind == "store":
        return {"kind": kind, "rows": log(1, 16000), "pad": rng.choice([0, 0, 1, 5]), "kv_heads": KV, "dim": dim, "page": page}
    if kind == "load":
        return {"kind": kind, "rows": log(1, 40000), "kv_heads": KV, "dim": dim, "page": page}
    H, KV, dim = rng.choice(HEADS)
    q_len = rng.choice([1, 1, 1, rng.randint(2, 8), rng.randint(2, 8), log(9, 500)])
    # no more scores than the chunk's, no more keys than the largest batch's
    ctx = log(max(1, q_len), max(q_len, min(64000, 130_000_000 // (H * q_len))))
    batch = log(1, max(1, min(48, 48 * 16000 // ctx, 130_000_000 // (H * q_len * ctx))))
    return {"kind": kind, "batch": batch, "ctx": ctx, "q_len": q_len, "heads": H, "kv_heads": KV, "dim": dim, "page": page}


# ------------------------------------------------------------------------------------------------ inputs
def uneven(n, batch):
    """Lengths of a batch: n, and shorter ones down to about half of it."""
    return [max(1, n - (i * n) // (2 * batch) - 3 * (i > 0)) for i in range(batch)]


def lengths(case):
    return [max(n, case["q_len"]) for n in uneven(case["ctx"], case["batch"])]


def normal(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(BF)


def a_cache(g, pages, page, KV, hd):
    """A cache that is full of keys: normal values around a mean per channel, some channels larger than others, as keys are behind their projection."""
    codes = torch.empty(pages, KV, page * (hd // 2 + 4), dtype=torch.uint8, device=DEV)
    mean, size = 0.5 * torch.randn(KV, 1, hd, generator=g, device=DEV), 0.5 + torch.rand(KV, 1, hd, generator=g, device=DEV)
    step = max(1, (1 << 26) // (page * KV * hd))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = (torch.randn(n, KV, page, hd, generator=g, device=DEV) * size + mean).to(BF).float()
        lo, hi = x.amin(3, keepdim=True), x.amax(3, keepdim=True)
        s = ((hi - lo) / 15).to(BF)
        c = ((x - lo) / s.float()).round().clamp(0, 15).to(torch.uint8)
        codes[p:p + n, :, :page * hd // 2] = (c[..., 0::2] | c[..., 1::2] << 4).flatten(2)
        codes[p:p + n, :, page * hd // 2:] = torch.cat([s, lo.to(BF)], 3).view(torch.uint8).flatten(2)
    return codes


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    s = dict(case)
    kind, KV, hd, page = case["kind"], case["kv_heads"], case["dim"], case["page"]
    if kind in ("rope", "store"):
        M = case["rows"] + case["pad"]
        pages = -(-case["rows"] // page) + 2
        # rows of a pass lie one behind the other in pages of any order; padding has no slot
        order = torch.randperm(pages, generator=g, device=DEV)[:, None] * page + torch.arange(page, device=DEV)
        slots = order.flatten()[5:5 + M].to(torch.int32)
        slots[case["rows"]:] = -1
        s["slots"] = slots.contiguous()
        s["k_cache"], s["v_cache"] = (torch.zeros(pages, KV, page * (hd // 2 + 4), dtype=torch.uint8, device=DEV) for _ in range(2))
        if kind == "store":
            s["k"], s["v"] = normal(g, M, KV, hd), normal(g, M, KV, hd, std=0.3)
            return s
        H, rot, top = case["heads"], case["rot"], 32768
        s["qkv"] = normal(g, M, (H + 2 * KV) * hd)
        s["positions"] = 7 + seed % 1000 + torch.arange(M, device=DEV)
        inv = 1.0 / 500000.0 ** (torch.arange(0, rot, 2, dtype=F64, device=DEV) / rot)
        angle = torch.arange(top, dtype=F64, device=DEV)[:, None] * inv
        s["angles"] = torch.cat([angle.cos(), angle.sin()], 1).to(F32)
        s["q_norm"], s["k_norm"] = (1 + 0.2 * normal(g, hd) for _ in range(2)) if case["norm"] else (None, None)
        return s
    if kind == "load":
        pages = -(-case["rows"] // page) + 2
        order = torch.randperm(pages, generator=g, device=DEV)[:, None] * page + torch.arange(page, device=DEV)
        s["slots"] = order.flatten()[:case["rows"]].to(torch.int32).contiguous()
        s["k_cache"], s["v_cache"] = a_cache(g, pages, page, KV, hd), a_cache(g, pages, page, KV, hd)
        return s
    lens = lengths(case)
    used = torch.tensor([-(-n // page) for n in lens], device=DEV)
    pages = int(used.sum()) + 2
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    at = torch.arange(int(used.max()), device=DEV)
    first = used.cumsum(0) - used
    s["table"] = torch.where(at < used[:, None], perm[(first[:, None] + at).clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["q"] = normal(g, case["batch"] * case["q_len"], case["heads"], hd)
    s["k_cache"], s["v_cache"] = a_cache(g, pages, page, KV, hd), a_cache(g, pages, page, KV, hd)
    s["scale"] = hd ** -0.5
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return run_own(s)
    return {"rope": plain_rope, "store": plain_store, "load": plain_load, "attention": plain_attention}[s["kind"]](s)


def run_own(s):
    from ssd_b200 import ops
    kind = s["kind"]
    if kind == "rope":
        q, k, v = ops.rope_store_kv4(s["qkv"], s["positions"], s["slots"], s["angles"], s["k_cache"], s["v_cache"], s["heads"], s["kv_heads"], s["dim"], s["q_norm"], s["k_norm"], 1e-6,
                                     values=True)
        return {"q": q, "k": k, "v": v, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if kind == "store":
        k, v = ops.store_kv4(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], values=True)
        return {"k": k, "v": v, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if kind == "load":
        k, v = ops.load_kv4(s["k_cache"], s["v_cache"], s["slots"], s["dim"])
        return {"k": k, "v": v}
    return {"out": ops.paged_attention_kv4(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["q_len"], s["scale"])}


def parts(cache, hd):
    """Views of a cache: codes [pages, KV, page, hd / 2], scales and minima [pages, KV, page, 2]."""
    page = cache.shape[2] // (hd // 2 + 4)
    return cache[:, :, :page * hd // 2].unflatten(2, (page, hd // 2)), cache[:, :, page * hd // 2:].view(BF).unflatten(2, (page, 2))


def quantise(x, cache, slots):
    """Rows [M, KV, hd] of bf16 into their slots; the values that then stand there."""
    hd = x.shape[2]
    codes, pairs = parts(cache, hd)
    page = codes.shape[2]
    x = x.to(F64)   # a quotient that is a code and a half goes up: the division has to be exact there
    lo, hi = x.amin(2, keepdim=True), x.amax(2, keepdim=True)
    scale = ((hi - lo) / 15).to(BF)
    c = torch.where(scale > 0, torch.floor((x - lo) / scale.to(F64) + 0.5), 0.0).to(torch.uint8)
    keep = (slots >= 0) & (slots < cache.shape[0] * page)
    at = slots[keep].long()
    codes[at // page, :, at % page] = (c[..., 0::2] | c[..., 1::2] << 4)[keep]
    pairs[at // page, :, at % page] = torch.cat([scale, lo.to(BF)], 2)[keep]
    return (scale.float() * c.float() + lo.float()).to(BF)


def plain_rope(s):
    H, KV, hd, half = s["heads"], s["kv_heads"], s["dim"], s["rot"] // 2
    M = s["qkv"].shape[0]
    x = s["qkv"].view(M, H + 2 * KV, hd)
    at = s["angles"][s["positions"]][:, None]

    def turned(y, w):
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.to(y.dtype)
        c, sn = at[..., :half].to(y.dtype), at[..., half:].to(y.dtype)
        a, b = y[..., :half], y[..., half:2 * half]
        return torch.cat([a * c - b * sn, b * c + a * sn, y[..., 2 * half:]], -1).to(BF)

    q = turned(x[:, :H].float(), s["q_norm"]).reshape(M, H * hd)
    k = quantise(turned(x[:, H:H + KV].to(F64), s["k_norm"]), s["k_cache"], s["slots"])   # (the rounding of a key decides its code next to a border)
    v = quantise(x[:, H + KV:], s["v_cache"], s["slots"])
    return {"q": q, "k": k, "v": v, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def plain_store(s):
    return {"k": quantise(s["k"], s["k_cache"], s["slots"]), "v": quantise(s["v"], s["v_cache"], s["slots"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def values(codes, pairs):
    """Values in fp32 of codes [..., hd / 2] and their scales and minima [..., 2]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return c * pairs[..., :1].float() + pairs[..., 1:].float()


def plain_load(s):
    out = {}
    for name in ("k", "v"):
        codes, pairs = parts(s[name + "_cache"], s["dim"])
        at, page = s["slots"].long(), codes.shape[2]
        out[name] = values(codes[at // page, :, at % page], pairs[at // page, :, at % page]).to(BF)
    return out


def plain_attention(s):
    B, Q, KV, hd, H = s["lens"].numel(), s["q_len"], s["kv_heads"], s["dim"], s["heads"]
    lens, pages = s["lens"].long(), s["table"].long().clamp(min=0)
    k, v = (values(*(x[pages] for x in parts(s[n + "_cache"], hd))).transpose(1, 2).flatten(2, 3) for n in "kv")   # [B, KV, N, hd]
    q = s["q"].float().view(B, Q, KV, -1, hd).permute(0, 2, 1, 3, 4).reshape(B, KV, -1, hd)
    pos = torch.arange(k.shape[2], device=DEV)
    limit = lens[:, None] - Q + torch.arange(Q, device=DEV).repeat_interleave(H // KV)   # [B, rows]
    seen = (pos <= limit[..., None])[:, None]
    x = torch.where(seen, q @ k.transpose(2, 3) * s["scale"], -math.inf)
    top = x.amax(3, keepdim=True)
    e = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    out = e @ torch.where((pos < lens[:, None])[:, None, :, None], v, 0.0) / e.sum(3, keepdim=True).clamp(min=1e-30)
    return {"out": out.view(B, KV, Q, -1, hd).permute(0, 2, 1, 3, 4).reshape(B * Q, -1).to(BF)}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": exact_rope, "store": exact_store, "load": exact_load, "attention": exact_attention}[case["kind"]](s)


def held(x, cache, slots):
    """What stands for rows x in the cache, and the cache, from the definition: a code is the number of borders that a value has reached."""
    M, KV, hd = x.shape
    page = cache.shape[2] // (hd // 2 + 4)
    x = x.to(F64)
    lo = x.min(2).values
    scale = ((x.max(2).values - lo) / 15).to(BF)
    width = scale.to(F64)
    c = torch.zeros(M, KV, hd, dtype=torch.int64, device=DEV)
    for k in range(15):
        c += ((x - lo[..., None] >= (k + 0.5) * width[..., None]) & (width[..., None] > 0)).long()
    value = width[..., None] * c + lo[..., None]
    out = cache.clone()
    raw = out.flatten(0, 1)
    byte = (c[..., ::2] + 16 * c[..., 1::2]).to(torch.uint8)
    two = torch.stack([scale, lo.to(BF)], 2).view(torch.uint8)   # [M, KV, 4]
    there = slots.long() >= 0
    slot = slots.long()[there]
    for h in range(KV):
        row = (slot // page * KV + h)[:, None]
        raw[row, (slot % page * (hd // 2))[:, None] + torch.arange(hd // 2, device=DEV)] = byte[there, h]
        raw[row, (page * (hd // 2) + slot % page * 4)[:, None] + torch.arange(4, device=DEV)] = two[there, h]
    return value, out


def exact_rope(s):
    H, KV, hd, rot = s["heads"], s["kv_heads"], s["dim"], s["rot"]
    x = s["qkv"].to(F64).unflatten(1, (H + 2 * KV, hd))
    q, k, v = x.split([H, KV, KV], 1)
    rows = s["angles"][s["positions"]].to(F64)
    turn = torch.complex(rows[:, :rot // 2].contiguous(), rows[:, rot // 2:].contiguous())

    def turned(y, w):
        if w is not None:
            y = y / (y.pow(2).sum(2, keepdim=True) / hd + 1e-6).sqrt() * w.to(F64)
        z = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * turn[:, None]
        return torch.cat([z.real, z.imag, y[..., rot:]], 2)

    kv, kc = held(turned(k, s["k_norm"]).to(BF), s["k_cache"], s["slots"])
    vv, vc = held(v, s["v_cache"], s["slots"])
    return {"q": turned(q, s["q_norm"]).flatten(1), "k": kv, "v": vv, "k_cache": kc, "v_cache": vc}


def exact_store(s):
    (k, kc), (v, vc) = held(s["k"], s["k_cache"], s["slots"]), held(s["v"], s["v_cache"], s["slots"])
    return {"k": k, "v": v, "k_cache": kc, "v_cache": vc}


def rows_of(cache, slots, hd):
    """Values in 64 bits [n, KV, hd] of slots."""
    page = cache.shape[2] // (hd // 2 + 4)
    out = torch.empty(slots.numel(), cache.shape[1], hd, dtype=F64, device=DEV)
    block, off = slots.long() // page, slots.long() % page
    for h in range(cache.shape[1]):
        at = block * cache.stride(0) + h * cache.stride(1)
        byte = cache.flatten()[(at + off * (hd // 2))[:, None] + torch.arange(hd // 2, device=DEV)].to(F64)
        two = cache.flatten()[(at + page * (hd // 2) + 4 * off)[:, None] + torch.arange(4, device=DEV)].view(BF).to(F64)
        out[:, h, 1::2] = torch.floor(byte / 16)
        out[:, h, ::2] = byte - 16 * out[:, h, 1::2]
        out[:, h] = out[:, h] * two[:, :1] + two[:, 1:]
    return out


def exact_load(s):
    return {n: rows_of(s[n + "_cache"], s["slots"], s["dim"]) for n in "kv"}


def exact_attention(s):
    Q, KV, hd, page = s["q_len"], s["kv_heads"], s["dim"], s["page"]
    G, out = s["heads"] // KV, []
    for b, n in enumerate(s["lens"].tolist()):
        i = torch.arange(n, device=DEV)
        slots = s["table"][b].long()[i // page] * page + i % page
        k, v = rows_of(s["k_cache"], slots, hd), rows_of(s["v_cache"], slots, hd)
        q = s["q"][b * Q:(b + 1) * Q].to(F64).view(Q, KV, G, hd)
        x = torch.einsum("qhgd,nhd->hgqn", q, k) * s["scale"]
        x = x.masked_fill(i > torch.arange(n - Q, n, device=DEV)[:, None], -math.inf)
        out.append(torch.einsum("hgqn,nhd->qhgd", torch.softmax(x, -1), v).reshape(Q, -1))
    return {"out": torch.cat(out)}


# ------------------------------------------------------------------------------------------------ what one pass cannot do without
def work(case):
    kind, KV, hd = case["kind"], case["kv_heads"], case["dim"]
    row = 2 * KV * (hd // 2 + 4)   # bytes of a token's keys and values in the cache
    if kind in ("rope", "store"):
        n, M = case["rows"], case["rows"] + case["pad"]
        moved = M * 4 * KV * hd * 2 + n * row + 4 * M   # rows in, the values that stand for them out; codes; slots
        if kind == "store":
            return {"bytes": moved, "flops": 8 * M * 2 * KV * hd}
        H, rot = case["heads"], case["rot"]
        return {"bytes": moved + M * (4 * H * hd + 8) + min(M, 32768) * 4 * rot, "flops": M * (8 * 2 * KV * hd + (H + KV) * (3 * rot + (4 * hd if case["norm"] else 0)))}
    if kind == "load":
        return {"bytes": case["rows"] * (row + 4 + 4 * KV * hd), "flops": 4 * case["rows"] * KV * hd}
    lens, Q, H = lengths(case), case["q_len"], case["heads"]
    # keys that a query sees: all but the new tokens behind it
    pairs = sum(Q * n - Q * (Q - 1) // 2 for n in lens)
    return {"bytes": sum(lens) * row + len(lens) * Q * H * hd * 4 + 4 * sum(-(-n // case["page"]) for n in lens), "flops": 4 * pairs * H * hd}
