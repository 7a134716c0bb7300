"""Measured operators of the paged cache: what comes before and around attention when a step reads only a part of a long cache.

Kinds (key "kind" of a case)
    place      pages, positions and slots of a step's new tokens from the lengths of its requests (ops.place_tokens)
    rope       rotary positions with several axes, and the cache write (ops.rope_axes_store_kv)
    bounds     per span of keys the smallest and largest value of every channel (ops.span_bounds)
    select     the spans of a long cache that a query can score highest with (ops.select_spans)
    attention  attention over the selected spans only (ops.span_attention)

Head counts and sizes are those of ssd_b200.synth.SHAPES (64 heads over 8 of 128, 32 over 8 of 64 or 128, 16 over 8 of 128) and odd groups; pages
of 256 tokens are the framework's default, smaller ones are what other deployments use.  Lengths follow from the case, values from the seed."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # a step that verifies seven rows for each of 64 users, as it runs between two decoding steps
        {"name": "place_verify_b64", "kind": "place", "batch": 64, "ctx": 8000, "new": 7, "rows": 512, "page": 256, "short": 0},
        # admission of 48 prompts of uneven lengths, more than the pass has room for
        {"name": "place_prompts", "kind": "place", "batch": 48, "ctx": 0, "new": 2100, "rows": 65536, "page": 16, "short": 0},
        # the seven rows that one user's step verifies, 70B heads
        {"name": "rope_verify_7", "kind": "rope", "rows": 7, "pad": 1, "heads": 64, "kv_heads": 8, "dim": 128, "rot": 128, "axes": 3, "interleaved": False, "norm": False},
        # a prompt of images (time, height, width) and text, an odd number of rows
        {"name": "rope_image_prompt", "kind": "rope", "rows": 4003, "pad": 0, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "axes": 3, "interleaved": False, "norm": False},
        # a video prompt, axes that take turns along the frequencies, norms per head in front
        {"name": "rope_video_prompt", "kind": "rope", "rows": 16000, "pad": 0, "heads": 16, "kv_heads": 8, "dim": 128, "rot": 128, "axes": 3, "interleaved": True, "norm": True},
        # bounds behind a step that wrote seven tokens for each of 64 users
        {"name": "bounds_verify_b64", "kind": "bounds", "batch": 64, "ctx": 8000, "new": 7, "kv_heads": 8, "dim": 128, "page": 256, "span": 32},
        # bounds of four long prompts
        {"name": "bounds_prompts", "kind": "bounds", "batch": 4, "ctx": 16001, "new": 16001, "kv_heads": 8, "dim": 128, "page": 256, "span": 32},
        # one user with a long context
        {"name": "select_one", "kind": "select", "batch": 1, "ctx": 32000, "q_len": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 256, "span": 32, "count": 64},
        # 24 users with contexts up to 64000 tokens, 70B heads
        {"name": "select_b24", "kind": "select", "batch": 24, "ctx": 64000, "q_len": 1, "heads": 64, "kv_heads": 8, "dim": 128, "page": 256, "span": 32, "count": 128},
        # one token of one user over 64 spans
        {"name": "attention_one", "kind": "attention", "batch": 1, "ctx": 32000, "q_len": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 256, "span": 32, "count": 64},
        # eight users, seven rows each (a step that verifies), 70B heads
        {"name": "attention_verify_b8", "kind": "attention", "batch": 8, "ctx": 16000, "q_len": 7, "heads": 64, "kv_heads": 8, "dim": 128, "page": 256, "span": 32, "count": 128},
        # one token for each of 48 users
        {"name": "attention_b48", "kind": "attention", "batch": 48, "ctx": 16000, "q_len": 1, "heads": 64, "kv_heads": 8, "dim": 128, "page": 256, "span": 32, "count": 128},
    ]


#: heads, heads of keys and values, size of a head
HEADS = [(64, 8, 128), (32, 8, 128), (32, 8, 64), (16, 8, 128), (4, 2, 64), (40, 8, 128), (6, 2, 64), (5, 1, 128)]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))))

    kind = rng.choice(["place", "rope", "bounds", "select", "attention"])
    page = rng.choice([16, 64, 128, 256, 256])
    if kind == "place":
        new = rng.choice([1, 1, rng.randint(2, 8), log(9, 3000)])
        batch = log(1, min(512, 65536 // new))
        # one in three has fewer rows than its requests ask for, one in three fewer pages
        rows = max(1, round(batch * new * rng.choice([0.6, 1, 1.25])))
        return {"kind": kind, "batch": batch, "ctx": rng.choice([0, log(1, 20000)]), "new": new, "rows": rows, "page": page, "short": rng.choice([0, 0, 1])}
    H, KV, dim = rng.choice(HEADS)
    if kind == "rope":
        rows = log(1, 8000)
        return {"kind": kind, "rows": rows, "pad": rng.choice([0, 0, 1, 5]), "heads": H, "kv_heads": KV, "dim": dim, "rot": rng.choice([dim, dim, dim // 2]),
                "axes": rng.choice([1, 2, 3, 3, 4]), "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5}
    span = rng.choice([s for s in (16, 32, 64, 128, 256) if page % s == 0])
    if kind == "bounds":
        ctx = log(17, 16000)
        new = rng.choice([1, rng.randint(2, 8), ctx])
        return {"kind": kind, "batch": log(1, max(1, min(64, 64000 // ctx))), "ctx": ctx, "new": min(new, ctx), "kv_heads": KV, "dim": dim, "page": page, "span": span}
    q_len = rng.choice([1, 1, 1, rng.randint(2, 8)])
    if kind == "select":
        ctx = log(24 * span, 64000)   # fewer spans than asked for are all taken, whatever their scores
        batch = log(1, max(1, min(32, 24 * 64000 // ctx, 24 * 2000 * span // ctx)))
        return {"kind": kind, "batch": batch, "ctx": ctx, "q_len": q_len, "heads": H, "kv_heads": KV, "dim": dim, "page": page, "span": span, "count": log(5, max(5, min(128, ctx // (3 * span))))}
    ctx = log(100, 16000)
    count = log(3, max(3, 4096 // span))
    batch = log(1, max(1, min(48, 48 * 4096 // (count * span))))
    return {"kind": kind, "batch": batch, "ctx": ctx, "q_len": q_len, "heads": H, "kv_heads": KV, "dim": dim, "page": page, "span": span, "count": count}


# ------------------------------------------------------------------------------------------------ inputs
def uneven(n, batch):
    """Lengths of a batch: n, and shorter ones down to about half of it."""
    return [max(1, n - (i * n) // (2 * batch) - 3 * (i > 0)) for i in range(batch)] if n else [0] * batch


def make_gen(seed, salt=0):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + salt)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def normal(g, *shape, std=1.0):
    out = torch.empty(*shape, dtype=BF, device=DEV)
    step = max(1, (1 << 27) // max(1, math.prod(shape[1:])))
    for r in range(0, shape[0], step):
        n = min(step, shape[0] - r)
        out[r:r + n] = torch.randn(n, *shape[1:], generator=g, device=DEV) * std
    return out


def tables(g, lens, page, spare=0):
    """Block tables of sequences of these lengths over pages in a random order, -1 behind the last; the pages left over, as a list of free ones."""
    used = [-(-n // page) for n in lens]
    total = sum(used) + spare
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    width = max(1, max(used))
    at = torch.arange(width, device=DEV)
    count = torch.tensor(used, device=DEV)
    first = count.cumsum(0) - count
    pick = (first[:, None] + at).clamp(max=total - 1)
    return torch.where(at < count[:, None], perm[pick], torch.full_like(perm[:1], -1)).contiguous(), perm[sum(used):].contiguous(), total


def prepare(case, seed):
    g = make_gen(seed, 11)
    s = dict(case)
    kind = case["kind"]
    if kind == "place":
        B, page = case["batch"], case["page"]
        ctx, new = uneven(case["ctx"], B), uneven(case["new"], B)
        turn = seed % B   # another order of the same requests
        ctx, new = ctx[turn:] + ctx[:turn], new[-turn:] + new[:-turn] if turn else new
        need = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(ctx, new))
        left = max(1, need // 2 if case["short"] else need + 5)
        t, free, total = tables(g, ctx, page, left + 40)
        free = free[:left + 3]
        width = max(-(-(c + n) // page) for c, n in zip(ctx, new))
        s["table"] = torch.full((B, width + 1), -1, dtype=torch.int32, device=DEV)
        s["table"][:, :t.shape[1]] = t[:, :width + 1]
        s.update(ctx=ints(ctx), new=ints(new), free=free, used=ints([3]), pages=total)
        return s
    if kind == "rope":
        M, H, KV, hd, rot, A = case["rows"] + case["pad"], case["heads"], case["kv_heads"], case["dim"], case["rot"], case["axes"]
        page, top = 256, 32768
        pages = -(-case["rows"] // page) + 2
        s["qkv"] = normal(g, M, (H + 2 * KV) * hd)
        # a grid of patches: rows of 40, pictures of 30 rows, behind a text that ends at another place for every seed
        i = torch.arange(M, device=DEV)
        start = 7 + seed % 1000
        grid = [start + i // 1200, start + (i // 40) % 30, start + i % 40, start + i]
        s["positions"] = torch.stack(grid[:A] if A > 1 else grid[3:]).contiguous()
        inv = 1.0 / 500000.0 ** (torch.arange(0, rot, 2, dtype=F64, device=DEV) / rot)
        angle = torch.arange(top, dtype=F64, device=DEV)[:, None] * inv
        s["angles"] = torch.cat([angle.cos(), angle.sin()], 1).to(F32)
        s["axis_of"] = axis_of(rot // 2, A, case["interleaved"])
        s["axis_index"] = torch.tensor(s["axis_of"], device=DEV)
        slots = torch.randperm(pages * page, generator=g, device=DEV)[:M].to(torch.int32)
        slots[case["rows"]:] = -1
        s["slots"] = slots
        s["k_cache"], s["v_cache"] = (torch.zeros(pages, page, KV, hd, dtype=BF, device=DEV) for _ in range(2))
        s["q_norm"], s["k_norm"] = (1 + 0.2 * normal(g, hd) for _ in range(2)) if case["norm"] else (None, None)
        return s
    B, KV, hd, page, span = (case[k] for k in ("batch", "kv_heads", "dim", "page", "span"))
    lens = [max(n, case.get("q_len", 1), case.get("new", 1)) for n in uneven(case["ctx"], B)]
    s["table"], _, pages = tables(g, lens, page, 2)
    s["lens"] = ints(lens)
    s["pages"] = pages
    if kind == "bounds":
        s["k_cache"] = normal(g, pages, page, KV, hd)
        s["bounds"] = torch.zeros(pages, page // span, KV, 2, hd, dtype=BF, device=DEV)
        return s
    H, Q = case["heads"], case["q_len"]
    s["q"] = normal(g, B * Q, H, hd)
    if kind == "select":
        # bounds as spans of keys around a mean have them: about two deviations to each side
        mid, half = normal(g, pages, page // span, KV, hd, std=0.4), normal(g, pages, page // span, KV, hd, std=0.3)
        s["bounds"] = torch.stack([mid - 2 - half.abs(), mid + 2 + half.abs()], 3).contiguous()
        return s
    s["k_cache"], s["v_cache"] = normal(g, pages, page, KV, hd), normal(g, pages, page, KV, hd)
    # lists as a selection makes them: the first and the last span and others between, ascending
    n, count = [-(-x // span) for x in lens], case["count"]
    width = max(n)
    rank = torch.rand(B, KV, width, generator=g, device=DEV)
    at = torch.arange(width, device=DEV)
    last = torch.tensor(n, device=DEV)[:, None, None]
    rank = torch.where((at == 0) | (at >= last - 1), torch.full_like(rank, 2.0), rank)
    rank = torch.where(at < last, rank, torch.full_like(rank, -1.0))
    best, pick = rank.topk(min(count, width), dim=2)
    pick = torch.where(best >= 0, pick, torch.full_like(pick, width)).sort(2).values
    pick = torch.where(pick < width, pick, torch.full_like(pick, -1))
    s["spans"] = torch.nn.functional.pad(pick, (0, count - pick.shape[2]), value=-1).to(torch.int32).contiguous()
    s["scale"] = hd ** -0.5
    return s


def axis_of(n, axes, interleaved):
    """The axis that each of n frequencies turns by: sections one behind the other (the first half as long as the others), or in turns."""
    if interleaved:
        return [i % axes for i in range(n)]
    first = max(1, n // (2 * axes - 1)) if axes > 1 else n
    return [0 if i < first else 1 + min(axes - 2, (i - first) * (axes - 1) // (n - first)) for i in range(n)]


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return run_own(s)
    return {"place": plain_place, "rope": plain_rope, "bounds": plain_bounds, "select": plain_select, "attention": plain_attention}[s["kind"]](s)


def run_own(s):
    from ssd_b200 import ops
    kind = s["kind"]
    if kind == "place":
        positions, slots, seqs, cu, lens, used = ops.place_tokens(s["ctx"], s["new"], s["table"], s["free"], s["used"], s["rows"], s["page"], s["pages"])
        return {"positions": positions, "slots": slots, "seqs": seqs, "cu": cu, "lens": lens, "used": used, "table": s["table"]}
    if kind == "rope":
        q = ops.rope_axes_store_kv(s["qkv"], s["positions"], s["axis_of"], s["slots"], s["angles"], s["k_cache"], s["v_cache"], s["heads"], s["kv_heads"], s["dim"],
                                   s["q_norm"], s["k_norm"], 1e-6)
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if kind == "bounds":
        ops.span_bounds(s["bounds"], s["k_cache"], s["table"], s["lens"], s["new"])
        return {"bounds": s["bounds"]}
    if kind == "select":
        return {"spans": ops.select_spans(s["q"], s["bounds"], s["table"], s["lens"], s["q_len"], s["page"], s["count"])}
    return {"out": ops.span_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["spans"], s["span"], s["q_len"], s["scale"])}


def plain_place(s):
    ctx, new, table, page, rows = s["ctx"].long(), s["new"].long(), s["table"], s["page"], s["rows"]
    B, width = table.shape
    used, F = s["used"].long(), s["free"].numel()
    ok = (ctx >= 0) & (new >= 0) & (ctx + new <= width * page)
    have = (ctx + page - 1) // page
    need = torch.where(ok, (ctx + new + page - 1) // page - have, 0)
    ok = ok & ((need == 0) | (used + need.cumsum(0) <= F))
    ok = ok & ((new == 0) | (torch.where(ok, new, 0).cumsum(0) <= rows))
    need, n = torch.where(ok, need, 0), torch.where(ok, new, 0)
    pages, ends = need.cumsum(0), n.cumsum(0)
    # pages handed out, in the order of the list
    k = torch.arange(F, device=DEV)
    b = torch.searchsorted(pages, k, right=True).clamp(max=B - 1)
    flat = torch.where(k < pages[-1], b * width + have[b] + k - (pages - need)[b], B * width)
    whole = torch.cat([table.flatten(), table.new_zeros(1)])
    whole[flat] = s["free"][(used + k).clamp(max=F - 1)]
    table.copy_(whole[:-1].view(B, width))
    # rows
    t = torch.arange(rows, device=DEV)
    b = torch.searchsorted(ends, t, right=True).clamp(max=B - 1)
    valid = t < ends[-1]
    pos = torch.where(valid, ctx[b] + t - (ends - n)[b], 0)
    at = table[b, pos // page].long()
    slot = torch.where(valid & (at >= 0) & (at < s["pages"]), at * page + pos % page, -1)
    cu = torch.cat([ends.new_zeros(1), ends])
    return {"positions": pos, "slots": slot.int(), "seqs": torch.where(valid, b, -1).int(), "cu": cu.int(), "lens": torch.where(ok, ctx + new, ctx).int(),
            "used": (used + pages[-1:]).int(), "table": table}


def plain_rope(s):
    H, KV, hd, half = s["heads"], s["kv_heads"], s["dim"], s["rot"] // 2
    M = s["qkv"].shape[0]
    x = s["qkv"].float().view(M, H + 2 * KV, hd)
    qk, v = x[:, :H + KV], x[:, H + KV:]
    if s["q_norm"] is not None:
        w = torch.cat([s["q_norm"].float().expand(H, hd), s["k_norm"].float().expand(KV, hd)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    at = s["positions"][s["axis_index"]].t()   # [M, half]
    f = torch.arange(half, device=DEV)
    c, sn = s["angles"][at, f][:, None], s["angles"][at, half + f][:, None]
    a, b = qk[..., :half], qk[..., half:2 * half]
    qk = torch.cat([a * c - b * sn, b * c + a * sn, qk[..., 2 * half:]], -1).to(BF)
    keep = s["slots"] >= 0
    to = s["slots"][keep].long()
    s["k_cache"].view(-1, KV, hd)[to] = qk[keep, H:]
    s["v_cache"].view(-1, KV, hd)[to] = v[keep].to(BF)
    return {"q": qk[:, :H].reshape(M, H * hd), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def plain_bounds(s):
    page, span, new = s["page"], s["span"], s["new"]
    lens = s["lens"].long()[:, None]
    at = (lens - new).clamp(min=0) // span + torch.arange((new + span - 2) // span + 1, device=DEV)   # [B, T]
    pos = at[..., None] * span + torch.arange(span, device=DEV)
    pages = s["table"].gather(1, (at * span // page).clamp(max=s["table"].shape[1] - 1)).long()
    k = s["k_cache"][pages.clamp(min=0)[..., None], pos % page].float()   # [B, T, span, KV, hd]
    seen = (pos < lens[..., None])[..., None, None]
    lo, hi = torch.where(seen, k, math.inf).amin(2), torch.where(seen, k, -math.inf).amax(2)
    keep = (at * span < lens) & (pages >= 0)
    s["bounds"][pages[keep], (at * span % page // span)[keep]] = torch.stack([lo, hi], 3).to(BF)[keep]
    return {"bounds": s["bounds"]}


def plain_select(s):
    page, span, count, Q = s["page"], s["span"], s["count"], s["q_len"]
    B, width = s["table"].shape
    KV, hd = s["kv_heads"], s["dim"]
    lens = s["lens"].long()[:, None]
    at = torch.arange(width * (page // span), device=DEV)
    pages = s["table"][:, at * span // page].long()   # [B, n]
    both = s["bounds"][pages.clamp(min=0), at * span % page // span].to(F64).permute(0, 2, 3, 4, 1)   # [B, KV, 2, hd, n]
    q = s["q"].to(F64).view(B, Q, KV, -1, hd).permute(0, 2, 1, 3, 4).reshape(B, KV, -1, hd)
    score = (q.clamp(max=0) @ both[:, :, 0] + q.clamp(min=0) @ both[:, :, 1]).amax(2)   # max(q lo, q hi) of every channel, summed
    n = (lens + span - 1) // span
    last = (Q + span - 2) // span + 1
    seen = ((at < n) & (pages >= 0))[:, None].expand_as(score)
    kept = ((at < 1) | (at >= n - last))[:, None] & seen
    score = torch.where(kept, math.inf, torch.where(seen, score, -math.inf))
    pick = score.sort(dim=2, descending=True, stable=True).indices[..., :count]
    pick = torch.where(seen.gather(2, pick), pick, at.numel()).sort(2).values
    pick = torch.where(pick < at.numel(), pick, -1)
    return {"spans": torch.nn.functional.pad(pick, (0, count - pick.shape[2]), value=-1).int()}


def plain_attention(s):
    page, span, Q, KV, hd = s["page"], s["span"], s["q_len"], s["kv_heads"], s["dim"]
    B = s["table"].shape[0]
    lens = s["lens"].long()
    named = s["spans"].long()[..., None].expand(-1, -1, -1, span).reshape(B, KV, -1)
    pos = named * span + torch.arange(span, device=DEV).repeat(s["spans"].shape[2])   # [B, KV, N]
    seen = (named >= 0) & (pos < lens[:, None, None])
    pos = torch.where(seen, pos, 0)
    pages = s["table"][torch.arange(B, device=DEV)[:, None, None], pos // page].long()
    head = torch.arange(KV, device=DEV)[:, None]
    k, v = (c[pages, pos % page, head].float() for c in (s["k_cache"], s["v_cache"]))   # [B, KV, N, hd]
    q = s["q"].float().view(B, Q, KV, -1, hd).permute(0, 2, 1, 3, 4).reshape(B, KV, -1, hd)
    limit = lens[:, None] - Q + torch.arange(Q, device=DEV).repeat_interleave(q.shape[2] // Q)   # [B, R]
    seen = seen[:, :, None] & (pos[:, :, None] <= limit[:, None, :, None])
    x = torch.where(seen, q @ k.transpose(2, 3) * s["scale"], -math.inf)
    top = x.amax(3, keepdim=True)
    e = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    out = e @ v / e.sum(3, keepdim=True).clamp(min=1e-30)
    return {"out": out.view(B, KV, Q, -1, hd).permute(0, 2, 1, 3, 4).reshape(B * Q, -1).to(BF)}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"place": exact_place, "rope": exact_rope, "bounds": exact_bounds, "select": exact_select, "attention": exact_attention}[case["kind"]](s)


def exact_place(s):
    page, rows, pages = s["page"], s["rows"], s["pages"]
    table, free, u = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy(), int(s["used"])
    positions, slots, seqs = np.zeros(rows, np.int64), np.full(rows, -1, np.int32), np.full(rows, -1, np.int32)
    cu, lens, at, stuck, full = [0], [], 0, False, False
    for b, (c, n) in enumerate(zip(s["ctx"].tolist(), s["new"].tolist())):
        need = -(-(c + n) // page) - -(-c // page)
        if need > 0 and (stuck or u + need > len(free)):
            stuck, n, need = True, 0, 0
        if n > 0 and (full or at + n > rows):
            full, n, need = True, 0, 0
        have = -(-c // page)
        table[b, have:have + need] = free[u:u + need]
        u += need
        p = np.arange(c, c + n)
        positions[at:at + n], seqs[at:at + n] = p, b
        named = table[b, p // page].astype(np.int64)
        slots[at:at + n] = np.where((named >= 0) & (named < pages), named * page + p % page, -1)
        at += n
        cu.append(at)
        lens.append(c + n)
    i32 = lambda v: torch.tensor(np.asarray(v, np.int32))  # noqa: E731
    return {"positions": torch.from_numpy(positions), "slots": i32(slots), "seqs": i32(seqs), "cu": i32(cu), "lens": i32(lens), "used": i32([u]), "table": i32(table)}


def exact_rope(s):
    H, KV, hd, rot = s["heads"], s["kv_heads"], s["dim"], s["rot"]
    x = s["qkv"].to(F64).unflatten(1, (H + 2 * KV, hd))
    q, k, v = x.split([H, KV, KV], 1)
    turn = torch.empty(x.shape[0], rot // 2, dtype=torch.complex128, device=DEV)
    for i, axis in enumerate(s["axis_of"]):
        rows = s["angles"][s["positions"][axis]].to(F64)
        turn[:, i] = torch.complex(rows[:, i], rows[:, rot // 2 + i])

    def turned(y, w):
        if w is not None:
            y = y / (y.pow(2).sum(2, keepdim=True) / hd + 1e-6).sqrt() * w.to(F64)
        z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * turn[:, None]
        return torch.cat([z.real, z.imag, y[..., rot:]], 2)

    kc, vc = torch.zeros_like(s["k_cache"], dtype=F64), torch.zeros_like(s["v_cache"], dtype=F64)
    n = s["rows"]
    kc.flatten(0, 1).index_copy_(0, s["slots"][:n].long(), turned(k, s["k_norm"])[:n])
    vc.flatten(0, 1).index_copy_(0, s["slots"][:n].long(), v[:n])
    return {"q": turned(q, s["q_norm"]).flatten(1), "k_cache": kc, "v_cache": vc}


def exact_bounds(s):
    page, span = s["page"], s["span"]
    out = s["bounds"].to(F64)
    for table, n in zip(s["table"].tolist(), s["lens"].tolist()):
        for i in range(max(0, n - s["new"]) // span, -(-n // span)):
            p, off = table[i * span // page], i * span % page
            keys = s["k_cache"][p, off:off + min(span, n - i * span)].to(F64)
            out[p, off // span, :, 0], out[p, off // span, :, 1] = keys.min(0).values, keys.max(0).values
    return {"bounds": out}


def exact_select(s):
    page, span, count, Q, KV = s["page"], s["span"], s["count"], s["q_len"], s["kv_heads"]
    out = np.full((len(s["lens"]), KV, count), -1, np.int32)
    for b, (table, length) in enumerate(zip(s["table"], s["lens"].tolist())):
        n, last = -(-length // span), -(-(Q - 1) // span) + 1
        i = torch.arange(n, device=DEV)
        both = s["bounds"][table[i * span // page].long(), i * span % page // span].to(F64)   # [n, KV, 2, hd]
        for h in range(KV):
            best = torch.full((n,), -math.inf, dtype=F64, device=DEV)
            for row in s["q"].view(len(s["lens"]), Q, KV, -1, s["dim"])[b, :, h].flatten(0, 1).to(F64):
                best = torch.maximum(best, torch.maximum(row * both[:, h, 0], row * both[:, h, 1]).sum(1))
            score = best.cpu().numpy()
            order = sorted(range(n), key=lambda j: (not (j < 1 or j >= n - last), -score[j], j))
            got = sorted(order[:count])
            out[b, h, :len(got)] = got
    return {"spans": torch.from_numpy(out)}


def exact_attention(s):
    page, span, Q, KV, hd = s["page"], s["span"], s["q_len"], s["kv_heads"], s["dim"]
    G, out = s["heads"] // KV, []
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // page)].long()
        k, v = (c[pages].flatten(0, 1)[:n].to(F64) for c in (s["k_cache"], s["v_cache"]))   # the whole context; what is not listed is masked
        listed_ = torch.zeros(KV, -(-n // span) + 1, dtype=torch.bool, device=DEV).scatter_(1, torch.where(s["spans"][b] < 0, -(-n // span), s["spans"][b]).long(), True)
        mask = listed_[:, :-1].repeat_interleave(span, 1)[:, :n]
        q = s["q"][b * Q:(b + 1) * Q].to(F64).view(Q, KV, G, hd)
        x = torch.einsum("qhgd,nhd->hgqn", q, k) * s["scale"]
        causal = torch.arange(n, device=DEV) <= torch.arange(n - Q, n, device=DEV)[:, None]
        x = x.masked_fill(~(mask[:, None, None] & causal), -math.inf)
        p = torch.nan_to_num(torch.softmax(x, -1))
        out.append(torch.einsum("hgqn,nhd->qhgd", p, v).reshape(Q, -1))
    return {"out": torch.cat(out)}


# ------------------------------------------------------------------------------------------------ what one pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "place":
        B, page = case["batch"], case["page"]
        ctx, new = uneven(case["ctx"], B), uneven(case["new"], B)
        rows = min(sum(new), case["rows"])
        pages = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(ctx, new)) // (2 if case["short"] else 1)
        touched = sum(-(-(c + n) // page) - c // page for c, n in zip(ctx, new))
        # lengths in, offsets and lengths out; position, slot and sequence of a row; a page read from the list and written to a table, or read from it
        return {"bytes": 16 * B + 16 * case["rows"] + 8 * pages + 4 * max(0, touched - pages), "flops": 4 * rows}
    H, KV, hd = case.get("heads", 0), case["kv_heads"], case["dim"]
    if kind == "rope":
        M = case["rows"] + case["pad"]
        moved = M * (H + 2 * KV) * hd * 4 - case["pad"] * 2 * KV * hd * 4   # 2 bytes in, 2 out; padded rows have no keys and values
        return {"bytes": moved + M * (8 * case["axes"] + 4) + min(M, 32768) * 4 * case["rot"] // (1200 if case["axes"] > 1 else 1),
                "flops": M * (H + KV) * (3 * case["rot"] + (4 * hd if case["norm"] else 0))}
    B, page, span = case["batch"], case["page"], case["span"]
    lens = [max(n, case.get("q_len", 1), case.get("new", 1)) for n in uneven(case["ctx"], B)]
    if kind == "bounds":
        spans = sum(-(-n // span) - (n - case["new"]) // span for n in lens)
        keys = sum(n - (n - case["new"]) // span * span for n in lens)
        return {"bytes": keys * KV * hd * 2 + spans * KV * hd * 4 + 8 * B, "flops": 2 * keys * KV * hd}
    Q, count = case["q_len"], case["count"]
    rows = B * Q * H
    if kind == "select":
        spans = sum(-(-n // span) for n in lens)
        return {"bytes": spans * KV * hd * 4 + rows * hd * 2 + B * KV * count * 4 + 4 * sum(-(-n // page) for n in lens), "flops": 4 * spans * Q * H * hd}
    keys = sum(min(n, count * span) for n in lens)
    return {"bytes": keys * KV * hd * 4 + rows * hd * 4 + B * KV * count * 4, "flops": 4 * keys * Q * H * hd}
