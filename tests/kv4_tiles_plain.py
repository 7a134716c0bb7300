"""Attention over a paged cache held in 4 bits with more than sixteen query rows to a key head, in 64 bits, and how far a kernel on tiles may be off: its own roundings, none of the streaming kernel's."""
import torch

from tests import kv4_plain as plain

BF, F64 = torch.bfloat16, torch.float64


def once(v):
    """v (64 bits) to bf16 in one rounding, as 64 bits: fp32 toward zero with the last bit set where it is not v, then bf16."""
    f = v.float()
    away = f.double().abs() > v.abs()
    bits = f.view(torch.int32) - away.int()
    return torch.where(f.double() == v, f, (bits | 1).view(torch.float32)).to(BF).double()


def attend(q, k, v, seen, scale, k_is=None, v_is=None):
    """Rows q [R, hd] over keys and values [n, hd], all in 64 bits; seen [R, n].  k_is, v_is: what the kernel has in their place.  -> out, slack."""
    k_is, v_is = k if k_is is None else k_is, v if v_is is None else v_is
    R, hd = q.shape
    some = seen.any(1, keepdim=True)
    x = (q @ k.t() * scale).masked_fill(~seen, -torch.inf)
    p = torch.where(some, torch.softmax(torch.where(some, x, 0.0), 1), 0.0).masked_fill(~seen, 0.0)
    out, size = p @ v, p @ v_is.abs()
    steps = -(-int(seen.sum(1).max()) // 16)
    terms = (q.abs() @ k_is.abs().t() * abs(scale)).masked_fill(~seen, 0.0).amax(1, keepdim=True)
    # a score: hd / 16 sums of sixteen exact products in fp32, each off by 2^-22 of the terms' size; scale and unit, 2^-22 of it; difference from the reference, exponential, raised references 2^-18; and what its
    # key is off by.  A weight is off by as much as its score, and so is their sum.
    score = terms * (hd / 16 * 2 ** -22 + 2 ** -22) + 2 ** -18 + (q.abs() @ (k - k_is).abs().t() * abs(scale)).masked_fill(~seen, 0.0).amax(1, keepdim=True)
    # a weight is rounded to bf16 once (no score of these tests passes the largest of the keys before it by 2^8), sums of sixteen products in fp32, parts joined; the output is rounded once
    slack = out.abs() * 2 ** -8 + size * (2 ** -8 + 2 * score + (steps + 16) * 2 ** -22) + p @ (v - v_is).abs()
    return out, slack


def attention(q, k_cache, v_cache, table, lens, q_len, scale, rounded):
    """The whole of a call.  rounded: over keys and values in bf16, as the kernel has them; else over scale x code + minimum as they are."""
    M, H, hd = q.shape
    kv, vv = plain.get(k_cache, hd)[0], plain.get(v_cache, hd)[0]
    num, S, KV, _ = kv.shape
    G = H // KV
    out, slack = torch.zeros(M, H, hd, dtype=F64), torch.zeros(M, H, hd, dtype=F64)
    for b in range(len(lens)):
        n = min(max(int(lens[b]), 0), table.shape[1] * S)
        pos = torch.tensor([i for i in range(n) if 0 <= int(table[b, i // S]) < num])
        if not len(pos):
            continue
        pages, off = table[b].long()[pos // S], pos % S
        seen = (pos <= n - q_len + torch.arange(q_len)[:, None]).repeat_interleave(G, 0)
        for g in range(KV):
            rows = q[b * q_len:(b + 1) * q_len, g * G:(g + 1) * G].to(F64).reshape(q_len * G, hd)
            k, v = kv[pages, off, g], vv[pages, off, g]
            k_is, v_is = (torch.where(torch.isfinite(t), once(t), t) for t in (k, v))
            got = attend(rows, k_is, v_is, seen, scale) if rounded else attend(rows, k, v, seen, scale, k_is, v_is)
            for t, x in zip((out, slack), got):
                t[b * q_len:(b + 1) * q_len, g * G:(g + 1) * G] = x.view(q_len, G, hd)
    return out.view(M, H * hd), slack.view(M, H * hd)
