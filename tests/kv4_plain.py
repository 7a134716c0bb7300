"""The paged cache held in 4 bits (ops.rope_store_kv4, store_kv4, load_kv4, paged_attention_kv4) from its definitions, in 64 bits, read as they are written."""
import math

import torch

BF, F64 = torch.bfloat16, torch.float64


def held(x):
    """Rows [..., hd] of bf16 -> codes (int64), scale, minimum (bf16)."""
    x = x.to(F64)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    spread = (hi - lo).float()
    fine = torch.isfinite(x).all(-1, keepdim=True) & torch.isfinite(spread)
    scale = (spread.double() / 15).to(BF)
    scale = torch.where(scale.float() < 2.0 ** -126, torch.zeros_like(scale), scale)
    border = (torch.arange(15, dtype=F64) + 0.5) * scale.to(F64)   # a code is the number of borders that have been reached
    codes = ((x - lo).unsqueeze(-1) >= border.unsqueeze(-2)).sum(-1)
    codes = torch.where(fine & (scale > 0), codes, 0)
    nan = torch.full_like(scale, math.nan)
    return codes, torch.where(fine, scale, nan), torch.where(fine, (lo + 0.0).to(BF), nan)


def values(codes, scale, low):
    """What stands there, in 64 bits."""
    return scale.to(F64) * codes + low.to(F64)


def rounded(v):
    return v.float().to(BF)


def empty(num_blocks, S, KV, hd, byte=0):
    return torch.full((num_blocks, KV, S * (hd // 2 + 4)), byte, dtype=torch.uint8)


def put(cache, hd, x, slots):
    """Rows x [M, KV, hd] into their slots of `cache` (in place); the values of all rows, in 64 bits."""
    num, KV, size = cache.shape
    S = size // (hd // 2 + 4)
    codes, scale, low = held(x)
    pair = torch.cat([scale, low], -1).contiguous().view(torch.uint8)   # [M, KV, 4]
    byte = (codes[..., ::2] + 16 * codes[..., 1::2]).to(torch.uint8)
    keep = (slots >= 0) & (slots < num * S)
    page, off = slots[keep].long() // S, slots[keep].long() % S
    cache[:, :, :S * (hd // 2)].unflatten(2, (S, hd // 2))[page, :, off] = byte[keep]
    cache[:, :, S * (hd // 2):].unflatten(2, (S, 4))[page, :, off] = pair[keep]
    return values(codes, scale, low)


def get(cache, hd):
    """Values in 64 bits of a whole cache: [num_blocks, S, KV, hd]."""
    num, KV, size = cache.shape
    S = size // (hd // 2 + 4)
    byte = cache[:, :, :S * hd // 2].reshape(num, KV, S, hd // 2).long()
    pair = cache[:, :, S * hd // 2:].contiguous().view(BF).reshape(num, KV, S, 2)
    codes = torch.stack([byte & 15, byte >> 4], -1).reshape(num, KV, S, hd)
    return values(codes, pair[..., :1], pair[..., 1:]).transpose(1, 2), codes.transpose(1, 2), pair.transpose(1, 2)


def turned(x, positions, table, w, eps):
    """Norm and rotation of rows x [M, n, hd] in 64 bits; positions are inside the table."""
    rot = table.shape[1]
    x = x.to(F64)
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)
    at = table.to(F64)[positions][:, None]
    c, s, a, b = at[..., :rot // 2], at[..., rot // 2:], x[..., :rot // 2], x[..., rot // 2:rot]
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), x[..., rot:].abs()], -1)
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1), size


def attention(q, k_cache, v_cache, table, lens, q_len, scale):
    """-> out in 64 bits and how far it may be off.  More than sixteen rows to a key head see values as load_kv4 gives them, in bf16."""
    M, H, hd = q.shape
    (kv, kc, kp), (vv, vc, vp) = get(k_cache, hd), get(v_cache, hd)
    num, S, KV, _ = kv.shape
    G = H // KV
    out, slack = torch.zeros(M, H, hd, dtype=F64), torch.zeros(M, H, hd, dtype=F64)
    for b in range(len(lens)):
        n = min(max(int(lens[b]), 0), table.shape[1] * S)
        at = [i for i in range(n) if 0 <= int(table[b, i // S]) < num]
        if not at:
            continue
        pos = torch.tensor(at)
        pages, off = table[b].long()[pos // S], pos % S
        for g in range(KV):
            k, c, pair = kv[pages, off, g], kc[pages, off, g].to(F64), kp[pages, off, g].to(F64)
            v, vcode, vpair = vv[pages, off, g], vc[pages, off, g].to(F64), vp[pages, off, g].to(F64)
            if G * q_len > 16:
                k, v = rounded(k).to(F64), rounded(v).to(F64)
            for j in range(q_len):
                seen = pos <= n - q_len + j
                if not bool(seen.any()):
                    continue
                rows = q[b * q_len + j, g * G:(g + 1) * G].to(F64)
                p = torch.softmax(rows @ k[seen].t() * scale, 1)
                o = p @ v[seen]
                # the two sums of an output: codes around their middle, and what is left
                one = p @ (v[seen] if G * q_len > 16 else vpair[seen, :1] * (vcode[seen] - 8)).abs()
                two = p @ (vpair[seen, 1:] + 8 * vpair[seen, :1]).abs().expand(-1, hd)
                # scores: hd / 16 sums of 16 products with 16 + code in fp32 at most, each off by 2^-22 of the terms' size, and the minimum's part; a weight moves by as much as its score
                size = rows.abs() @ (pair[seen, :1].abs() * (16 + c[seen])).t() + rows.abs().sum(1, keepdim=True) * (pair[seen, 1:] - 16 * pair[seen, :1]).abs().t()
                spread = (size * abs(scale)).amax(1, keepdim=True) * 2 ** -19
                # a query's values as whole numbers of sixteen bits: off by half a unit, 2^-15 of the row's largest, before they meet scale x code
                spread = spread + abs(scale) * rows.abs().amax(1, keepdim=True) * 2 ** -15 * (pair[seen, :1].abs() * c[seen]).sum(1).amax()
                # weights times scale are rounded to bf16 once (2^-8 at most), the output once more; sums over all keys in fp32
                out[b * q_len + j, g * G:(g + 1) * G] = o
                slack[b * q_len + j, g * G:(g + 1) * G] = (o.abs() + one) * 2 ** -8 + (one + two) * (2 ** -16 + 2 * spread + 2 * int(seen.sum()) * 2 ** -23) + 1e-30
    return out.view(M, H * hd), slack.view(M, H * hd)
