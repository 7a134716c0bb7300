"""The operators around a long paged cache (ops.place_tokens, rope_axes_store_kv, span_bounds, select_spans, span_attention) from their
definitions, in 64 bits, one sequence after the other."""
import math

import torch

F64 = torch.float64


def place(ctx, new, table, free, used, rows, block_size, num_blocks):
    """-> positions, slots, seqs, cu, lens, used, table (lists; `table` a new one)."""
    table, cap = [list(r) for r in table], len(table[0]) * block_size
    used = max(used, 0)
    asked = used              # what the sequences so far would have taken, placed or not
    brought = 0               # rows of those that have their pages, placed or not
    positions, slots, seqs, cu, lens = [], [], [], [0], []
    for b, (c, n) in enumerate(zip(ctx, new)):
        ok = c >= 0 and n >= 0 and c + n <= cap
        need = -(-(c + n) // block_size) - -(-c // block_size) if ok else 0
        asked += need
        ok = ok and (need == 0 or asked <= len(free))
        brought += n if ok else 0
        ok = ok and (n == 0 or brought <= rows)
        if ok:
            have = -(-c // block_size)
            for i in range(need):
                table[b][have + i] = free[used]
                used += 1
            for pos in range(c, c + n):
                page = table[b][pos // block_size]
                positions.append(pos)
                slots.append(page * block_size + pos % block_size if 0 <= page < num_blocks else -1)
                seqs.append(b)
        lens.append(c + n if ok else c)
        cu.append(len(positions))
    left = rows - len(positions)
    return positions + [0] * left, slots + [-1] * left, seqs + [-1] * left, cu, lens, used, table


def rope(qkv, positions, axis_of, slots, table, k_cache, v_cache, heads, kv_heads, hd, q_norm, k_norm, eps):
    """-> q, k_cache, v_cache in 64 bits, and how far each may be off (fp32 sums of two products, a norm, one rounding to bf16)."""
    M, rot, half = qkv.shape[0], table.shape[1], table.shape[1] // 2
    x = qkv.to(F64).view(M, heads + 2 * kv_heads, hd)
    q = torch.full((M, heads, hd), math.nan, dtype=F64)
    kc, vc = k_cache.to(F64).clone(), v_cache.to(F64).clone()
    slack_q, slack_k = torch.zeros_like(q), torch.zeros_like(kc)
    n_slots = kc.shape[0] * kc.shape[1]
    for m in range(M):
        at = [int(a) for a in positions[:, m]]
        if any(a < 0 or a >= table.shape[0] for a in at):
            continue
        c = torch.stack([table[at[axis_of[i]], i].to(F64) for i in range(half)])
        s = torch.stack([table[at[axis_of[i]], half + i].to(F64) for i in range(half)])

        def turned(y, w):
            if w is not None:
                y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)
            a, b = y[:, :half], y[:, half:rot]
            out = torch.cat([a * c - b * s, b * c + a * s, y[:, rot:]], 1)
            size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), y[:, rot:].abs()], 1)
            return out, out.abs() * 2 ** -8 + size * 2 ** -19

        q[m], slack_q[m] = turned(x[m, :heads], q_norm)
        slot = int(slots[m])
        if 0 <= slot < n_slots:
            page, off = divmod(slot, kc.shape[1])
            kc[page, off], slack_k[page, off] = turned(x[m, heads:heads + kv_heads], k_norm)
            vc[page, off] = x[m, heads + kv_heads:]
    return q.view(M, -1), kc, vc, slack_q.view(M, -1), slack_k


def held(length, table, block_size):
    return min(max(int(length), 0), table.shape[1] * block_size)


def bounds(old, k_cache, table, lens, new):
    out = old.clone()
    num, block_size = k_cache.shape[:2]
    span = block_size // old.shape[1]
    for b in range(len(lens)):
        n = held(lens[b], table, block_size)
        for s in range(max(n - new, 0) // span, -(-n // span)):
            page = int(table[b, s * span // block_size])
            if 0 <= page < num:
                off = s * span % block_size
                keys = k_cache[page, off:off + min(span, n - s * span)]
                out[page, off // span, :, 0], out[page, off // span, :, 1] = keys.amin(0), keys.amax(0)
    return out


def select(q, both, table, lens, q_len, block_size, count, first, last):
    B, (num, subs, KV, _, hd) = len(lens), both.shape
    span = block_size // subs
    out = torch.full((B, KV, count), -1, dtype=torch.int32)
    for b in range(B):
        n = -(-held(lens[b], table, block_size) // span)
        there = [s for s in range(n) if 0 <= int(table[b, s // subs]) < num]
        if not there:
            continue
        pages = torch.tensor([int(table[b, s // subs]) for s in there])
        mine = both[pages, torch.tensor(there) % subs].to(F64)   # [n, KV, 2, hd]
        for g in range(KV):
            rows = q[b * q_len:(b + 1) * q_len].view(q_len, KV, -1, hd)[:, g].reshape(-1, hd).to(F64)
            score = torch.maximum(rows[:, None] * mine[:, g, 0], rows[:, None] * mine[:, g, 1]).sum(2)   # [rows, n]
            odd, score = torch.isnan(score).any(0).tolist(), torch.nan_to_num(score, nan=0.0, posinf=math.inf, neginf=-math.inf).amax(0).tolist()
            order = sorted(range(len(there)), key=lambda i: (not (there[i] < first or there[i] >= n - last), not odd[i], 0.0 if odd[i] else -score[i], there[i]))
            got = sorted(there[i] for i in order[:count])
            out[b, g, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return out


def attention(q, k_cache, v_cache, table, lens, spans, span, q_len, scale):
    """-> out in 64 bits and how far it may be off."""
    (num, block_size, KV, hd), (M, H, _) = k_cache.shape, q.shape
    G, B = H // KV, len(lens)
    out, slack = torch.zeros(M, H, hd, dtype=F64), torch.zeros(M, H, hd, dtype=F64)
    for b in range(B):
        n = held(lens[b], table, block_size)
        for g in range(KV):
            at = []
            for s in spans[b, g].tolist():
                if 0 <= s and s * span < n and 0 <= int(table[b, s * span // block_size]) < num:
                    at += range(s * span, min((s + 1) * span, n))
            if not at:
                continue
            pos = torch.tensor(at)
            pages = table[b].long()[pos // block_size]
            k, v = (c[pages, pos % block_size, g].to(F64) for c in (k_cache, v_cache))
            for j in range(q_len):
                seen = pos <= n - q_len + j
                if not bool(seen.any()):
                    continue
                rows = q[b * q_len + j, g * G:(g + 1) * G].to(F64)
                ks, vs = k[seen], v[seen]
                x = rows @ ks.t() * scale
                p = torch.softmax(x, 1)
                o, size = p @ vs, p @ vs.abs()
                # scores: products exact, hd / 16 sums of 16 in fp32 each off by 2^-22 of the terms' size; a weight moves by as much as its score.
                # weights: two bf16 pieces, 2^-16; their sum and the second product: fp32 over all keys
                spread = (rows.abs() @ ks.abs().t() * abs(scale)).amax(1, keepdim=True)
                out[b * q_len + j, g * G:(g + 1) * G] = o
                slack[b * q_len + j, g * G:(g + 1) * G] = o.abs() * 2 ** -8 + size * (2 ** -16 + 2 * spread * 2 ** -19 + 2 * ks.shape[0] * 2 ** -23) + 1e-30
    return out.view(M, H * hd), slack.view(M, H * hd)
