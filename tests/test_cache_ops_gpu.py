"""Operators around a long paged cache on the GPU, through ssd_b200.ops, against their definitions in 64 bits (tests/cache_ops_plain.py)."""
import math

import pytest
import torch

from tests import cache_ops_plain as plain
from tests.cache_ops_util import BF, PLACES, angles, gen, place_case, tables, within

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    from ssd_b200 import lib
    lib.load()
    return torch.device("cuda:0")


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------------------------------------------- place_tokens
def _place(dev, ctx, new, table, free, used, rows, S, total):
    from ssd_b200 import ops
    t = torch.as_tensor(table, dtype=torch.int32).to(dev).contiguous()
    out = ops.place_tokens(i32(ctx, dev), i32(new, dev), t, torch.tensor(free, dtype=torch.int32, device=dev), i32([used], dev), rows, S, total)
    want = plain.place(ctx, new, torch.as_tensor(table).tolist(), free, used, rows, S, total)
    for a, b, what in zip((*out, t), (*want[:5], [want[5]], want[6]), ("positions", "slots", "seqs", "cu", "lens", "used", "table")):
        assert a.tolist() == b, what


@pytest.mark.parametrize("name", sorted(PLACES))
def test_place_tokens(dev, name):
    ctx, new, table, free, used, rows, S, total = place_case(name)
    _place(dev, ctx, new, table, free, used, rows, S, total)


@pytest.mark.parametrize("B,ctx,new,S,short,room", [(513, 40, 1, 16, 0, 1.0), (1500, 70, 5, 64, 0, 1.3), (4600, 33, 2, 16, 1, 1.0), (3, 9, 30011, 256, 0, 1.0), (37, 0, 900, 16, 0, 0.7)])
def test_place_tokens_many(dev, B, ctx, new, S, short, room):
    g = gen(B, new, S)
    c = torch.randint(0, ctx + 1, (B,), generator=g).tolist()
    n = torch.randint(0, new + 1, (B,), generator=g).tolist()
    width = -(-(ctx + new) // S)
    need = sum(-(-(a + b) // S) - -(-a // S) for a, b in zip(c, n))
    table, total = tables(g, c, S, spare=need + 3, width=width)
    have = set(table.flatten().tolist())
    free = [p for p in range(total) if p not in have]
    _place(dev, c, n, table, free[:need // 2] if short else free, 2 if not short else 0, max(1, int(sum(n) * room)), S, total)


def test_place_tokens_bad_pages(dev):
    _place(dev, [17, 3, 0], [3, 2, 5], [[0, 99], [-7, -1], [-1, -1]], [2147483647, 5], 0, 12, 16, 6)


# ---------------------------------------------------------------------------------------------------- rope_axes_store_kv
@pytest.mark.parametrize("M,H,KV,hd,rot,axes,norm", [
    (1, 64, 8, 128, 128, 3, False), (7, 32, 8, 64, 64, 3, True), (64, 16, 8, 128, 128, 1, True), (33, 40, 8, 128, 64, 4, False),
    (300, 6, 2, 64, 32, 2, True), (5, 5, 1, 128, 16, 3, False), (9, 4, 2, 256, 256, 3, True), (700, 64, 8, 128, 128, 3, False), (2, 1, 1, 64, 48, 2, True),
])
@pytest.mark.parametrize("turns", [False, True])
def test_rope_axes_store_kv(dev, M, H, KV, hd, rot, axes, norm, turns):
    from ssd_b200 import ops
    g = gen(M, H, hd, rot, axes)
    top, S, eps = 300, 16, 1e-6
    pages = M // S + 3
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF)
    positions = torch.randint(0, top, (axes, M), generator=g)
    slots = torch.randperm(pages * S, generator=g)[:M].to(torch.int32)
    for i, bad in enumerate((top, -1, 1 << 45)):
        if M > 4:
            positions[i % axes, i + 1] = bad
    if M > 6:
        slots[5], slots[6] = -1, pages * S
    n = rot // 2
    axis_of = [i % axes for i in range(n)] if turns else sorted(i % axes for i in range(n))
    qn, kn = ((1 + 0.2 * torch.randn(2, hd, generator=g)).to(BF)) if norm else (None, None)
    table = angles(top, rot)
    old = torch.randn(2, pages, S, KV, hd, generator=g).to(BF)
    kc, vc = old.to(dev)
    up = lambda t: None if t is None else t.to(dev)  # noqa: E731
    q = ops.rope_axes_store_kv(up(qkv), up(positions), axis_of, up(slots), up(table), kc, vc, H, KV, hd, up(qn), up(kn), eps)
    wq, wk, wv, slack_q, slack_k = plain.rope(qkv, positions, axis_of, slots, table, old[0], old[1], H, KV, hd, qn, kn, eps)
    within(q, wq, slack_q)
    within(kc, wk, slack_k)
    assert torch.equal(vc.double().cpu(), wv)


def test_rope_axes_many_rows(dev):
    """More rows than warps: a warp has all heads of its row."""
    from ssd_b200 import ops
    g = gen(31)
    M, H, KV, hd, rot, axes, S = 3001, 20, 5, 64, 64, 3, 64
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF)
    positions = torch.randint(0, 200, (axes, M), generator=g)
    slots = torch.randperm(50 * S, generator=g)[:M].to(torch.int32)
    w = (1 + 0.2 * torch.randn(2, hd, generator=g)).to(BF)
    table, axis_of = angles(200, rot), [0] * 8 + [1] * 13 + [2] * 11
    kc, vc = torch.zeros(2, 50, S, KV, hd, dtype=BF, device=dev)
    q = ops.rope_axes_store_kv(qkv.to(dev), positions.to(dev), axis_of, slots.to(dev), table.to(dev), kc, vc, H, KV, hd, w[0].to(dev), w[1].to(dev))
    zero = torch.zeros(50, S, KV, hd, dtype=BF)
    wq, wk, wv, slack_q, slack_k = plain.rope(qkv, positions, axis_of, slots, table, zero, zero, H, KV, hd, w[0], w[1], 1e-6)
    within(q, wq, slack_q)
    within(kc, wk, slack_k)
    assert torch.equal(vc.double().cpu(), wv)


def test_rope_axes_passes_what_does_not_turn(dev):
    """Channels behind rot_dim keep their bits, infinities among them; a norm on one side only."""
    from ssd_b200 import ops
    g = gen(3)
    H, KV, hd, rot, M = 4, 2, 128, 32, 6
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF)
    x = qkv.view(M, H + 2 * KV, hd)
    x[:, :, rot] = INF
    x[:, :, rot + 1] = -0.0
    kc, vc = torch.zeros(2, 1, 16, KV, hd, dtype=BF, device=dev)
    pos, slots, table = torch.arange(M).repeat(2, 1), torch.arange(M, dtype=torch.int32), angles(10, rot)
    q = ops.rope_axes_store_kv(qkv.to(dev), pos.to(dev), [0, 1] * 8, slots.to(dev), table.to(dev), kc, vc, H, KV, hd)
    bits = lambda t: t.cpu().view(torch.int16)  # noqa: E731
    assert torch.equal(bits(q.view(M, H, hd)[..., rot:].contiguous()), bits(x[:, :H, rot:].contiguous()))
    assert torch.equal(bits(kc[0, :M, :, rot:].contiguous()), bits(x[:, H:H + KV, rot:].contiguous()))
    x[:, :, rot] = 1.0
    w = torch.full((hd,), 2.0, dtype=BF)
    q2 = ops.rope_axes_store_kv(qkv.to(dev), pos.to(dev), [0, 1] * 8, slots.to(dev), table.to(dev), kc, vc, H, KV, hd, None, w.to(dev))
    wq, wk, _, slack_q, slack_k = plain.rope(qkv, pos, [0, 1] * 8, slots, table, torch.zeros(1, 16, KV, hd), torch.zeros(1, 16, KV, hd), H, KV, hd, None, w, 1e-6)
    within(q2, wq, slack_q)
    within(kc, wk, slack_k)


# ---------------------------------------------------------------------------------------------------- span_bounds
def _same(a, b):
    a, b = a.cpu(), b.cpu()
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


@pytest.mark.parametrize("KV,hd,S,span,new,lens", [
    (8, 128, 256, 32, 1, [1, 31, 32, 33, 255, 256, 257, 1000]), (8, 128, 256, 32, 1000, [1000, 5, 0]), (1, 64, 64, 16, 7, [64, 70, 3]), (5, 128, 16, 16, 40, [33, 16, 100]),
    (8, 128, 256, 32, 16000, [16000, 9001, 77]), (1, 64, 64, 16, 64000, [64000]), (5, 128, 64, 16, 9000, [9000, 8100]), (5, 64, 128, 64, 20000, [20000, 19999]), (2, 64, 32, 32, 40000, [40000]),
    (2, 64, 128, 128, 1, [1, 128, 129, 384]), (20, 128, 32, 32, 9, [40, 41]), (8, 64, 256, 64, 300, [-5, 768, 100000]), (1, 128, 16, 16, 1 << 30, [48]),
])
def test_span_bounds(dev, KV, hd, S, span, new, lens):
    from ssd_b200 import ops
    g = gen(KV, hd, S, span, new)
    width = 4 if max(lens) < 5000 or max(lens) == 100000 else -(-max(lens) // S)
    table, total = tables(g, [min(max(n, 0), width * S) for n in lens], S, width=width)
    if len(lens) > 2:
        table[0, 0] = total       # outside the cache
        table[1, 0] = -5
    keys = torch.randn(total, S, KV, hd, generator=g).to(BF)
    keys[:, 3::11] = NAN          # in the context of some spans, behind it in others
    old = torch.full((total, S // span, KV, 2, hd), 5.0, dtype=BF)
    got = ops.span_bounds(old.to(dev), keys.to(dev), table.to(dev), i32(lens, dev), new)
    _same(got, plain.bounds(old, keys, table, lens, new))


# ---------------------------------------------------------------------------------------------------- select_spans
def _bounds(g, total, subs, KV, hd):
    mid, half = torch.randn(2, total, subs, KV, hd, generator=g)
    return torch.stack([0.4 * mid - 2 - 0.3 * half.abs(), 0.4 * mid + 2 + 0.3 * half.abs()], 3).to(BF).contiguous()


def _select(dev, q, both, table, lens, q_len, S, count, first=1, last=None):
    from ssd_b200 import ops
    got = ops.select_spans(q.to(dev), both.to(dev), table.to(dev), i32(lens, dev), q_len, S, count, first, last)
    span = S // both.shape[1]
    last = min((q_len + span - 2) // span + 1, count - first) if last is None else last
    want = plain.select(q, both, table, lens, q_len, S, count, first, last)
    assert torch.equal(got.cpu(), want)
    return want


@pytest.mark.parametrize("H,KV,hd", [(64, 8, 128), (32, 8, 64), (4, 2, 64), (5, 1, 128), (6, 2, 64), (40, 8, 128), (2, 2, 128), (32, 1, 128)])
@pytest.mark.parametrize("q_len,S,span,count,lens", [
    (1, 256, 32, 8, [1000, 40, 33, 1, 0]), (7, 256, 64, 5, [3000, 7, 64, 65]), (1, 16, 16, 20, [5000]), (3, 128, 128, 2, [900, 1027]), (1, 64, 16, 64, [1500, 1024, 1023]),
    (1, 256, 256, 2, [4000, 256, 257]),
])
def test_select_spans(dev, H, KV, hd, q_len, S, span, count, lens):
    g = gen(H, hd, q_len, S, span)
    table, total = tables(g, lens, S)
    q = torch.randn(len(lens) * q_len, H, hd, generator=g).to(BF)
    _select(dev, q, _bounds(g, total, S // span, KV, hd), table, lens, q_len, S, count)


@pytest.mark.parametrize("n,count,first,last", [(9000, 128, 1, 1), (5000, 1, 0, 0), (5000, 1, 1, 0), (3001, 2000, 4, 3), (24576, 700, 0, 2), (1025, 1024, 0, 0), (2048, 3, 0, 3)])
def test_select_spans_long(dev, n, count, first, last):
    g = gen(n, count)
    S, span, KV, hd = 64, 16, 1, 64
    lens = [n * span - 5, n * span // 3]
    table, total = tables(g, lens, S)
    q = torch.randn(2, 4, hd, generator=g).to(BF)
    _select(dev, q, _bounds(g, total, S // span, KV, hd), table, lens, 1, S, count, first, last)


@pytest.mark.parametrize("q_len,count", [(1, 40), (3, 7)])
def test_select_spans_batch(dev, q_len, count):
    """Enough sequences that a warp has several groups of spans, of very uneven lengths."""
    g = gen(17, q_len)
    S, span, KV, hd, H = 64, 16, 8, 64, 32
    lens = [max(q_len, (i * 2477) % 9600) for i in range(24)] + [9600, q_len]
    table, total = tables(g, lens, S)
    q = torch.randn(len(lens) * q_len, H, hd, generator=g).to(BF)
    _select(dev, q, _bounds(g, total, S // span, KV, hd), table, lens, q_len, S, count)


@pytest.mark.parametrize("width", [None, 200])
def test_select_spans_ties_and_odd_values(dev, width):
    """Whole numbers make equal scores: the lowest index goes first.  Zeros of both signs are equal, NaN is above all, infinities are in order.  Short tables take one
    kernel, wide ones two."""
    g = gen(11)
    S, span, KV, hd, H = 64, 16, 2, 64, 8
    lens = [40 * span, 40 * span - 3, 17]
    table, total = tables(g, lens, S, width=width)
    for kind in range(6):
        q = torch.randint(-1, 2, (3, H, hd), generator=g).to(BF)
        both = torch.randint(-1, 2, (total, S // span, KV, 2, hd), generator=g).to(BF)
        both = both.sort(3).values.contiguous()
        if kind == 1:
            both.zero_()
        if kind == 2:
            both = torch.where(both == 0, torch.tensor(-0.0, dtype=BF), both) * 0
        if kind == 3:
            both[:, 1, 0, 1, 5] = INF
            both[:, 2, 0, :, 7] = -INF
        if kind == 4:
            both[::2, 3, 1, 0, 9] = NAN
            both[1::2, 0, 1, 1, 63] = INF
        if kind == 5:
            q[0, 3, 2] = INF
            q[1, 0, 0] = NAN
            both = both * 3e38
        for count in (3, 11, 39):
            _select(dev, q, both, table, lens, 1, S, count)


def test_select_spans_close_scores(dev):
    """Scores that differ in their last bits only, far below what 32 bits hold."""
    g = gen(12)
    S, span, KV, hd = 64, 16, 1, 128
    n = 600
    table, total = tables(g, [n * span], S)
    both = torch.ones(total, S // span, KV, 2, hd, dtype=BF)
    both[..., 0] = 2.0 ** 20
    both[..., 1] = (2.0 ** -8 * torch.randint(1, 200, (total, S // span, KV, 1), generator=g)).to(BF)
    both[..., 2] = -(2.0 ** 20)
    q = torch.ones(1, 4, hd, dtype=BF)
    for count in (5, 50, 333):
        _select(dev, q, both, table, [n * span], 1, S, count)


@pytest.mark.parametrize("width", [10, 300])
def test_select_spans_bad_pages(dev, width):
    g = gen(13)
    S, span, KV, hd = 32, 16, 2, 64
    lens = [300, 299, -4, 100000]
    table, total = tables(g, [300, 299, 0, 320], S, width=width)
    table[0, 2], table[0, 5], table[1, 0], table[1, 9], table[3, 4] = total, -9, 2147483647, -2147483648, total + 1
    q = torch.randn(4, 4, hd, generator=g).to(BF)
    for count in (4, 30):
        got = _select(dev, q, _bounds(g, total, 2, KV, hd), table, lens, 1, S, count, 2, 2)
        assert 4 not in got[0].tolist()


# ---------------------------------------------------------------------------------------------------- span_attention
def _lists(g, lens, KV, span, count):
    out = torch.full((len(lens), KV, count), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        m = max(0, -(-n // span))
        for h in range(KV):
            pick = torch.randperm(m, generator=g)[:count].sort().values if m else torch.zeros(0)
            out[b, h, :len(pick)] = pick.to(torch.int32)
    return out


def ops_attention(dev, q, kc, vc, table, lens, spans, span, q_len, scale):
    from ssd_b200 import ops
    return ops.span_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32(lens, dev), spans.to(dev), span, q_len, scale)


def _attend(dev, q, kc, vc, table, lens, spans, span, q_len, scale):
    got = ops_attention(dev, q, kc, vc, table, lens, spans, span, q_len, scale)
    want, slack = plain.attention(q, kc, vc, table, lens, spans, span, q_len, scale)
    within(got, want, slack)
    return got


@pytest.mark.parametrize("H,KV,hd", [(64, 8, 128), (32, 8, 64), (4, 2, 64), (5, 1, 128), (6, 2, 64), (2, 2, 128), (32, 1, 128)])
@pytest.mark.parametrize("q_len,S,span,count,lens", [
    (1, 256, 32, 6, [1000, 40, 33, 1, 0]), (7, 256, 64, 4, [900, 7, 64, 3]), (1, 16, 16, 30, [700, 15]), (3, 128, 128, 2, [300, 131]), (40, 64, 16, 12, [300]), (2, 256, 256, 3, [600, 257]),
])
def test_span_attention(dev, H, KV, hd, q_len, S, span, count, lens):
    g = gen(H, hd, q_len, S, span)
    table, total = tables(g, lens, S)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    q = torch.randn(len(lens) * q_len, H, hd, generator=g).to(BF)
    _attend(dev, q, kc, vc, table, lens, _lists(g, lens, KV, span, count), span, q_len, hd ** -0.5)


@pytest.mark.parametrize("count,q_len,H,KV,hd", [(256, 1, 8, 1, 128), (512, 3, 8, 2, 64), (4096, 1, 4, 1, 64), (300, 8, 8, 1, 128), (1000, 2, 16, 1, 128), (4096, 9, 4, 1, 128)])
def test_span_attention_long(dev, count, q_len, H, KV, hd):
    g = gen(count, q_len, H)
    S, span = 64, 16
    lens = [count * span + 77, 12 * span + 1]
    table, total = tables(g, lens, S)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    q = (3 * torch.randn(2 * q_len, H, hd, generator=g)).to(BF)
    _attend(dev, q, kc, vc, table, lens, _lists(g, lens, KV, span, count), span, q_len, hd ** -0.5)


@pytest.mark.parametrize("B,H,KV,hd,q_len", [(40, 16, 8, 64, 1), (70, 8, 8, 128, 2), (33, 32, 4, 64, 3)])
def test_span_attention_batch(dev, B, H, KV, hd, q_len):
    """Batches that fill the SMs with a block per key head."""
    g = gen(B, H, q_len)
    S, span, count = 32, 16, 3
    lens = [q_len + (i * 37) % 90 for i in range(B)]
    table, total = tables(g, lens, S)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    q = torch.randn(B * q_len, H, hd, generator=g).to(BF)
    _attend(dev, q, kc, vc, table, lens, _lists(g, lens, KV, span, count), span, q_len, hd ** -0.5)


def test_span_attention_many_rows_stale_and_odd(dev):
    """The same for more than sixteen rows to a key head: stale values, odd lists, spans of 48 tokens, scales of both signs and zero."""
    g = gen(24)
    S, span, KV, hd, H, q_len = 96, 48, 2, 128, 16, 5
    lens = [200, 131, 96, 5, 3, 0, 400]
    table, total = tables(g, [min(n, 4 * S) for n in lens], S, spare=3, width=4)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    for c, v in ((kc, NAN), (vc, INF)):
        c[[p for p in range(total) if p not in table.flatten().tolist()]] = v
        for b, n in enumerate(lens[:5]):
            page, off = divmod(n, S)
            if off:
                c[table[b, page], off:] = v
    table[6, 1] = total
    spans = torch.tensor([[4, 0, 2, -1, 1], [2, 2, 1, 0, 9], [1, -7, 0, 5, 1], [0, 1, 2, 3, 4], [0, -1, 0, 7, 7], [0, 1, 2, 3, 4], [2, 8, 0, 7, 3]], dtype=torch.int32)
    spans = torch.stack([spans, spans.flip(1)], 1).contiguous()
    q = torch.randn(len(lens) * q_len, H, hd, generator=g).to(BF)
    for scale in (0.09, -0.09, 0.0):
        got = _attend(dev, q, kc, vc, table, lens, spans, span, q_len, scale)
        assert bool(torch.isfinite(got.float()).all()) and not bool(got.view(len(lens), -1)[5].any())


def test_span_attention_stale_values(dev):
    """NaN and infinities behind the context, on pages that are not listed and on pages of nobody."""
    g = gen(21)
    S, span, KV, hd, H = 64, 16, 2, 128, 8
    lens = [40, 129, 16]
    table, total = tables(g, lens, S, spare=3)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    free = [p for p in range(total) if p not in table.flatten().tolist()]
    for c, v in ((kc, NAN), (vc, INF)):
        c[free] = v
        for b, n in enumerate(lens):
            page, off = divmod(n, S)
            if off:
                c[table[b, page], off:] = v
    kc[table[1, 1]] = NAN   # spans 4 to 7 of the second sequence are not listed
    vc[table[1, 1]] = NAN
    spans = torch.tensor([[0, 1, 2], [0, 3, 8], [0, -1, -1]], dtype=torch.int32)[:, None].expand(3, KV, 3).contiguous()
    q = torch.randn(3, H, hd, generator=g).to(BF)
    got = _attend(dev, q, kc, vc, table, lens, spans, span, 1, 0.09)
    assert bool(torch.isfinite(got.float()).all())


@pytest.mark.parametrize("q_len,H", [(1, 4), (3, 8), (6, 16)])
def test_span_attention_nan_rows(dev, q_len, H):
    """A query of NaN (a position outside the angles' table makes one) has NaN in its row, and only there; a key of NaN in every row that sees it."""
    g = gen(25, q_len)
    S, span, KV, hd = 64, 16, 2, 128
    lens = [200, 70, 3000]
    table, total = tables(g, lens, S)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    q = torch.randn(len(lens) * q_len, H, hd, generator=g).to(BF)
    q[0], q[q_len, 1] = NAN, NAN
    q[2 * q_len, 0, 5] = NAN
    spans = _lists(g, lens, KV, span, 9)
    spans[0] = torch.tensor([0, 1, 2, 3, -1, -1, -1, -1, 12])
    got = _attend(dev, q, kc, vc, table, lens, spans, span, q_len, 0.09).view(-1, H, hd)
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isnan(got[q_len, 1]).all()) and not bool(torch.isnan(got[q_len, 0]).any())
    kc[table[0, 0], 3, 0, 7] = NAN
    kc[table[0, 3], 6, 1] = NAN   # token 198: of three queries or more the last two see it
    _attend(dev, q, kc, vc, table, lens, spans, span, q_len, 0.09)


@pytest.mark.parametrize("q_len,H,hd,span,count", [(2, 4, 128, 16, 9), (8, 4, 64, 32, 5), (3, 10, 64, 16, 200), (9, 8, 128, 16, 9), (40, 8, 64, 32, 40), (70, 16, 128, 16, 5), (4, 16, 128, 64, 64)])
def test_span_attention_values_of_new_tokens(dev, q_len, H, hd, span, count):
    """Infinite and NaN values of new tokens reach the queries that see them, as often as they are listed, and no others."""
    g = gen(26, q_len, H)
    S, KV = 64, 2
    lens = [200, 70, 3000, 65, 4000]
    table, total = tables(g, lens, S)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    spans = _lists(g, lens, KV, span, count)
    for b, n in enumerate(lens):
        ends = [(n - 1) // span, max(n - q_len, 0) // span]
        spans[b, :, :2] = torch.tensor(ends if b % 2 else ends[:1] * 2, dtype=torch.int32)   # (one span twice)
        for j, (d, v) in enumerate([(3, INF), (hd - 1, NAN), (5, -INF), (3, -INF), (20, INF)]):
            pos = n - 1 - j * q_len // 8 - (b == 1)
            vc[table[b, pos // S], pos % S, j % KV, d] = v
            kc[table[b, pos // S], pos % S, 0, d] = NAN if b == 3 and j == 0 else 1.0
    q = torch.randn(len(lens) * q_len, H, hd, generator=g).to(BF)
    got = ops_attention(dev, q, kc, vc, table, lens, spans, span, q_len, 0.09).double().cpu()
    want, slack = plain.attention(q, kc, vc, table, lens, spans, span, q_len, 0.09)
    odd = ~torch.isfinite(want)
    assert bool(odd.any()) and torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[odd].nan_to_num(7.0, INF, -INF), want[odd].nan_to_num(7.0, INF, -INF))
    within(got.masked_fill(odd, 0), want.masked_fill(odd, 0), slack.masked_fill(odd, 0))


def test_span_attention_odd_lists(dev):
    """Any order, entries twice, outside the context, on bad pages; rows that see nothing."""
    g = gen(22)
    S, span, KV, hd, H = 64, 32, 1, 64, 4
    lens = [200, 200, 200, 2, 0, -3, 100000, 200]
    table, total = tables(g, [200, 200, 200, 2, 0, 0, 256, 200], S, width=4)
    table[7] = torch.tensor([total, -1, 2147483647, table[7, 3]], dtype=torch.int32)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    spans = torch.tensor([[5, 0, 3, -1, 6], [2, 2, 2, 1, 0], [-1, 7, 2147483647, -2147483648, 100], [0, 1, 2, 3, 4], [0, 1, -1, 2, 3], [0, 0, 0, 0, 0], [7, 0, 8, 9, 3],
                          [0, 2, 4, 6, 1]], dtype=torch.int32)[:, None].contiguous()
    for q_len in (1, 5):
        q = torch.randn(len(lens) * q_len, H, hd, generator=g).to(BF)
        got = _attend(dev, q, kc, vc, table, lens, spans, span, q_len, 0.125).view(len(lens), q_len, -1)
        assert not bool(got[2].any()) and not bool(got[4].any()) and not bool(got[5].any())


def test_span_attention_large_scores(dev):
    """Scores up to some thousands, of both signs of the scale: nothing overflows, the largest take all."""
    g = gen(23)
    S, span, KV, hd, H = 64, 16, 2, 64, 4
    table, total = tables(g, [300], S)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    q = (40 * torch.randn(2, H, hd, generator=g)).to(BF)
    spans = _lists(g, [300], KV, span, 9)
    for scale in (1.0, -1.0, 0.0):
        _attend(dev, q, kc, vc, table, [300], spans, span, 2, scale)


# ---------------------------------------------------------------------------------------------------- together
class Step:
    """One layer's cache and a batch in it: place, rotate and store, bounds, select, attend, as a program with a long context runs them."""

    def __init__(self, dev, seed, ctx, new, H=8, KV=2, hd=64, S=64, span=16, count=6, rows=None):
        g = gen(seed, len(ctx), new)
        self.H, self.KV, self.hd, self.S, self.span, self.count, self.new = H, KV, hd, S, span, count, new
        self.B, self.M = len(ctx), rows or len(ctx) * new
        table, total = tables(g, ctx, S, spare=2 * len(ctx), width=-(-(max(ctx) + new) // S) + 1)
        have = set(table.flatten().tolist())
        self.pages = total
        self.host = {"ctx": ctx, "table": table, "free": [p for p in range(total) if p not in have]}
        self.kc, self.vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF).to(dev)
        self.qkv = torch.randn(self.M, (H + 2 * KV) * hd, generator=g).to(BF).to(dev)
        self.table, self.ctx, self.news = table.to(dev), i32(ctx, dev), i32([new] * len(ctx), dev)
        self.free, self.used = i32(self.host["free"], dev), i32([0], dev)
        self.angles = angles(4096, hd).to(dev)
        self.axis_of = [i % 3 for i in range(hd // 2)]
        self.bounds = torch.zeros(total, S // span, KV, 2, hd, dtype=BF, device=dev)
        from ssd_b200 import ops
        ops.span_bounds(self.bounds, self.kc, self.table, self.ctx, max(ctx) + 1)

    def run(self, count=None):
        from ssd_b200 import ops
        positions, slots, _, cu, lens, used = ops.place_tokens(self.ctx, self.news, self.table, self.free, self.used, self.M, self.S, self.pages)
        q = ops.rope_axes_store_kv(self.qkv, torch.stack([positions, positions // 2, positions // 3]), self.axis_of, slots, self.angles, self.kc, self.vc, self.H, self.KV, self.hd)
        q = q.view(self.M, self.H, self.hd)[:self.B * self.new]
        ops.span_bounds(self.bounds, self.kc, self.table, lens, self.new)
        spans = ops.select_spans(q, self.bounds, self.table, lens, self.new, self.S, count or self.count)
        out = ops.span_attention(q, self.kc, self.vc, self.table, lens, spans, self.span, self.new, self.hd ** -0.5)
        return out, spans, q, lens, slots


@pytest.mark.parametrize("new,ctx,rows", [(1, [300, 64, 0, 511], 7), (5, [700, 63, 130], None)])
def test_step(dev, new, ctx, rows):
    s = Step(dev, 5, ctx, new, rows=rows)
    kc0 = s.kc.cpu()
    out, spans, q, lens, slots = s.run()
    place = plain.place(ctx, [new] * s.B, s.host["table"].tolist(), s.host["free"], 0, s.M, s.S, s.pages)
    assert slots.tolist() == place[1] and lens.tolist() == place[4] and s.table.tolist() == place[6]
    pos = torch.tensor(place[0])
    wq, wk, _, slack_q, slack_k = plain.rope(s.qkv.cpu(), torch.stack([pos, pos // 2, pos // 3]), s.axis_of, torch.tensor(place[1]), s.angles.cpu(), kc0, kc0, s.H, s.KV, s.hd, None, None, 1e-6)
    within(q.reshape(-1, s.H * s.hd), wq[:s.B * new], slack_q[:s.B * new])
    within(s.kc, wk, slack_k)
    both = plain.bounds(torch.zeros_like(s.bounds).cpu(), s.kc.cpu(), s.table.cpu(), place[4], 1 << 20)
    _same(s.bounds, both)
    want = plain.select(q.cpu(), both, s.table.cpu(), place[4], new, s.S, s.count, 1, (new + s.span - 2) // s.span + 1)
    assert torch.equal(spans.cpu(), want)
    within(out, *plain.attention(q.cpu(), s.kc.cpu(), s.vc.cpu(), s.table.cpu(), place[4], want, s.span, new, s.hd ** -0.5))


def test_step_with_all_spans_is_paged_attention(dev):
    """With room for every span the result is attention over the whole context."""
    from ssd_b200 import ops
    s = Step(dev, 6, [300, 64, 5, 511], 4)
    out, spans, q, lens, _ = s.run(count=64)
    dense = ops.paged_attention(q.contiguous(), s.kc, s.vc, s.table, lens, 4, s.hd ** -0.5)
    want, slack = plain.attention(q.cpu(), s.kc.cpu(), s.vc.cpu(), s.table.cpu(), lens.tolist(), spans.cpu(), s.span, 4, s.hd ** -0.5)
    within(out, want, slack)
    assert float((out.float() - dense.float()).abs().max()) <= 2 ** -6   # paged_attention's weights are one bf16 piece


def test_step_again_gives_the_same_bits(dev):
    s = Step(dev, 7, [900, 640, 77], 3)
    a = s.run()
    b = s.run()
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_a_sequence_does_not_depend_on_its_neighbours_values(dev):
    """Another sequence's keys and queries leave a sequence's bits alone."""
    s = Step(dev, 8, [900, 640, 77], 1)
    a = s.run()[0][1].clone()
    s.qkv[0] = 1.5
    s.kc[s.table[2, 0]] = 0.25
    assert torch.equal(s.run()[0][1], a)


def test_step_on_another_stream_and_two_at_once(dev):
    one, two = Step(dev, 9, [900, 640, 77], 3), Step(dev, 10, [100, 1640, 7, 80], 2)
    want = [one.run()[0].clone(), two.run()[0].clone()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for st, s in zip(streams, (one, two)):
            with torch.cuda.stream(st):
                got.append(s.run()[0])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_step_captured(dev):
    """The step as a CUDA graph, replayed with other lengths, keys and queries; two graphs in flight at once."""
    a, b = Step(dev, 14, [500, 64, 30], 2), Step(dev, 15, [300, 640], 1)
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for s in (a, b):
        with torch.cuda.stream(side):
            s.run()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(s.run())
        graphs.append(g)
    for turn in range(3):
        for s in (a, b):
            s.qkv.copy_(torch.randn(s.qkv.shape, generator=gen(30 + turn)).to(BF))
            s.ctx.copy_(i32([max(0, c - 40 * turn) for c in s.host["ctx"]], dev))
            s.table.copy_(s.host["table"])
            from ssd_b200 import ops
            ops.span_bounds(s.bounds, s.kc, s.table, s.ctx, 4096)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for s, o in zip((a, b), got):
            s.table.copy_(s.host["table"])
            for x, y in zip(s.run(), o):
                assert torch.equal(x, y)


def test_a_call_behind_an_event(dev):
    """Inputs that another stream makes: the call waits for them, also where a call of its own stream is right in front."""
    s = Step(dev, 18, [900, 640, 77], 2)
    want = s.run()[0].clone()
    qkv, other = s.qkv.clone(), torch.cuda.Stream()
    for _ in range(3):
        s.qkv.zero_()
        torch.cuda.synchronize()
        s.run()
        with torch.cuda.stream(other):
            torch.cuda._sleep(20000000)
            s.qkv.copy_(qkv)
            ready = torch.cuda.Event()
            ready.record()
        torch.cuda.current_stream().wait_event(ready)
        got = s.run()[0]
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_a_wait_that_ran_out_is_reported_once(dev):
    """The word that a bounded wait would set is set by the host here: calls on tiles look at it, the others leave it."""
    from ssd_b200 import lib
    word = lib.load().ssdk_debug_op_wait_word()
    s = Step(dev, 19, [300, 64], 6, H=16)
    s.run()
    few = Step(dev, 20, [300, 64], 1)
    torch.cuda.synchronize()
    word[0] = 1
    few.run()
    assert word[0] == 1
    with pytest.raises(RuntimeError, match="ran out"):
        s.run()
    assert word[0] == 0
    s.run()


def test_offsets_past_32_bits(dev):
    """A cache of more than 2^32 bytes and 2^31 elements: its last pages are as good as its first."""
    from ssd_b200 import ops
    g = gen(40)
    S, span, KV, hd, H = 256, 32, 8, 128, 8
    pages = 8300   # 8300 * 256 * 8 * 128 = 2.18e9 elements
    kc = torch.zeros(pages, S, KV, hd, dtype=BF, device=dev)
    vc = torch.zeros(pages, S, KV, hd, dtype=BF, device=dev)
    both = torch.zeros(pages, S // span, KV, 2, hd, dtype=BF, device=dev)
    far = [8299, 8290, 3, 8295]
    small = torch.randn(2, 4, S, KV, hd, generator=g).to(BF)
    qkv = torch.randn(1, (H + 2 * KV) * hd, generator=g).to(BF)
    for i, p in enumerate(far):
        kc[p], vc[p] = small[0, i].to(dev), small[1, i].to(dev)
    table, lens = i32([far], dev), i32([4 * S - 9], dev)
    rope = angles(16, hd)
    slot = 8295 * S + 246
    q = ops.rope_axes_store_kv(qkv.to(dev), torch.tensor([[5]], device=dev), [0] * (hd // 2), i32([slot], dev), rope.to(dev), kc, vc, H, KV, hd)
    wq, wk, wv, slack_q, slack_k = plain.rope(qkv, torch.tensor([[5]]), [0] * (hd // 2), [3 * S + 246], rope, small[0], small[1], H, KV, hd, None, None, 1e-6)
    within(q, wq, slack_q)
    within(kc[far], wk, slack_k)
    assert torch.equal(vc[far].double().cpu(), wv)
    ops.span_bounds(both, kc, table, lens, 4 * S)
    mine, k4, v4, t4 = both[far].cpu(), kc[far].cpu(), vc[far].cpu(), torch.tensor([[0, 1, 2, 3]], dtype=torch.int32)
    _same(mine, plain.bounds(torch.zeros_like(mine), k4, t4, lens.tolist(), 4 * S))
    q = q.view(1, H, hd)
    spans = ops.select_spans(q, both, table, lens, 1, S, 7)
    assert torch.equal(spans.cpu(), plain.select(q.cpu(), mine, t4, lens.tolist(), 1, S, 7, 1, 1))
    out = ops.span_attention(q, kc, vc, table, lens, spans, span, 1, 0.088)
    within(out, *plain.attention(q.cpu(), k4, v4, t4, lens.tolist(), spans.cpu(), span, 1, 0.088))


def test_refusals_leave_the_device_alone(dev):
    from ssd_b200 import ops
    s = Step(dev, 16, [64, 20], 1)
    with pytest.raises(ValueError):
        ops.place_tokens(s.ctx, s.news.cpu(), s.table, s.free, s.used, 4, s.S, s.pages)
    with pytest.raises(RuntimeError, match="spans"):
        ops.select_spans(torch.zeros(2, s.H, s.hd, dtype=BF, device=dev), s.bounds, s.table, s.ctx, 1, s.S, 1, 1, 1)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        ops.span_attention(torch.zeros(2, s.H, s.hd, dtype=BF, device=dev), s.kc, s.vc, s.table, s.ctx, torch.zeros(2, s.KV, 4, dtype=torch.int32, device=dev), 8, 1, 1.0)
    odd = torch.zeros(s.qkv.numel() + 1, dtype=BF, device=dev)[1:].view_as(s.qkv)
    with pytest.raises(RuntimeError, match="16 bytes"):
        ops.rope_axes_store_kv(odd, torch.zeros(3, s.M, dtype=torch.int64, device=dev), s.axis_of, i32([0] * s.M, dev), s.angles, s.kc, s.vc, s.H, s.KV, s.hd)
    assert math.isfinite(float(s.run()[0].float().sum()))
