"""The paged cache held in 4 bits on the GPU, through ssd_b200.ops, against its definitions in 64 bits (tests/kv4_plain.py)."""
import math

import pytest
import torch

from tests import kv4_plain as plain
from tests.cache_ops_util import BF, angles, gen, tables, within

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


def same_bits(a, b):
    a, b = a.cpu().contiguous(), b.cpu().contiguous()
    if a.dtype == BF:
        nan = torch.isnan(b)
        assert torch.equal(torch.isnan(a), nan)
        a, b = a.view(torch.int16).masked_fill(nan, 0), b.view(torch.int16).masked_fill(nan, 0)
    assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------- store_kv4, load_kv4
def awkward(g, M, KV, hd):
    """Rows of many sizes: ties, constant rows, zeros of both signs, the type's lowest and smallest, what is not finite."""
    x = torch.randn(M, KV, hd, generator=g) * torch.exp2(torch.randint(-30, 30, (M, KV, 1), generator=g).float())
    x[::5] = torch.randint(-40, 41, x[::5].shape, generator=g).float() / 4          # quotients of a code and a half
    rows = [torch.full((hd,), 3.25), torch.zeros(hd), -torch.zeros(hd), torch.full((hd,), 1e-40), torch.linspace(0, 15, hd).round(), torch.linspace(-7.5, 7.5, hd),
            torch.cat([torch.zeros(hd - 1), torch.tensor([NAN])]), torch.cat([torch.tensor([INF]), torch.ones(hd - 1)]), torch.cat([torch.tensor([-INF, INF]), torch.ones(hd - 2)]),
            torch.cat([torch.tensor([3e38, -3e38]), torch.zeros(hd - 2)]), torch.cat([torch.tensor([3e38, -1e37]), torch.zeros(hd - 2)]),
            torch.cat([torch.tensor([2e-38, 0.0]), torch.full((hd - 2,), 1e-38)]), torch.cat([torch.tensor([1e-45, 0.0]), torch.zeros(hd - 2)]), torch.cat([torch.tensor([1e6]), torch.linspace(-1, 1, hd - 1)])]
    for i, r in enumerate(rows):
        if M > 20:
            x[i + 3, i % KV] = r
    return x.to(BF)


@pytest.mark.parametrize("M,KV,hd,S", [(1, 8, 128, 256), (2, 1, 64, 16), (40, 5, 128, 16), (301, 8, 64, 64), (77, 3, 64, 80), (1000, 8, 128, 256), (5000, 2, 128, 32)])
def test_store_and_load(dev, M, KV, hd, S):
    from ssd_b200 import ops
    g = gen(M, KV, hd, S)
    pages = M // S + 3
    k, v = awkward(g, M, KV, hd), awkward(g, M, KV, hd)
    slots = torch.randperm(pages * S, generator=g)[:M].to(torch.int32)
    if M > 6:
        slots[4], slots[5], slots[6] = -1, pages * S, 2147483647
    kc, vc = plain.empty(pages, S, KV, hd, 7), plain.empty(pages, S, KV, hd, 9)
    kd, vd = kc.to(dev), vc.to(dev)
    got = ops.store_kv4(k.to(dev), v.to(dev), slots.to(dev), kd, vd, values=True)
    want = [plain.rounded(plain.put(c, hd, x, slots)) for c, x in ((kc, k), (vc, v))]
    for a, b in zip((*got, kd, vd), (*want, kc, vc)):
        same_bits(a, b)
    k2, v2 = torch.full_like(kd, 7), torch.full_like(vd, 9)
    assert ops.store_kv4(k.to(dev), v.to(dev), slots.to(dev), k2, v2) is None
    same_bits(k2, kc)
    same_bits(v2, vc)
    kr, vr = ops.load_kv4(kd, vd, slots.to(dev), hd)
    out = (slots < 0) | (slots >= pages * S)
    for a, b in ((kr, want[0]), (vr, want[1])):
        same_bits(a, b.masked_fill(out[:, None, None], 0.0))


def test_rows_apart(dev):
    """Rows of keys and values as views of a projection's output, and one row for all slots."""
    from ssd_b200 import ops
    g = gen(5)
    M, H, KV, hd, S = 37, 4, 2, 64, 16
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF)
    x = qkv.view(M, H + 2 * KV, hd)
    slots = torch.randperm(5 * S, generator=g)[:M].to(torch.int32)
    for k, v in ((x[:, H:H + KV], x[:, H + KV:]), (x[:1, H:H + KV].expand(M, KV, hd), x[:, H + KV:]), (x[::2][:9, H:H + KV], x[:9, H + KV:])):
        n = k.shape[0]
        kc, vc = plain.empty(5, S, KV, hd), plain.empty(5, S, KV, hd)
        kd, vd = kc.to(dev), vc.to(dev)
        whole = qkv.to(dev).view(M, H + 2 * KV, hd)
        up = lambda t: torch.as_strided(whole, t.shape, t.stride(), t.storage_offset())  # noqa: E731
        ops.store_kv4(up(k), up(v), slots[:n].to(dev), kd, vd)
        plain.put(kc, hd, k, slots[:n])
        plain.put(vc, hd, v, slots[:n])
        same_bits(kd, kc)
        same_bits(vd, vc)


# ---------------------------------------------------------------------------------------------------- rope_store_kv4
@pytest.mark.parametrize("M,H,KV,hd,rot,S,norm", [
    (1, 64, 8, 128, 128, 256, False), (7, 32, 8, 64, 64, 64, True), (64, 16, 8, 128, 128, 256, True), (33, 40, 8, 128, 64, 16, False), (300, 6, 2, 64, 32, 80, True),
    (5, 5, 1, 128, 16, 16, False), (9, 4, 2, 128, 128, 48, True), (700, 64, 8, 128, 128, 256, False), (2, 1, 1, 64, 48, 16, True), (2001, 20, 5, 64, 64, 64, True),
])
@pytest.mark.parametrize("values", [False, True])
def test_rope_store_kv4(dev, M, H, KV, hd, rot, S, norm, values):
    from ssd_b200 import ops
    g = gen(M, H, hd, rot, S)
    top, eps = 300, 1e-6
    pages = M // S + 3
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF)
    positions = torch.randint(0, top, (M,), generator=g)
    slots = torch.randperm(pages * S, generator=g)[:M].to(torch.int32)
    bad = torch.zeros(M, dtype=torch.bool)
    for i, at in enumerate((top, -1, 1 << 45)):
        if M > 4:
            positions[i + 1], bad[i + 1] = at, True
    if M > 6:
        slots[5], slots[6] = -1, pages * S
    qn, kn = ((1 + 0.2 * torch.randn(2, hd, generator=g)).to(BF)) if norm else (None, None)
    table = angles(top, rot)
    kc, vc = plain.empty(pages, S, KV, hd, 3), plain.empty(pages, S, KV, hd, 4)
    kd, vd = kc.to(dev), vc.to(dev)
    up = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = ops.rope_store_kv4(up(qkv), up(positions), up(slots), up(table), kd, vd, H, KV, hd, up(qn), up(kn), eps, values)
    x = qkv.view(M, H + 2 * KV, hd)
    safe = positions.masked_fill(bad, 0)
    wq, size = plain.turned(x[:, :H], safe, table, qn, eps)
    # a norm in fp32 (sum of hd squares, reciprocal root, two products: 2^-19 of the value), two products and their sum, one rounding
    slack = wq.abs() * 2 ** -8 + size * 2 ** -19
    wq = wq.masked_fill(bad[:, None, None], NAN)
    within(got[0] if values else got, wq.view(M, -1), slack.view(M, -1))
    k = plain.rounded(plain.turned(x[:, H:H + KV], safe, table, kn, eps)[0])
    at = slots.masked_fill(bad, -1)
    want = [plain.rounded(plain.put(c, hd, y, at)).masked_fill(bad[:, None, None], NAN) for c, y in ((kc, k), (vc, x[:, H + KV:]))]
    same_bits(kd, kc)
    same_bits(vd, vc)
    if values:
        same_bits(got[1], want[0])
        same_bits(got[2], want[1])


# ---------------------------------------------------------------------------------------------------- paged_attention_kv4
def a_case(g, KV, hd, S, lens, width=None, stale=True):
    """Caches of normal keys, tables; rows behind the contexts and pages of nobody are NaN."""
    table, total = tables(g, [max(n, 0) for n in lens], S, width=width)
    caches = []
    for size in (1.0, 0.5):
        cache = plain.empty(total, S, KV, hd)
        x = (torch.randn(total * S, KV, hd, generator=g) * (0.5 + torch.rand(KV, hd, generator=g)) + torch.randn(KV, hd, generator=g)) * size
        if stale:
            of = torch.zeros(total * S, dtype=torch.bool)
            for row, n in zip(table.long(), lens):
                i = torch.arange(max(n, 0))
                of[row[i // S] * S + i % S] = True
            x[~of] = NAN
        plain.put(cache, hd, x.to(BF), torch.arange(total * S))
        if stale:   # (the codes of a NaN row are zero; here they are anything)
            cache[:, :, :S * hd // 2] |= torch.where(~of.view(total, 1, S, 1).expand(total, KV, S, hd // 2), 0x5a, 0).to(torch.uint8).reshape(total, KV, -1)
        caches.append(cache)
    return caches[0], caches[1], table


ATTENTION = [
    (1, 8, 1, 128, 256, [1]), (1, 64, 8, 128, 256, [300]), (1, 32, 8, 64, 64, [1, 15, 16, 17, 63, 64, 65, 0]), (1, 6, 2, 64, 16, [33, 128, 129]), (1, 5, 1, 128, 16, [100, 7]),
    (1, 4, 4, 128, 32, [40, 500]), (2, 8, 1, 128, 256, [2, 1, 0, 257]), (7, 64, 8, 128, 256, [7, 300, 5]), (7, 8, 2, 64, 80, [200, 79]), (3, 40, 8, 128, 64, [64, 130]),
    (1, 32, 1, 64, 64, [200]), (33, 4, 2, 64, 64, [40, 100]), (5, 32, 1, 128, 48, [90, 5]), (17, 16, 8, 128, 128, [130, 17, 16]), (130, 8, 4, 64, 64, [200, 131]),
]


@pytest.mark.parametrize("Q,H,KV,hd,S,lens", ATTENTION)
def test_paged_attention_kv4(dev, Q, H, KV, hd, S, lens):
    from ssd_b200 import ops
    g = gen(Q, H, KV, hd, S)
    kc, vc, table = a_case(g, KV, hd, S, lens)
    q = torch.randn(len(lens) * Q, H, hd, generator=g).to(BF)
    got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32(lens, dev), Q, hd ** -0.5)
    within(got, *plain.attention(q, kc, vc, table, lens, Q, hd ** -0.5))


@pytest.mark.parametrize("B,Q,H,KV,hd,S,ctx", [(2, 1, 8, 1, 128, 256, 9000), (1, 1, 2, 2, 64, 64, 5000), (1, 7, 16, 2, 128, 256, 4000), (40, 1, 8, 8, 64, 16, 300), (2, 40, 8, 1, 64, 64, 2500)])
def test_long_and_many(dev, B, Q, H, KV, hd, S, ctx):
    from ssd_b200 import ops
    g = gen(B, Q, H, ctx)
    lens = [ctx - 13 * i for i in range(B)]
    kc, vc, table = a_case(g, KV, hd, S, lens)
    q = (2 * torch.randn(B * Q, H, hd, generator=g)).to(BF)
    for scale in (hd ** -0.5, -0.5, 0.0):
        got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32(lens, dev), Q, scale)
        within(got, *plain.attention(q, kc, vc, table, lens, Q, scale))


@pytest.mark.parametrize("Q,H,KV,hd,S,lens,width", [
    (1, 8, 1, 128, 256, [30000], 118), (1, 4, 2, 64, 64, [1, 0, 25000, 31, 128, 129, 4000], 400), (2, 16, 2, 128, 16, [700, 9000, 2], 5000), (1, 5, 5, 128, 256, [3000, 60, 0], 2000),
    (7, 2, 1, 64, 80, [12000, 7, 3, 333], 300), (1, 2, 2, 64, 16, [130] * 37, 4000), (8, 16, 2, 64, 64, [20000, 100, 8], 400), (7, 16, 2, 128, 256, [5000, 3, 9000], 200), (40, 8, 2, 64, 16, [4000, 50], 3000),
])
def test_shares_of_long_tables(dev, Q, H, KV, hd, S, lens, width):
    """Tables with room for much: blocks have equal stretches of all sequences' keys, which begin and end anywhere, or none; short and empty sequences between long ones."""
    from ssd_b200 import ops
    g = gen(Q, H, KV, hd, sum(lens))
    kc, vc, table = a_case(g, KV, hd, S, lens, width=width)
    q = torch.randn(len(lens) * Q, H, hd, generator=g).to(BF)
    got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32(lens, dev), Q, hd ** -0.5)
    within(got, *plain.attention(q, kc, vc, table, lens, Q, hd ** -0.5))


@pytest.mark.parametrize("Q,H", [(1, 4), (6, 16)])
def test_bad_pages_and_lengths(dev, Q, H):
    """Pages outside the cache are passed over; lengths below zero, below the new tokens and past the table."""
    from ssd_b200 import ops
    g = gen(8, Q)
    KV, hd, S, lens = 2, 64, 16, [100, 60, 40, 80, 64]
    kc, vc, table = a_case(g, KV, hd, S, lens, width=8, stale=False)
    num = kc.shape[0]
    table[0, 1], table[0, 3], table[1, 0], table[1, 3], table[2] = num, -5, 2147483647, -2147483648, -1
    lens[3], lens[4] = -7, 2147483647
    table[4, :8] = torch.randperm(num, generator=g)[:8].to(torch.int32)
    q = torch.randn(5 * Q, H, hd, generator=g).to(BF)
    got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32(lens, dev), Q, 0.3)
    want, slack = plain.attention(q, kc, vc, table, lens, Q, 0.3)
    within(got, want, slack)
    assert not want[2 * Q:4 * Q].any() and not got[2 * Q:4 * Q].any()


@pytest.mark.parametrize("Q,H", [(1, 4), (3, 8), (6, 16)])
def test_what_is_not_finite(dev, Q, H):
    """A NaN row of keys or values, or a NaN query, makes NaN of the rows that see it and of no others."""
    from ssd_b200 import ops
    g = gen(9, Q)
    KV, hd, S, n = 2, 64, 16, 70
    kc, vc, table = a_case(g, KV, hd, S, [n, n, n, n])
    bad = torch.full((1, KV, hd), NAN, dtype=BF)
    last = n - max(1, Q - 1)   # of a token that not all of the new ones see, if there are several
    for cache, b, pos in ((kc, 0, last), (vc, 1, last), (kc, 2, 5)):
        plain.put(cache, hd, bad, torch.tensor([int(table[b, pos // S]) * S + pos % S]))
    q = torch.randn(4 * Q, H, hd, generator=g).to(BF)
    q[3 * Q, H - 1, 3] = INF
    want, slack = plain.attention(q, kc, vc, table, [n] * 4, Q, 0.3)
    want.view(4 * Q, H, hd)[3 * Q, H - 1] = NAN
    got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32([n] * 4, dev), Q, 0.3)
    within(got, want, slack)
    assert torch.isnan(want).any() and (Q == 1 or not torch.isnan(want[:Q]).all())


def test_large_scores(dev):
    """References far apart between keys, warps and blocks; scores far below and above zero."""
    from ssd_b200 import ops
    g = gen(12)
    KV, hd, S, H, Q, lens = 2, 128, 64, 8, 2, [3000, 700]
    kc, vc, table = a_case(g, KV, hd, S, lens)
    q = (30 * torch.randn(4, H, hd, generator=g)).to(BF)
    got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32(lens, dev), Q, 0.4)
    within(got, *plain.attention(q, kc, vc, table, lens, Q, 0.4))


# ---------------------------------------------------------------------------------------------------- as they are used
class Step:
    """A decoder layer's part of a step: places, rotation and write, attention, over a cache that holds contexts already."""

    def __init__(self, dev, seed, lens, Q, H=8, KV=2, hd=64, S=16):
        g = gen(seed, Q)
        self.Q, self.H, self.KV, self.hd, self.S, self.lens, self.B = Q, H, KV, hd, S, lens, len(lens)
        self.kc, self.vc, table = a_case(g, KV, hd, S, lens, width=max(lens) // S + 3)
        n = self.kc.shape[0]
        self.kc, self.vc = (torch.cat([c, plain.empty(2 * self.B + 1, S, KV, hd, 255)]) for c in (self.kc, self.vc))
        self.table, self.M = table, self.B * Q
        self.qkv = torch.randn(self.M, (H + 2 * KV) * hd, generator=g).to(BF)
        self.angles = angles(max(lens) + Q, hd)
        self.dev = {k: getattr(self, k).to(dev) for k in ("kc", "vc", "table", "qkv", "angles")}
        self.free, self.ctx, self.new, self.used = (i32(x, dev) for x in (list(range(n, n + 2 * self.B + 1)), lens, [Q] * self.B, [0]))

    def run(self):
        from ssd_b200 import ops
        d = self.dev
        positions, slots, _, _, lens, _ = ops.place_tokens(self.ctx, self.new, d["table"], self.free, self.used, self.M, self.S, self.kc.shape[0])
        q = ops.rope_store_kv4(d["qkv"], positions, slots, d["angles"], d["kc"], d["vc"], self.H, self.KV, self.hd).view(self.M, self.H, self.hd)
        return ops.paged_attention_kv4(q, d["kc"], d["vc"], d["table"], lens, self.Q, 0.125), q, slots

    def want(self, q, slots):
        """Attention in 64 bits for the device's own queries and places."""
        kc, vc = self.kc.clone(), self.vc.clone()
        x = self.qkv.view(self.M, -1, self.hd)
        positions = torch.cat([torch.arange(n, n + self.Q) for n in self.lens])
        plain.put(kc, self.hd, plain.rounded(plain.turned(x[:, self.H:self.H + self.KV], positions, self.angles, None, 0)[0]), slots.cpu())
        plain.put(vc, self.hd, x[:, self.H + self.KV:], slots.cpu())
        same_bits(self.dev["kc"], kc)
        same_bits(self.dev["vc"], vc)
        return plain.attention(q.cpu(), kc, vc, self.dev["table"].cpu(), [n + self.Q for n in self.lens], self.Q, 0.125)


@pytest.mark.parametrize("Q,lens", [(1, [5, 64, 31]), (4, [100, 15]), (7, [0, 300])])
def test_a_step(dev, Q, lens):
    s = Step(dev, 30, lens, Q)
    out, q, slots = s.run()
    within(out, *s.want(q, slots))


def test_prompt_on_its_own_values(dev):
    """What a write returns is what the cache holds: attention of a prompt over its values is attention over the cache."""
    from ssd_b200 import ops
    g = gen(33)
    M, H, KV, hd, S = 50, 8, 2, 64, 16
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF).to(dev)
    kc, vc = ops.kv4_caches(5, S, KV, hd, dev)
    table = i32([[3, 0, 4, 1]], dev)
    pos = torch.arange(M, device=dev)
    slots = (table[0, pos // S] * S + pos % S).to(torch.int32)
    q, k, v = ops.rope_store_kv4(qkv, pos, slots, angles(M, hd).to(dev), kc, vc, H, KV, hd, values=True)
    same_bits(k, ops.load_kv4(kc, vc, slots, hd)[0])
    same_bits(v, ops.load_kv4(kc, vc, slots, hd)[1])
    got = ops.paged_attention_kv4(q.view(M, H, hd), kc, vc, table, i32([M], dev), M, 0.125)
    k2, v2 = (torch.zeros(5, S, KV, hd, dtype=BF, device=dev) for _ in range(2))
    k2.view(-1, KV, hd)[slots.long()], v2.view(-1, KV, hd)[slots.long()] = k, v
    other = ops.paged_attention(q.view(M, H, hd), k2, v2, table, i32([M], dev), M, 0.125).double()
    # values rounded to bf16 against not: 2^-8 of a value, of a key through scores of up to eight or so; outputs' and weights' roundings
    assert float((got.double() - other).abs().max()) < 0.08 and float((got.double() - other).norm() / other.norm()) < 0.02


def test_streams_and_graphs(dev):
    """Two captured graphs, replayed with changed inputs on streams of their own, beside eager calls."""
    a, b = Step(dev, 40, [64, 20], 1), Step(dev, 41, [90, 333], 6)
    want = [s.run()[0].clone() for s in (a, b)]
    tables_ = [s.dev["table"].clone() for s in (a, b)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in (a, b):
        s.dev["table"].copy_(s.table.to(dev))
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(s.run()[0])
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s in (a, b):
            s.dev["table"].copy_(s.table.to(dev))
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for o, w, s, t in zip(outs, want, (a, b), tables_):
            assert torch.equal(o, w) and torch.equal(s.dev["table"], t)


def test_offsets_past_32_bits(dev):
    """A cache of more than 2^32 bytes: its last pages are as good as its first."""
    from ssd_b200 import ops
    g = gen(50)
    S, KV, hd, H = 256, 8, 128, 16
    pages = 33000   # 33000 * 8 * 17408 = 4.6e9 bytes
    kc, vc = ops.kv4_caches(pages, S, KV, hd, dev)
    k, v = torch.randn(2, 700, KV, hd, generator=g).to(BF)
    table = torch.tensor([[32999, 5, 32001]], dtype=torch.int32)
    pos = torch.arange(700)
    slots = (table[0, pos // S] * S + pos % S).to(torch.int32)
    ops.store_kv4(k.to(dev), v.to(dev), slots.to(dev), kc, vc)
    small = [plain.empty(3, S, KV, hd) for _ in range(2)]
    want = [plain.rounded(plain.put(c, hd, x, pos)) for c, x in zip(small, (k, v))]
    for c, s in ((kc, small[0]), (vc, small[1])):
        same_bits(c[table[0].long().to(dev)], s)
    for a, b in zip(ops.load_kv4(kc, vc, slots.to(dev), hd), want):
        same_bits(a, b)
    for Q in (1, 5):
        q = torch.randn(Q, H, hd, generator=g).to(BF)
        got = ops.paged_attention_kv4(q.to(dev), kc, vc, table.to(dev), i32([700], dev), Q, 0.088)
        within(got, *plain.attention(q, *small, torch.tensor([[0, 1, 2]], dtype=torch.int32), [700], Q, 0.088))
    assert not kc[6:32000].any()


def test_same_bits_every_time(dev):
    s = Step(dev, 60, [700, 33, 1], 3)
    first = s.run()[0].clone()
    for _ in range(5):
        s.dev["table"].copy_(s.table.to(dev))
        assert torch.equal(s.run()[0], first)


def test_refusals_leave_the_device_alone(dev):
    from ssd_b200 import ops
    s = Step(dev, 61, [64, 20], 1)
    kc, vc, q = s.dev["kc"], s.dev["vc"], torch.zeros(2, s.H, s.hd, dtype=BF, device=dev)
    with pytest.raises(RuntimeError, match="scale"):
        ops.paged_attention_kv4(q, kc, vc, s.dev["table"], s.ctx, 1, INF)
    with pytest.raises(ValueError, match="block_tables"):
        ops.paged_attention_kv4(q, kc, vc, s.dev["table"].cpu(), s.ctx, 1, 1.0)
    odd = torch.zeros(2 * s.KV * s.hd + 1, dtype=BF, device=dev)[1:].view(2, s.KV, s.hd)
    with pytest.raises(RuntimeError, match="16 bytes"):
        ops.store_kv4(odd, odd, i32([0, 1], dev), kc, vc)
    with pytest.raises(RuntimeError, match="lies over"):
        ops.store_kv4(q[:, :2], q[:, :2], i32([0, 1], dev), kc, kc)
    assert math.isfinite(float(s.run()[0].float().sum()))


# ---------------------------------------------------------------------------------------------------- more than sixteen rows to a key head
@pytest.mark.parametrize("Q,H,KV,hd,S,lens,width", [
    (9, 16, 2, 128, 16, [500, 9, 100, 0], None), (33, 4, 2, 128, 48, [90, 33, 4], None), (300, 8, 1, 128, 64, [300, 700], None), (3, 6, 1, 128, 112, [113, 64, 2], None),
    (5, 32, 1, 64, 32, [63, 65], None), (16, 16, 2, 128, 80, [6000, 16, 0, 300], 200), (11, 9, 1, 128, 256, [256, 20000, 257], 100), (2, 32, 1, 128, 16, [1] * 9 + [700], 2000), (6, 3, 1, 64, 16, [48] * 40, 1500),
])
def test_tiles(dev, Q, H, KV, hd, S, lens, width):
    """One tile and several, rows that lie in one twice or not, clusters and equal stretches; pages that end inside a chunk of keys, holes in tables."""
    from ssd_b200 import ops
    g = gen(70, Q, H, KV, hd, S)
    kc, vc, table = a_case(g, KV, hd, S, lens, width=width)
    for b in range(0, len(lens), 2):
        if lens[b] > 3 * S:
            table[b, 1] = -1 - b
    q = torch.randn(len(lens) * Q, H, hd, generator=g).to(BF)
    for scale in (hd ** -0.5, -0.2):
        got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32(lens, dev), Q, scale)
        within(got, *plain.attention(q, kc, vc, table, lens, Q, scale))


@pytest.mark.parametrize("Q,H,hd", [(1, 4, 128), (8, 8, 128), (20, 8, 64)])
def test_largest_numbers(dev, Q, H, hd):
    """Rows up to bf16's largest number, whose scale is rounded up so far that code 15 would pass it: a query of zeros has their mean."""
    from ssd_b200 import ops
    top, low = 255 * 2.0 ** 120, 5 * 2.0 ** 119
    scale = float(torch.tensor((top - low) / 15).to(BF))
    assert 15 * scale + low >= 511 * 2.0 ** 119   # what fp32 rounds to bf16's infinity
    n, S = 40, 16
    x = torch.ones(n, 1, hd)
    x[7, 0, ::2], x[7, 0, 1::2] = top, low
    x = x.to(BF).to(dev)
    kc, vc = ops.kv4_caches(5, S, 1, hd, dev)
    ops.store_kv4(x, x, i32(range(n), dev), kc, vc)
    got = ops.paged_attention_kv4(torch.zeros(Q, H, hd, dtype=BF, device=dev), kc, vc, i32([[0, 1, 2, 3, 4]], dev), i32([n + Q - 1], dev), Q, 1.0).double().cpu().view(Q, H, hd)
    x = x.double().cpu()[:, 0]
    for j in range(Q):
        rows = n + j   # those behind the n that are stored are zero
        want = x.sum(0) / rows
        # half a code, a scale that is a step off (15 2^-7 of it), a weight and the output rounded
        assert ((got[j] - want).abs() <= (scale / 2 + 15 * scale * 2 ** -7) / rows + want * 2 ** -7).all()


def test_a_wait_that_ran_out_is_reported_once(dev):
    """The word that a bounded wait would set is set by the host here: calls on tiles look at it, the others leave it."""
    from ssd_b200 import lib
    word = lib.load().ssdk_debug_op_wait_word()
    s, few = Step(dev, 71, [300, 64], 6, H=16), Step(dev, 72, [300, 64], 1)
    s.run()
    torch.cuda.synchronize()
    word[0] = 1
    few.run()
    assert word[0] == 1
    with pytest.raises(RuntimeError, match="ran out"):
        s.run()
    assert word[0] == 0
    s.dev["table"].copy_(s.table.to(dev))
    s.run()


@pytest.mark.parametrize("Q", [1, 7])
def test_calls_at_once(dev, Q):
    """Calls with parts of their own on streams of their own, over the same cache, and one whose inputs another stream has just written."""
    from ssd_b200 import ops
    g = gen(73, Q)
    KV, hd, S, lens = 2, 128, 64, [9000, 5, 700]
    kc, vc, table = (t.to(dev) for t in a_case(g, KV, hd, S, lens, width=400))
    qs = [torch.randn(3 * Q, 16, hd, generator=g).to(BF).to(dev) for _ in range(3)]
    lens = i32(lens, dev)
    want = [ops.paged_attention_kv4(q, kc, vc, table, lens, Q, 0.1).clone() for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for q, st in zip(qs, streams):
            with torch.cuda.stream(st):
                got.append(ops.paged_attention_kv4(q, kc, vc, table, lens, Q, 0.1))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    with torch.cuda.stream(streams[0]):
        torch.cuda._sleep(20000000)
        late = qs[0].clone()
        ready = torch.cuda.Event()
        ready.record()
    torch.cuda.current_stream().wait_event(ready)
    got = ops.paged_attention_kv4(late, kc, vc, table, lens, Q, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
