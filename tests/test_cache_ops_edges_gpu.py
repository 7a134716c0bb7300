"""Operators around a long paged cache on the GPU at their edges: what is not finite in every form of the selection, scales of zero, scores of minus infinity, outputs over queries."""
import pytest
import torch

from tests import cache_ops_plain as plain
from tests.cache_ops_util import BF, gen, tables, within

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    from ssd_b200 import lib
    lib.load()
    return torch.device("cuda:0")


def _select(dev, q, both, table, lens, q_len, S, count, first=1, last=0):
    from ssd_b200 import ops
    got = ops.select_spans(q.to(dev), both.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), q_len, S, count, first, last)
    want = plain.select(q, both, table, lens, q_len, S, count, first, last)
    assert torch.equal(got.cpu(), want)
    return want


def _whole(g, total, subs, KV, hd):
    """Bounds of whole numbers (many equal scores), the smaller one first."""
    return torch.randint(-1, 2, (total, subs, KV, 2, hd), generator=g).to(BF).sort(3).values.contiguous()


# q_len, H over KV: rows to a key head with and without a remainder of eight
ROWS = [(3, 6, 2), (5, 4, 2), (2, 16, 2), (7, 8, 1), (9, 1, 1)]


# ---------------------------------------------------------------------------------------------------- select_spans
@pytest.mark.parametrize("q_len,H,KV", ROWS)
def test_select_spans_many_rows_ties_and_odd_values(dev, q_len, H, KV):
    """More than eight rows to a key head: equal scores, zeros of both signs, NaN and infinities in bounds and in single rows of the queries."""
    g = gen(51, q_len, H)
    S, span, hd = 64, 16, 64
    lens = [40 * span, 40 * span - 3, 17]
    table, total = tables(g, lens, S)
    for kind in range(7):
        q = torch.randint(-1, 2, (3 * q_len, H, hd), generator=g).to(BF)
        both = _whole(g, total, S // span, KV, hd)
        if kind == 1:
            both.zero_()
        if kind == 2:
            both = torch.where(both == 0, torch.tensor(-0.0, dtype=BF), both) * 0
        if kind == 3:
            both[:, 1, 0, 1, 5] = INF
            both[:, 2, 0, :, 7] = -INF
        if kind == 4:
            both[::2, 3, KV - 1, 0, 9] = NAN
            both[1::2, 0, KV - 1, 1, 63] = INF
        if kind == 5:
            q[q_len - 1, H - 1, 2] = INF   # the first sequence's last row
            q[q_len, 0, 0] = NAN           # the second one's first
            both = both * 3e38
        if kind == 6:
            q[0, 0, 3] = -INF
        for count in (3, 11, 39):
            _select(dev, q, both, table, lens, q_len, S, count)


@pytest.mark.parametrize("q_len,H,KV", [(1, 4, 2), (5, 4, 2)])
@pytest.mark.parametrize("kind", ["few", "infinite", "nan", "query"])
def test_select_spans_odd_values_of_long_contexts(dev, q_len, H, KV, kind):
    """Where something is not finite all spans' scores are made in 64 bits, and of more than 256 the line is found bit by bit: between NaN, infinities of both signs, equal and finite scores."""
    g = gen(52, q_len, len(kind))
    S, span, hd, n = 64, 16, 64, 700
    lens = [n * span, 513 * span - 1, 300 * span]
    table, total = tables(g, lens, S)
    q = torch.randint(-1, 2, (3 * q_len, H, hd), generator=g).to(BF)
    both = _whole(g, total, S // span, KV, hd)
    at = torch.rand(total, S // span, KV, generator=g)
    if kind == "few":
        both[..., 1, 7] = torch.where(at < 0.02, INF, both[..., 1, 7].float()).to(BF)
        both[..., 0, 8] = torch.where(at > 0.99, NAN, both[..., 0, 8].float()).to(BF)
    if kind == "infinite":   # of half of the spans the score is an infinity of one sign or the other, or NaN
        both[..., 1, 7] = torch.where(at < 0.3, INF, both[..., 1, 7].float()).to(BF)
        both[..., 9] = torch.where(at[..., None] > 0.8, -INF, both[..., 9].float()).to(BF)
    if kind == "nan":
        both[..., 1, 7] = torch.where(at < 0.6, NAN, both[..., 1, 7].float()).to(BF)
    if kind == "query":
        q[0, 0, 3], q[q_len, H - 1, 5] = INF, NAN
    for count in (1, 5, 50, 333, 650):
        _select(dev, q, both, table, lens, q_len, S, count)


@pytest.mark.parametrize("width", [10, 300])
@pytest.mark.parametrize("q_len,H,KV", ROWS[:2])
def test_select_spans_many_rows_bad_pages(dev, q_len, H, KV, width):
    g = gen(53, q_len)
    S, span, hd = 32, 16, 64
    lens = [300, 299, -4, 100000]
    table, total = tables(g, [300, 299, 0, 320], S, width=width)
    table[0, 2], table[0, 5], table[1, 0], table[1, 9], table[3, 4] = total, -9, 2147483647, -2147483648, total + 1
    q = torch.randn(4 * q_len, H, hd, generator=g).to(BF)
    both = torch.randn(total, 2, KV, 2, hd, generator=g).sort(3).values.to(BF).contiguous()
    for count in (4, 30):
        got = _select(dev, q, both, table, lens, q_len, S, count, 2, 2)
        assert 4 not in got[0].tolist()
    both[table[0, 1], 0, 0, 1, 5] = NAN
    _select(dev, q, both, table, lens, q_len, S, 5, 2, 2)


# ---------------------------------------------------------------------------------------------------- span_attention
def _attention(dev, q, kc, vc, table, lens, spans, span, q_len, scale):
    from ssd_b200 import ops
    return ops.span_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), spans.to(dev), span, q_len, scale)


@pytest.mark.parametrize("q_len,H,hd", [(1, 4, 128), (3, 8, 64), (6, 16, 128), (9, 8, 64)])
@pytest.mark.parametrize("scale", [0.0, -0.0])
def test_span_attention_scale_zero(dev, q_len, H, hd, scale):
    """0 times NaN or an infinity is NaN, in queries and in keys, on both kinds of kernel; what a row does not see, and all that is finite, has equal weights."""
    g = gen(61, q_len, H)
    S, span, KV = 64, 16, 2
    lens = [200, 70, 700, 129]
    table, total = tables(g, lens, S)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    q = torch.randn(len(lens) * q_len, H, hd, generator=g).to(BF)
    spans = torch.tensor([[0, 1, 2, 3, 12, -1], [4, 0, 1, 2, -1, -1], [43, 0, 7, 20, 30, 31], [8, 7, 0, 1, 2, 3]], dtype=torch.int32)[:, None].expand(4, KV, 6).contiguous()
    kc[table[3, 2], 1:] = NAN   # behind the context
    got = _attention(dev, q, kc, vc, table, lens, spans, span, q_len, scale)
    within(got, *plain.attention(q, kc, vc, table, lens, spans, span, q_len, scale))
    assert bool(torch.isfinite(got.float()).all())
    q[0, 0, 3], q[q_len, 1, 5], q[q_len, H - 1, 6] = NAN, INF, -INF
    kc[table[2, 0], 3, 0, 7], kc[table[2, 10], 6, 1, 8] = INF, -INF   # tokens 3 and 646 (span 40: not listed)
    kc[table[2, 10], 59, 1, 9] = -INF                                # token 699, the last: only the last query sees it
    got = _attention(dev, q, kc, vc, table, lens, spans, span, q_len, scale)
    want, slack = plain.attention(q, kc, vc, table, lens, spans, span, q_len, scale)
    assert bool(torch.isnan(want).any())
    within(got, want, slack)


@pytest.mark.parametrize("q_len,H,B", [(1, 4, 1), (1, 4, 40), (3, 4, 7), (6, 16, 2), (70, 16, 3)])
def test_span_attention_over_its_queries(dev, q_len, H, B):
    """out may be q itself: with a block and with several to a key head, and with tiles of a sequence's rows."""
    from ssd_b200 import lib, ops
    g = gen(63, q_len, B)
    S, span, KV, hd = 64, 16, 2, 64
    lens = [q_len + 190 + 7 * i for i in range(B)]
    table, total = tables(g, lens, S)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF).to(dev)
    q = torch.randn(B * q_len, H, hd, generator=g).to(BF).to(dev)
    spans = torch.arange(11, dtype=torch.int32).expand(B, KV, 11).contiguous().to(dev)
    table, lens = table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    want = ops.span_attention(q, kc, vc, table, lens, spans, span, q_len, 0.125)
    so = lib.load()
    assert so.ssdk_span_attn(q.data_ptr(), kc.data_ptr(), vc.data_ptr(), table.data_ptr(), lens.data_ptr(), spans.data_ptr(), q.data_ptr(), B, q_len, H, KV, hd, S, table.shape[1], total,
                             span, 11, 0.125, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(q.view_as(want), want)


def test_the_public_names_do_as_well(dev, monkeypatch):
    """Where PyTorch has no private functions for the current device and stream the public ones are called: on the default stream and on another."""
    from ssd_b200 import ops
    args = [torch.tensor(v, dtype=torch.int32, device=dev) for v in ([5, 20], [3, 1], [[0, -1], [2, 3]], [1, 4, 5], [0])]
    want = [t.clone() for t in ops.place_tokens(*args, 6, 16, 6)]
    monkeypatch.setattr(ops, "_gpu_now", torch.cuda.current_device)
    monkeypatch.setattr(ops, "_stream_of", lambda gpu: torch.cuda.current_stream(gpu).cuda_stream)
    torch.cuda.synchronize()
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            got = ops.place_tokens(*args, 6, 16, 6)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("q_len,H", [(1, 4), (6, 16)])
def test_span_attention_scores_of_minus_infinity(dev, q_len, H):
    """A score of minus infinity has the weight 0; a row that has no other is zero, as one that sees no key."""
    g = gen(62, q_len)
    S, span, KV, hd = 64, 16, 2, 128
    lens = [200, 70]
    table, total = tables(g, lens, S)
    kc, vc = torch.randn(2, total, S, KV, hd, generator=g).to(BF)
    q = torch.randn(len(lens) * q_len, H, hd, generator=g).to(BF)
    q[..., 4] = q[..., 4].abs() + 1
    spans = torch.tensor([[0, 1, 5, 12], [0, 2, 3, 4]], dtype=torch.int32)[:, None].expand(2, KV, 4).contiguous()
    kc[table[0, :2].long(), :, 0, 4] = -INF   # tokens 0 to 127: all that is listed but the last span
    kc[table[1].long(), :, 1, 4] = -INF       # every token
    got = _attention(dev, q, kc, vc, table, lens, spans, span, q_len, 0.09).view(len(lens), q_len, KV, -1)
    want, slack = (t.view(len(lens), q_len, KV, -1) for t in plain.attention(q, kc, vc, table, lens, spans, span, q_len, 0.09))
    assert bool(torch.isnan(want[1, :, 1]).all()) and not bool(got[1, :, 1].any())
    rest = ~torch.isnan(want)
    within(got.cpu()[rest], want[rest], slack[rest].nan_to_num(0.0))
