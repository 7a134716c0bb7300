"""Operators around a long paged cache on the GPU at their edges: scales of zero."""
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
