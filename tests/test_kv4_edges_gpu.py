"""The paged cache held in 4 bits on the GPU, where it can go wrong: rows at the borders of codes and of bf16 against the definition in fractions (tests/kv4_exact.py)."""
import pytest
import torch

from tests import kv4_exact as exact
from tests import kv4_plain as plain
from tests.cache_ops_util import BF, gen, within
from tests.test_kv4_gpu import a_case, i32, same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    from ssd_b200 import lib
    lib.load()
    return torch.device("cuda:0")


# ---------------------------------------------------------------------------------------------------- codes and values
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [exact.far_below_borders, exact.every_scale])
def test_codes_at_borders(dev, rows, hd):
    """As rows of keys and of values, and as keys at position 0, which do not turn."""
    from ssd_b200 import ops
    x, M = rows(hd), len(rows(hd))
    want, _ = exact.cache_of(x, range(M), -(-M // 16), 16)
    slots, up = i32(range(M), dev), x.to(dev)
    caches = [torch.zeros_like(want, device=dev) for _ in range(4)]
    ops.store_kv4(up, up, slots, *caches[:2])
    table = torch.cat([torch.ones(1, hd // 2), torch.zeros(1, hd // 2)], 1).to(dev)
    q = ops.rope_store_kv4(up.expand(M, 3, hd).reshape(M, 3 * hd), torch.zeros(M, dtype=torch.int64, device=dev), slots, table, *caches[2:], 1, 1, hd)
    same_bits(q, x[:, 0])
    for got in caches:
        same_bits(got, want)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [exact.rounded_twice, exact.far_below_borders, exact.every_scale])
def test_values_are_rounded_once(dev, rows, hd):
    """What writes return and a read gives is scale x code + minimum rounded to bf16, not to fp32 first."""
    from ssd_b200 import ops
    x, M = rows(hd), len(rows(hd))
    cache, want = exact.cache_of(x, range(M), -(-M // 16), 16)
    slots, up = i32(range(M), dev), x.to(dev)
    caches = [torch.zeros_like(cache, device=dev) for _ in range(2)]
    table = torch.cat([torch.ones(1, hd // 2), torch.zeros(1, hd // 2)], 1).to(dev)
    got = [*ops.store_kv4(up, up, slots, *caches, values=True)]
    got += ops.rope_store_kv4(up.expand(M, 3, hd).reshape(M, 3 * hd), torch.zeros(M, dtype=torch.int64, device=dev), slots, table, *caches, 1, 1, hd, values=True)[1:]
    got += ops.load_kv4(cache.to(dev), cache.to(dev), slots, hd)
    for v in got:
        same_bits(v, want)


# ---------------------------------------------------------------------------------------------------- sizes of values
def times(cache, hd, e):
    """The same codes, scales and minima 2^e as large."""
    S = cache.shape[2] // (hd // 2 + 4)
    out = cache.clone()
    pair = cache[:, :, S * hd // 2:].contiguous().view(BF).double() * 2.0 ** e
    out[:, :, S * hd // 2:] = pair.to(BF).view(torch.uint8)
    return out


#: few rows, more than sixteen in one tile (twice in it or once) and in several; clusters, equal stretches
FORMS = [(1, 8, 1, 128, 64, [300, 70], None), (2, 8, 1, 64, 16, [200], None), (1, 4, 1, 64, 64, [3000, 60], 2000), (7, 8, 2, 128, 64, [300, 70], None), (20, 4, 1, 64, 16, [250], None),
         (7, 8, 1, 128, 64, [3000, 60], 400), (40, 4, 1, 128, 16, [300], None)]


@pytest.mark.parametrize("Q,H,KV,hd,S,lens,width", FORMS)
@pytest.mark.parametrize("e", [-80, -96, -110, 60, 100, 120])
def test_values_of_all_sizes(dev, Q, H, KV, hd, S, lens, width, e):
    """Values 2^e as large are outputs 2^e as large, to the same number of bits."""
    from ssd_b200 import ops
    g = gen(81, Q, H, hd)
    kc, vc, table = a_case(g, KV, hd, S, lens, width=width)
    q = torch.randn(len(lens) * Q, H, hd, generator=g).to(BF)
    got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), times(vc, hd, e).to(dev), table.to(dev), i32(lens, dev), Q, hd ** -0.5)
    want, slack = plain.attention(q, kc, vc, table, lens, Q, hd ** -0.5)
    # weights times scales below 2^-126 are off by half of bf16's smallest number, 2^-134, for a code less eight; the sum of weights is one at least
    within(got.double() * 2.0 ** -e, want, slack + max(lens) * 2.0 ** (-134 + 3 - e))


@pytest.mark.parametrize("Q,H,KV,hd,S,lens,width", FORMS)
def test_large_values_among_small_ones(dev, Q, H, KV, hd, S, lens, width):
    """Rows near bf16's largest number before, among and behind rows of 2^-60 and ordinary ones: the outputs are theirs where they are seen, whatever came first."""
    from ssd_b200 import ops
    g = gen(82, Q, H, hd)
    kc, vc, table = a_case(g, KV, hd, S, lens, width=width)
    small, large = times(vc, hd, -60), times(vc, hd, 124)
    q = torch.randn(len(lens) * Q, H, hd, generator=g).to(BF)
    n = lens[0]
    for at in ([0], [n // 2], [n - 1], [33, n - 40]):
        v = small.clone()
        for i, pos in enumerate(at):
            page, off = int(table[0, pos // S]), pos % S
            for a, b in ((off * (hd // 2), hd // 2), (S * (hd // 2) + 4 * off, 4)):
                v[page, :, a:a + b] = (large if i == 0 else vc)[page, :, a:a + b]
        got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), v.to(dev), table.to(dev), i32(lens, dev), Q, hd ** -0.5)
        want, slack = plain.attention(q, kc, v, table, lens, Q, hd ** -0.5)
        far = slice(Q, None)   # (the other sequences see none of them)
        within(got, want, slack)
        within(got[far].double() * 2.0 ** 60, want[far] * 2.0 ** 60, slack[far] * 2.0 ** 60)
