"""The paged cache held in 4 bits on the GPU, where it can go wrong: rows at the borders of codes and of bf16 against the definition in fractions (tests/kv4_exact.py), values and scores of all sizes, attention on
tiles to its own roundings (tests/kv4_tiles_plain.py), calls that no other test makes."""
import pytest
import torch

from tests import kv4_exact as exact
from tests import kv4_plain as plain
from tests import kv4_tiles_plain as tiles
from tests.cache_ops_util import BF, angles, gen, within
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


@pytest.mark.parametrize("Q,H,KV,hd,S,lens,width", FORMS)
@pytest.mark.parametrize("e", [-100, -60, 100])
def test_scores_of_queries_and_keys_far_apart(dev, Q, H, KV, hd, S, lens, width, e):
    """Keys 2^e as large under queries 2^-e as large: the same scores."""
    from ssd_b200 import ops
    g = gen(86, Q, H, hd)
    kc, vc, table = a_case(g, KV, hd, S, lens, width=width)
    q = torch.randn(len(lens) * Q, H, hd, generator=g).to(BF)
    up = (q.double() * 2.0 ** -e).to(BF)   # (exact)
    got = ops.paged_attention_kv4(up.to(dev), times(kc, hd, e).to(dev), vc.to(dev), table.to(dev), i32(lens, dev), Q, hd ** -0.5)
    within(got, *plain.attention(q, kc, vc, table, lens, Q, hd ** -0.5))


# ---------------------------------------------------------------------------------------------------- attention on tiles, to its own roundings
def parts_of(B, Q, H, KV, hd, S, width):
    """Bytes that a call leaves of its parts: not zero where blocks have equal stretches of all keys."""
    from ssd_b200 import lib
    return lib.load().ssdk_paged_attn_kv4_scratch_bytes(B, Q, H, KV, hd, S, width)


@pytest.mark.parametrize("Q,H,KV,hd,S,lens,width,shared", [
    (20, 8, 2, 64, 64, [9000, 5, 0, 700], 400, True), (11, 9, 1, 64, 80, [12000, 63, 65], 200, True), (128, 1, 1, 64, 16, [6000, 300], 500, True),   # heads of 64, one tile whose rows lie in it once
    (16, 8, 1, 128, 256, [9000, 40], 80, True), (7, 8, 1, 128, 64, [8000, 9, 70], 300, True), (5, 8, 2, 64, 64, [9000, 17], 400, True),
    (20, 8, 2, 64, 64, [300, 20], None, False), (7, 8, 1, 128, 256, [700, 7, 8], None, False), (3, 32, 1, 64, 16, [100, 64], None, False), (300, 2, 1, 128, 48, [700], None, False),
    (77, 6, 2, 64, 4096, [5000, 76], None, False),
])
def test_tiles_to_their_own_roundings(dev, Q, H, KV, hd, S, lens, width, shared):
    """Over keys and values in bf16, as load_kv4 gives them, and over scale x code + minimum as they are."""
    from ssd_b200 import ops
    g = gen(83, Q, H, KV, hd, S)
    kc, vc, table = a_case(g, KV, hd, S, lens, width=width)
    assert bool(parts_of(len(lens), Q, H, KV, hd, S, table.shape[1])) == shared
    q = torch.randn(len(lens) * Q, H, hd, generator=g).to(BF)
    got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32(lens, dev), Q, hd ** -0.5)
    for rounded in (True, False):
        within(got, *tiles.attention(q, kc, vc, table, lens, Q, hd ** -0.5, rounded))


def test_a_prompt_over_what_its_write_returns(dev):
    """Rotation and write of a prompt's rows, attention over the cache: softmax over the values that the write returned, to the kernel's roundings; its last tokens again, few rows to a key head."""
    from ssd_b200 import ops
    g = gen(84)
    M, H, KV, hd, S = 150, 8, 2, 64, 16
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF).to(dev)
    kc, vc = ops.kv4_caches(12, S, KV, hd, dev)
    table = torch.randperm(12, generator=g)[:10].to(torch.int32)[None].to(dev)
    pos = torch.arange(M, device=dev)
    slots = (table[0, pos // S] * S + pos % S).to(torch.int32)
    q, k, v = ops.rope_store_kv4(qkv, pos, slots, angles(M, hd).to(dev), kc, vc, H, KV, hd, values=True)
    q = q.view(M, H, hd)
    got = ops.paged_attention_kv4(q, kc, vc, table, i32([M], dev), M, 0.125)
    few = ops.paged_attention_kv4(q[-3:], kc, vc, table, i32([M], dev), 3, 0.125)
    seen = (torch.arange(M) <= torch.arange(M)[:, None]).repeat_interleave(H // KV, 0)
    want, slack = torch.empty(2, M, H, hd, dtype=torch.float64).unbind(0)
    for h in range(KV):
        heads = slice(h * H // KV, (h + 1) * H // KV)
        out = tiles.attend(q[:, heads].double().cpu().reshape(-1, hd), k[:, h].double().cpu(), v[:, h].double().cpu(), seen, 0.125)
        for t, x in zip((want, slack), out):
            t[:, heads] = x.view(M, -1, hd)
    within(got, want.view(M, -1), slack.view(M, -1))
    within(few, *plain.attention(q[-3:].cpu(), kc.cpu(), vc.cpu(), table.cpu(), [M], 3, 0.125))


@pytest.mark.parametrize("Q,H", [(1, 2), (20, 1)])
def test_more_sequences_than_share_a_launch(dev, Q, H):
    """Beyond 1024 sequences no block goes through all lengths: clusters take long tables too."""
    from ssd_b200 import ops
    g = gen(85, Q)
    B, KV, hd, S = 1100, 1, 64, 16
    lens = [(7 * i) % 40 for i in range(B)]
    lens[3], lens[1050], lens[1099] = 900, 1500, 33
    kc, vc, table = a_case(g, KV, hd, S, lens, width=2000)
    assert parts_of(B, Q, H, KV, hd, S, 2000) == 0 and parts_of(64, Q, H, KV, hd, S, 2000) > 0
    q = torch.randn(B * Q, H, hd, generator=g).to(BF)
    got = ops.paged_attention_kv4(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), i32(lens, dev), Q, 0.125)
    within(got, *(plain.attention(q, kc, vc, table, lens, Q, 0.125) if Q == 1 else tiles.attention(q, kc, vc, table, lens, Q, 0.125, True)))


@pytest.mark.parametrize("which", ["q", "k"])
def test_one_norm_of_the_two(dev, which):
    """A norm of queries without one of keys, and the other way round."""
    from ssd_b200 import ops
    g = gen(87)
    M, H, KV, hd, S, eps = 41, 5, 2, 128, 16, 1e-5
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF)
    w = (1 + 0.2 * torch.randn(hd, generator=g)).to(BF)
    qn, kn = (w, None) if which == "q" else (None, w)
    table, positions, slots = angles(60, 64), torch.randint(0, 60, (M,), generator=g), torch.randperm(64, generator=g)[:M].to(torch.int32)
    kc, vc = plain.empty(4, S, KV, hd), plain.empty(4, S, KV, hd)
    kd, vd = kc.to(dev), vc.to(dev)
    up = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = ops.rope_store_kv4(up(qkv), up(positions), up(slots), up(table), kd, vd, H, KV, hd, up(qn), up(kn), eps)
    x = qkv.view(M, -1, hd)
    want, size = plain.turned(x[:, :H], positions, table, qn, eps)
    within(got, want.view(M, -1), (want.abs() * 2 ** -8 + size * 2 ** -19).view(M, -1))   # (test_rope_store_kv4 has the bound's parts)
    plain.put(kc, hd, plain.rounded(plain.turned(x[:, H:H + KV], positions, table, kn, eps)[0]), slots)
    plain.put(vc, hd, x[:, H + KV:], slots)
    same_bits(kd, kc)
    same_bits(vd, vc)
