"""The paged cache held in 4 bits on the GPU, where it can go wrong: rows at the borders of codes and of bf16 against the definition in fractions (tests/kv4_exact.py)."""
import pytest
import torch

from tests import kv4_exact as exact
from tests.test_kv4_gpu import i32, same_bits

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
