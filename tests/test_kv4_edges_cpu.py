"""The paged cache held in 4 bits without a GPU, where it can go wrong: the order of hand-offs in its sources; the sources of
kv4_store_kernel and kv4_load_kernel on host threads against the definition in fractions, on rows at the borders of codes and of bf16."""
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from tests import kv4_exact as exact
from tests.cache_ops_util import BF
from tests.test_kv4_cpu import _run, _take, i32, needs_gxx
from tests.test_kv4_gpu import same_bits

CSRC = Path(__file__).resolve().parent.parent / "ssd_b200" / "csrc"


def _source(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


# ---------------------------------------------------------------------------------------------------- order
def test_positions_are_written_before_their_chunk_is_announced():
    """Four lanes of the copying warp write where a chunk's keys are, one lane arrives for all of them: a vote orders no memory, so a barrier of the warp stands between them."""
    body = _source("kv4_tiles.cuh")
    written = [m.end() for m in re.finditer(r"codes_pos\[c\]\[lane\]\s*=", body)]
    arrives = [m.start() for m in re.finditer(r"mbar_arrive_expect_tx\(&codes_full", body)]
    assert len(written) == len(arrives) == 1
    between = body[written[0]:arrives[0]]
    assert "__syncwarp()" in between and between.rindex("__syncwarp()") < between.rindex("if (lane == 0)")


# ---------------------------------------------------------------------------------------------------- codes and values
def _stored(tmp_path, x, values):
    """Rows x [M, 1, hd] stored as keys and as values by the kernel's source: caches (and values) as it leaves them."""
    M, KV, hd = x.shape
    pages = -(-M // 16)
    data = _run("store", [i32([M, 0, KV, hd, 0, 0, 16, pages, 0, int(values), 16]), np.float32([0]), np.zeros(M, np.int64), torch.arange(M, dtype=torch.int32), torch.zeros(2 * hd, dtype=BF),
                          torch.cat([x, x], 1), torch.zeros(2, pages, KV, 16 * (hd // 2 + 4), dtype=torch.uint8)], tmp_path)
    return _take(data, *[(torch.uint8, (pages, KV, 16 * (hd // 2 + 4)))] * 2, *[(BF, (M, KV, hd))] * (2 * values))


@needs_gxx
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [exact.far_below_borders, exact.every_scale])
def test_codes_at_borders(tmp_path, rows, hd):
    x = rows(hd)
    want, _ = exact.cache_of(x, range(len(x)), -(-len(x) // 16), 16)
    for got in _stored(tmp_path, x, False):
        same_bits(got, want)


@needs_gxx
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [exact.rounded_twice, exact.far_below_borders])
def test_values_are_rounded_once(tmp_path, rows, hd):
    """What a write returns and a read gives is scale x code + minimum rounded to bf16, not to fp32 first."""
    x = rows(hd)
    M, pages = len(x), -(-len(x) // 16)
    cache, want = exact.cache_of(x, range(M), pages, 16)
    for got in _stored(tmp_path, x, True)[2:]:
        same_bits(got, want)
    data = _run("load", [i32([M, 1, hd, 16, pages, 2]), cache, cache, torch.arange(M, dtype=torch.int32)], tmp_path)
    for got in _take(data, *[(BF, (M, 1, hd))] * 2):
        same_bits(got, want)


# ---------------------------------------------------------------------------------------------------- refusals
def test_too_many_heads_of_rows_are_refused_by_their_own_name():
    """More groups of heads than 32 bits count, arrays far apart: the call that is refused says who it is."""
    from ssd_b200 import lib
    so, P = lib.load(), 1 << 50   # addresses that no call gets to use
    rope = [P, 2 * P, 3 * P, 4 * P, 100, 64, None, None, 1e-6, *(P * i for i in range(5, 10)), 2, 16, 1 << 20, 65535, 1, 64, None]
    rows = [P, 2 * P, 64 * 65535, 64 * 65535, *(P * i for i in range(3, 8)), 2, 16, 1 << 20, 65535, 64, None]
    for name, args in (("rope_store_kv4", rope), ("store_kv4", rows)):
        assert getattr(so, "ssdk_" + name)(*args) != 0
        assert so.ssdk_last_error().decode().startswith(name + ": 1048576 rows of "), so.ssdk_last_error()


@pytest.mark.parametrize("sizes", [(1 << 20, 2048, 1, 64), (2, 65552, 1, 128), (2, 16, 65536, 64)])
def test_caches_that_no_operator_takes_are_not_made(sizes):
    """Slots past 32 bits, pages of more than 65536 tokens, more than 65535 heads: refused before memory is asked for, as the operators refuse them."""
    from ssd_b200 import ops
    with pytest.raises(ValueError, match="kv4_caches"):
        ops.kv4_caches(*sizes, device="meta")
    assert ops.kv4_caches((1 << 20) - 1, 2048, 1, 64, device="meta")[1].shape == ((1 << 20) - 1, 1, 2048 * 36)
