"""The sources of span_estimate_kernel and span_pick_kernel on host threads (AddressSanitizer watches the ends of the arrays and what lies in front of the bounds)
against the selection's definition."""
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from tests import cache_ops_plain as plain
from tests.cache_ops_util import BF, gen, tables

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "emu", "run_select_spans.cpp")
BIN = os.path.join(ROOT, "tests", "emu", "_build", "run_select_spans")
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++ (C++20)")


def _run(tmp_path, q, both, table, lens, q_len, S, count, first, last, own, warps=8, later=None):
    """The lists that the kernels make; `later`: the tables as the second of the two kernels finds them."""
    deps = [SRC] + [os.path.join(ROOT, "tests", "emu", f) for f in ("cuda_emu.h", "pairs_emu.h")] + [os.path.join(ROOT, "ssd_b200", "csrc", f) for f in ("span_ops.cuh", "cache_ops.cuh", "common.cuh")]
    if not os.path.exists(BIN) or any(os.path.getmtime(BIN) < os.path.getmtime(d) for d in deps):
        os.makedirs(os.path.dirname(BIN), exist_ok=True)
        subprocess.run(["g++", "-std=c++20", "-O1", "-fsanitize=address", "-pthread", "-Wno-unknown-pragmas", "-Wno-attributes", "-o", BIN, SRC], check=True)
    num, subs, KV, _, hd = both.shape
    B, width = table.shape
    inp, out = tmp_path / "in", tmp_path / "out"
    with open(inp, "wb") as f:
        for a in ([B, q_len, q.shape[1], KV, hd, S, S // subs, width, num, count, first, last, warps, own], table, table if later is None else later, lens):
            np.asarray(a, dtype=np.int32).tofile(f)
        for t in (q, both):
            t.contiguous().view(torch.int16).numpy().tofile(f)
    res = subprocess.run([BIN, str(inp), str(out)], capture_output=True, text=True, timeout=1800, env={**os.environ, "ASAN_OPTIONS": "detect_leaks=0"})
    assert res.returncode == 0, res.stderr[-2000:]
    return torch.from_numpy(np.fromfile(out, dtype=np.int32)).view(B, KV, count)


@pytest.mark.parametrize("zero", [True, False])
@pytest.mark.parametrize("q_len", [1, 5])
def test_pages_that_go_between_the_kernels(tmp_path, zero, q_len):
    """A table that another stream changes while a call runs is an error of the caller's; the scores in 64 bits still read no page that is not there."""
    g = gen(71, q_len)
    S, span, KV, hd, H = 32, 16, 1, 64, 2
    table, total = tables(g, [300], S, width=12)
    q = torch.randn(q_len, H, hd, generator=g).to(BF)
    both = torch.randn(total, S // span, KV, 2, hd, generator=g).sort(3).values.to(BF).contiguous()
    if zero:
        both.zero_()            # all on the line: as many as there is room for are scored and ranked
    else:
        both[:, 0, 0, 1, 3] = float("nan")   # not finite: all are scored
    later = table.clone()
    later[0, 2], later[0, 4], later[0, 7] = -1, total, -2147483648
    got = _run(tmp_path, q, both, table, [300], q_len, S, 9, 1, 1, 0, later=later)
    assert bool(((got >= 0) & (got < 19)).all()) and bool((got[..., 1:] > got[..., :-1]).all())


# one kernel, two, and two with more than eight rows to a key head
FORMS = [(1, 4, 2, 1), (1, 4, 2, 0), (5, 4, 2, 0)]


@pytest.mark.parametrize("q_len,H,KV,own", FORMS)
@pytest.mark.parametrize("kind", ["whole", "zero", "infinite", "nan", "query", "random"])
def test_select_source(tmp_path, q_len, H, KV, own, kind):
    """Equal scores, zeros of both signs, what is not finite in bounds and queries, and pages outside the cache."""
    g = gen(72, q_len, len(kind), own)
    S, span, hd, width = 32, 16, 64, 11
    lens = [310, 299, 20]
    table, total = tables(g, lens, S, width=width)
    table[0, 3], table[1, 0], table[1, 8] = total, -9, 2147483647
    q = torch.randint(-1, 2, (3 * q_len, H, hd), generator=g).to(BF)
    both = torch.randint(-1, 2, (total, S // span, KV, 2, hd), generator=g).to(BF).sort(3).values.contiguous()
    if kind == "zero":
        both = torch.where(both == 0, torch.tensor(-0.0, dtype=BF), both) * 0
    if kind == "infinite":
        both[::3, 1, 0, 1, 5] = float("inf")
        both[1::3, 0, 0, :, 7] = -float("inf")
    if kind == "nan":
        both[::2, 1, KV - 1, 0, 9] = float("nan")
    if kind == "query":
        q[q_len - 1, H - 1, 2], q[q_len, 0, 0] = float("inf"), float("nan")
        both = both * 3e38
    if kind == "random":
        q, both = torch.randn(q.shape, generator=g).to(BF), torch.randn(both.shape, generator=g).sort(3).values.to(BF).contiguous()
    for count, first, last in ((5, 1, 1), (13, 0, 0)):
        got = _run(tmp_path, q, both, table, lens, q_len, S, count, first, last, own)
        assert torch.equal(got, plain.select(q, both, table, lens, q_len, S, count, first, last))


@pytest.mark.parametrize("hd,q_len,H,KV,own,warps", [(128, 1, 3, 1, 1, 8), (128, 2, 3, 1, 0, 3), (128, 9, 2, 2, 0, 8), (64, 3, 8, 1, 0, 16)])
def test_select_source_sizes(tmp_path, hd, q_len, H, KV, own, warps):
    """Heads of 128, odd groups, warps that take several groups of spans and warps that find none; count, first and last at their ends."""
    g = gen(73, hd, q_len, H)
    S, span = 48, 16
    lens = [900, 33, 5]
    table, total = tables(g, lens, S)
    q = torch.randn(3 * q_len, H, hd, generator=g).to(BF)
    both = torch.randn(total, S // span, KV, 2, hd, generator=g).sort(3).values.to(BF).contiguous()
    for count, first, last in ((1, 0, 0), (7, 3, 4), (56, 1, 2)):
        got = _run(tmp_path, q, both, table, lens, q_len, S, count, first, last, own, warps)
        assert torch.equal(got, plain.select(q, both, table, lens, q_len, S, count, first, last))
