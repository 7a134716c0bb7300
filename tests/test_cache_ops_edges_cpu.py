"""Refusals of the operators around a long paged cache that need no GPU."""
import os
import subprocess
import sys

import pytest
import torch

from tests.cache_ops_util import BF

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096   # an address that no call below gets to use


def _refused(name, args, text):
    from ssd_b200 import lib
    so = lib.load()
    assert len(args) == len(lib.SIGNATURES[name][1])
    assert getattr(so, name)(*args) < 0
    got = so.ssdk_last_error().decode()
    assert text in got, got


@pytest.mark.parametrize("scale", [2.4e38, -3e38])
def test_scales_past_32_bits_in_base_2(scale):
    """Scores are scaled by scale log2(e): where that is infinite a score of 0 would be NaN."""
    for q_len in (1, 40):
        _refused("ssdk_span_attn", [P * i for i in range(1, 8)] + [2, q_len, 4, 2, 64, 32, 2, 4, 16, 3, scale, None], "scale")


# (arguments, {index: bytes} of the arrays that are written, of those that are read, pairs that may be one array)
M = 1 << 20
APART = {
    "ssdk_place_tokens": ([M * i for i in range(1, 12)] + [2, 4, 8, 6, 16, 8, None], {2: 32, 5: 48, 6: 24, 7: 24, 8: 12, 9: 8, 10: 4}, {0: 8, 1: 8, 3: 32, 4: 4}, ()),
    "ssdk_rope_axes_store_kv": ([M, 2 * M, 2, bytes(32), 3 * M, 4 * M, 10, 64, 5 * M, 6 * M, 1e-6, 7 * M, 8 * M, 9 * M, 32, 3, 2, 1, 64, None],
                                {11: 768, 12: 4096, 13: 4096}, {0: 1536, 1: 48, 4: 12, 5: 2560, 8: 128, 9: 128}, ()),
    "ssdk_span_bounds": ([M, 2 * M, 3 * M, 4 * M, 2, 1, 2, 64, 32, 2, 4, 16, None], {3: 4096}, {0: 32768, 1: 16, 2: 8}, ()),
    "ssdk_select_spans": ([M, 2 * M, 3 * M, 4 * M, 5 * M, 6 * M, 2, 1, 4, 2, 64, 32, 2, 4, 16, 3, 1, 1, None], {4: 48, 5: 192}, {0: 1024, 1: 4096, 2: 16, 3: 8}, ()),
    "ssdk_span_attn": ([M, 2 * M, 3 * M, 4 * M, 5 * M, 6 * M, 7 * M, 2, 1, 4, 2, 64, 32, 2, 4, 16, 3, 0.1, None], {6: 1024}, {0: 1024, 1: 32768, 2: 32768, 3: 16, 4: 8, 5: 48}, ((6, 0),)),
}


@pytest.mark.parametrize("name", sorted(APART))
def test_outputs_over_other_arrays(name):
    """Every output beside every other array of a call: sharing its first or its last sixteen bytes is refused."""
    from ssd_b200 import lib
    so = lib.load()
    good, written, read, one = APART[name]
    sizes = {**read, **written}
    for w in written:
        for other in sizes:
            if other == w:
                continue
            for at in (good[other], good[other] + (sizes[other] - 1) // 16 * 16, good[other] - (written[w] - 1) // 16 * 16):
                args = list(good)
                args[w] = at
                if (w, other) in one and at == good[other]:
                    continue
                _refused(name, args, "of its own")
    if name == "ssdk_rope_axes_store_kv":   # (more slots and positions than an address space holds: the bytes are counted without passing 64 bits)
        _refused(name, [*good[:6], 1 << 61, *good[7:13], 8 * M + 16, 1 << 61, *good[15:]], "of its own")
    if name == "ssdk_select_spans":
        assert so.ssdk_select_spans_scratch_bytes(2, 2, 32, 2, 16) == written[5]


def test_import_without_the_private_names():
    """A PyTorch that lacks the two private functions of its CUDA build (one without CUDA does) imports the module, and a call says what it needs."""
    code = """
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
from ssd_b200 import ops
one = torch.zeros(1, dtype=torch.int32)
try:
    ops.place_tokens(one, one, one[None], one, one, 1, 16, 1)
except RuntimeError as e:
    assert "CUDA" in str(e), e
else:
    raise SystemExit("no error")
"""
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]


@pytest.mark.parametrize("far", [(1 << 32) + 16, -(1 << 32) + 16])
def test_numbers_past_32_bits(far):
    """Whole numbers that the library's 32 bits would hold as another one (16)."""
    from ssd_b200 import ops
    ints = lambda *shape: torch.ones(*shape, dtype=torch.int32)  # noqa: E731
    place = dict(context_lens=ints(2), new_lens=ints(2), block_tables=ints(2, 4), free_blocks=ints(8), free_used=ints(1), rows=16, block_size=16, num_blocks=8)
    cache, both = torch.zeros(4, 32, 2, 64, dtype=BF), torch.zeros(4, 1, 2, 2, 64, dtype=BF)
    q, lens, table = torch.zeros(2, 4, 64, dtype=BF), ints(2), ints(2, 2)
    select = dict(q=q, bounds=both, block_tables=table, context_lens=lens, q_len=1, block_size=16, count=16, first=0, last=0)
    attend = dict(q=q, k_cache=cache, v_cache=cache.clone(), block_tables=table, context_lens=lens, spans=ints(2, 2, 16), span=16, q_len=1, scale=1.0)
    bound = dict(bounds=both, k_cache=cache, block_tables=table, context_lens=lens, new_tokens=16)
    for call, args, names in ((ops.place_tokens, place, ("rows", "block_size")), (ops.select_spans, select, ("block_size", "count", "first", "last")), (ops.span_attention, attend, ("span",)),
                              (ops.span_bounds, bound, ("new_tokens",))):
        for name in names:
            if name == "new_tokens" and far > 0:   # more new tokens than there are cost time only
                continue
            with pytest.raises(ValueError, match="32 bits"):
                call(**{**args, name: far})
