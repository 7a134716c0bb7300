"""Operators around a long paged cache without a GPU: the sources of place_tokens_kernel, rope_axes_kernel and span_bounds_kernel on host threads
(AddressSanitizer watches the ends of the arrays) against their definitions, bad pages and positions among them, and the refusals of all entry points."""
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from tests import cache_ops_plain as plain
from tests.cache_ops_util import BF, PLACES, angles, gen, place_case, tables, within

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "emu", "run_cache_ops.cpp")
BIN = os.path.join(ROOT, "tests", "emu", "_build", "run_cache_ops")
needs_gxx = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++ (C++20)")


def _run(mode, parts, tmp_path):
    deps = [SRC, os.path.join(ROOT, "tests", "emu", "cuda_emu.h")] + [os.path.join(ROOT, "ssd_b200", "csrc", f) for f in ("cache_ops.cuh", "common.cuh")]
    if not os.path.exists(BIN) or any(os.path.getmtime(BIN) < os.path.getmtime(d) for d in deps):
        os.makedirs(os.path.dirname(BIN), exist_ok=True)
        subprocess.run(["g++", "-std=c++20", "-O1", "-fsanitize=address", "-pthread", "-Wno-unknown-pragmas", "-Wno-attributes", "-o", BIN, SRC], check=True)
    inp, out = tmp_path / "in", tmp_path / "out"
    with open(inp, "wb") as f:
        for a in parts:
            a = a.contiguous().view(torch.int16).numpy() if isinstance(a, torch.Tensor) and a.dtype == BF else np.ascontiguousarray(a)
            a.tofile(f)
    res = subprocess.run([BIN, mode, str(inp), str(out)], capture_output=True, text=True, timeout=1800, env={**os.environ, "ASAN_OPTIONS": "detect_leaks=0"})
    assert res.returncode == 0, res.stderr[-2000:]
    return out.read_bytes()


def _take(data, *shapes):
    """The arrays (dtype, shape) that stand one behind the other in `data`."""
    out, at = [], 0
    for dtype, shape in shapes:
        n = int(np.prod(shape))
        raw = np.frombuffer(data, dtype=np.int16 if dtype is BF else dtype, count=n, offset=at).copy()
        at += raw.nbytes
        t = torch.from_numpy(raw).reshape(shape)
        out.append(t.view(BF) if dtype is BF else t)
    return out


def i32(v):
    return np.asarray(v, dtype=np.int32)


@needs_gxx
@pytest.mark.parametrize("name", sorted(PLACES))
@pytest.mark.parametrize("blocks", [1, 3])
def test_place_source(tmp_path, name, blocks):
    ctx, new, table, free, used, rows, S, total = place_case(name)
    B, width = table.shape
    data = _run("place", [i32([B, width, len(free), rows, S, total, blocks]), i32(ctx), i32(new), table, i32(free), i32([used])], tmp_path)
    got = _take(data, (np.int64, (rows,)), (np.int32, (rows,)), (np.int32, (rows,)), (np.int32, (B + 1,)), (np.int32, (B,)), (np.int32, (1,)), (np.int32, (B, width)))
    want = plain.place(ctx, new, table.tolist(), free, used, rows, S, total)
    for a, b, what in zip(got, (*want[:5], [want[5]], want[6]), ("positions", "slots", "seqs", "cu", "lens", "used", "table")):
        assert a.tolist() == b, what


@needs_gxx
def test_place_source_bad_pages(tmp_path):
    """Pages outside the cache, in the tables and in the free list: no slot, and nothing else is touched."""
    ctx, new, S = [17, 3, 0], [3, 2, 5], 16
    table, free = i32([[0, 99], [-7, -1], [-1, -1]]), [2147483647, 5]
    data = _run("place", [i32([3, 2, 2, 12, S, 6, 1]), i32(ctx), i32(new), table, i32(free), i32([0])], tmp_path)
    got = _take(data, (np.int64, (12,)), (np.int32, (12,)))
    want = plain.place(ctx, new, table.tolist(), free, 0, 12, S, 6)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    assert want[1][:10] == [-1] * 10


@needs_gxx
@pytest.mark.parametrize("H,KV,hd,rot,axes,norm,shares", [(2, 1, 64, 64, 3, 0, 1), (6, 2, 128, 128, 3, 1, 4), (5, 1, 128, 64, 2, 1, 1), (4, 2, 64, 32, 4, 0, 4), (1, 1, 128, 16, 1, 1, 1), (20, 7, 128, 128, 3, 0, 2), (30, 5, 64, 64, 2, 1, 1)])
def test_rope_axes_source(tmp_path, H, KV, hd, rot, axes, norm, shares):
    g = gen(H, hd, rot, axes)
    M, top, pages, S, eps = 7, 40, 2, 16, 1e-6
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF)
    positions = torch.randint(0, top, (axes, M), generator=g)
    positions[axes - 1, 4], positions[0, 5] = top, -1   # outside the table
    positions[0, 6] = 1 << 40
    slots = torch.tensor([3, 31, -1, 0, 5, 6, 7], dtype=torch.int32)
    if M > 1:
        slots[1] = pages * S   # behind the cache
    axis_of = [i % axes for i in range(rot // 2)]
    qn, kn = (1 + 0.2 * torch.randn(2, hd, generator=g)).to(BF)
    table = angles(top, rot)
    data = _run("rope", [i32([M, H, KV, hd, rot, axes, top, pages * S, norm, shares]), np.float32([eps]), i32(axis_of), positions.numpy(), slots, table, qn, kn, qkv], tmp_path)
    q, kc, vc = _take(data, (BF, (M, H * hd)), (BF, (pages, S, KV, hd)), (BF, (pages, S, KV, hd)))
    zeros = torch.zeros(pages, S, KV, hd, dtype=BF)
    wq, wk, wv, slack_q, slack_k = plain.rope(qkv, positions, axis_of, slots, table, zeros, zeros, H, KV, hd, qn if norm else None, kn if norm else None, eps)
    within(q, wq, slack_q)
    within(kc, wk, slack_k)
    assert torch.equal(vc.double(), wv)


@needs_gxx
@pytest.mark.parametrize("KV,hd,S,span,new,lens", [(1, 64, 32, 16, 3, [1, 0, 40, 64]), (5, 128, 16, 16, 40, [33, 16]), (2, 64, 64, 32, 1, [64, 65, -3, 1000]), (20, 128, 16, 16, 1, [16])])
@pytest.mark.parametrize("split", [0, 1])
def test_span_bounds_source(tmp_path, KV, hd, S, span, new, lens, split):
    g = gen(KV, S, span, new)
    table, total = tables(g, [min(max(n, 0), 3 * S) for n in lens], S, width=3)
    table[0, 0] = total if len(lens) > 2 else table[0, 0]   # outside the cache
    keys = torch.randn(total, S, KV, hd, generator=g).to(BF)
    keys[:, 1::7] = float("nan")
    old = torch.full((total, S // span, KV, 2, hd), 5.0, dtype=BF)
    data = _run("bounds", [i32([len(lens), 3, total, S, span, KV, hd, new, split]), table, i32(lens), keys, old], tmp_path)
    got, = _take(data, (BF, tuple(old.shape)))
    want = plain.bounds(old, keys, table, lens, new)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))


@needs_gxx
def test_span_bounds_source_long_spans(tmp_path):
    """Spans so long that some of the grid's rounded-up warps are past 2^31 tokens: they are behind the end.  (No entry is a page: nothing is read.)"""
    long, width = 1 << 28, 7
    table, lens = torch.full((1, width), -1, dtype=torch.int32), [width * long]
    data = _run("bounds", [i32([1, width, 0, long, long, 1, 64, 1, 0]), table, i32(lens), torch.zeros(0, dtype=BF), torch.zeros(0, dtype=BF)], tmp_path)
    assert data == b""


# ---------------------------------------------------------------------------------------------------- refusals
def _place_args(**change):
    a = dict(context_lens=torch.zeros(2, dtype=torch.int32), new_lens=torch.ones(2, dtype=torch.int32), block_tables=torch.zeros(2, 4, dtype=torch.int32),
             free_blocks=torch.arange(8, dtype=torch.int32), free_used=torch.zeros(1, dtype=torch.int32), rows=4, block_size=16, num_blocks=8)
    return {**a, **change}


def _rope_args(**change):
    a = dict(qkv=torch.zeros(3, 4 * 64, dtype=BF), positions=torch.zeros(2, 3, dtype=torch.int64), axis_of=[0, 1] * 16, slot_mapping=torch.zeros(3, dtype=torch.int32),
             rope_table=torch.zeros(10, 64), k_cache=torch.zeros(2, 16, 1, 64, dtype=BF), v_cache=torch.zeros(2, 16, 1, 64, dtype=BF), heads=2, kv_heads=1, head_dim=64)
    return {**a, **change}


def _cache(**change):
    a = dict(q=torch.zeros(2, 4, 64, dtype=BF), k_cache=torch.zeros(4, 32, 2, 64, dtype=BF), v_cache=torch.zeros(4, 32, 2, 64, dtype=BF),
             bounds=torch.zeros(4, 2, 2, 2, 64, dtype=BF), block_tables=torch.zeros(2, 2, dtype=torch.int32), context_lens=torch.ones(2, dtype=torch.int32),
             spans=torch.zeros(2, 2, 3, dtype=torch.int32))
    return {**a, **change}


def _of(a, *names, **more):
    return {**{n: a[n] for n in names}, **more}


def test_refusals_of_types_and_shapes():
    from ssd_b200 import ops
    i64 = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(TypeError, match="new_lens"):
        ops.place_tokens(**_place_args(new_lens=i64))
    with pytest.raises(ValueError, match="new_lens"):
        ops.place_tokens(**_place_args(new_lens=torch.ones(3, dtype=torch.int32)))
    with pytest.raises(ValueError, match="block_tables"):
        ops.place_tokens(**_place_args(block_tables=torch.zeros(4, 2, dtype=torch.int32).t()))
    with pytest.raises(TypeError, match="positions"):
        ops.rope_axes_store_kv(**_rope_args(positions=torch.zeros(2, 3, dtype=torch.int32)))
    with pytest.raises(ValueError, match="axis_of"):
        ops.rope_axes_store_kv(**_rope_args(axis_of=[0] * 31))
    with pytest.raises(ValueError):
        ops.rope_axes_store_kv(**_rope_args(axis_of=[-1] * 32))
    with pytest.raises(TypeError):
        ops.rope_axes_store_kv(**_rope_args(axis_of=32))
    with pytest.raises(ValueError, match="axis_of"):
        ops.rope_axes_store_kv(**_rope_args(axis_of=np.zeros(4, dtype=np.int64)))   # (its bytes would be 32)
    with pytest.raises(ValueError, match="qkv"):
        ops.rope_axes_store_kv(**_rope_args(heads=3))
    with pytest.raises(ValueError, match="v_cache"):
        ops.rope_axes_store_kv(**_rope_args(v_cache=torch.zeros(3, 16, 1, 64, dtype=BF)))
    with pytest.raises(TypeError, match="k_norm_w"):
        ops.rope_axes_store_kv(**_rope_args(k_norm_w=torch.zeros(64)))
    a = _cache()
    names = ("bounds", "k_cache", "block_tables", "context_lens")
    with pytest.raises(ValueError, match="bounds"):
        ops.span_bounds(**_of(a, *names[1:], bounds=torch.zeros(4, 2, 2, 64, dtype=BF), new_tokens=1))
    with pytest.raises(ValueError, match="spans"):
        ops.span_bounds(**_of(a, *names[1:], bounds=torch.zeros(4, 3, 2, 2, 64, dtype=BF), new_tokens=1))
    with pytest.raises(ValueError, match="q"):
        ops.select_spans(torch.zeros(8, dtype=BF), **_of(a, "bounds", "block_tables", "context_lens", q_len=1, block_size=32, count=3))
    with pytest.raises(ValueError, match="q"):
        ops.select_spans(**_of(a, "q", "bounds", "block_tables", "context_lens", q_len=2, block_size=32, count=3))
    with pytest.raises(ValueError, match="spans"):
        ops.span_attention(**_of(_cache(spans=torch.zeros(2, 3, 3, dtype=torch.int32)), "q", "k_cache", "v_cache", "block_tables", "context_lens", "spans", span=16, q_len=1, scale=1.0))
    with pytest.raises(ValueError, match="contiguous"):
        ops.span_attention(**_of(_cache(q=torch.zeros(2, 64, 4, dtype=BF).transpose(1, 2)), "q", "k_cache", "v_cache", "block_tables", "context_lens", "spans", span=16, q_len=1, scale=1.0))


def test_no_cpu_path():
    from ssd_b200 import ops
    a = _cache()
    for call in (lambda: ops.place_tokens(**_place_args()), lambda: ops.rope_axes_store_kv(**_rope_args()),
                 lambda: ops.span_bounds(**_of(a, "bounds", "k_cache", "block_tables", "context_lens", new_tokens=1)),
                 lambda: ops.select_spans(**_of(a, "q", "bounds", "block_tables", "context_lens", q_len=1, block_size=32, count=3)),
                 lambda: ops.span_attention(**_of(a, "q", "k_cache", "v_cache", "block_tables", "context_lens", "spans", span=16, q_len=1, scale=1.0))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


P = 4096   # an address that no call below gets to use


def test_refusals_of_shared_arrays():
    """Outputs that lie over inputs which other blocks still read."""
    from ssd_b200 import lib
    so = lib.load()
    place = [P * i for i in range(1, 12)] + [2, 4, 8, 4, 16, 8, None]
    for at, over in ((9, 0), (9, 1), (10, 4)):
        for off in (0, 4) if at == 9 else (0,):
            args = list(place)
            args[at] = args[over] + off
            assert so.ssdk_place_tokens(*args) < 0 and "of their own" in so.ssdk_last_error().decode()
    row = 4 * 64 * 2
    rope = [16 * P, P, 2, bytes(32), P, P, 10, 64, None, None, 1e-6, 16 * P + 2 * row, 8 * P, 8 * P, 32, 3, 2, 1, 64, None]
    assert so.ssdk_rope_axes_store_kv(*rope) < 0 and "of its own" in so.ssdk_last_error().decode()


@pytest.mark.parametrize("name,good,bad", [
    # (index of an argument, value) that an entry point refuses before it touches the device
    ("ssdk_place_tokens", [P * i for i in range(1, 12)] + [2, 4, 8, 4, 16, 8, None],
     [(0, None), (3, None), (10, None), (11, 0), (11, 20000), (12, 0), (13, -1), (14, 0), (15, 0), (16, 0), (12, 1 << 28), (16, 1 << 28), (14, (1 << 30) + 1)]),
    ("ssdk_rope_axes_store_kv", [P, P, 2, bytes(32), P, P, 10, 64, None, None, 1e-6, 64 * P, P, P, 32, 3, 2, 1, 64, None],
     [(0, None), (1, None), (2, 0), (2, 5), (3, None), (3, bytes([2] * 32)), (6, 0), (7, 8), (7, 24), (7, 80), (0, P + 2), (8, P + 8), (14, 0), (15, 0), (16, 0), (17, 0), (18, 96)]),
    ("ssdk_span_bounds", [P, P, P, P, 2, 1, 2, 64, 32, 2, 4, 16, None],
     [(0, None), (3, None), (4, 0), (4, 70000), (5, 0), (6, 0), (7, 80), (8, 0), (9, 0), (10, 0), (11, 8), (11, 24), (11, 64), (0, P + 8)]),
    ("ssdk_span_attn", [P] * 7 + [2, 1, 4, 2, 64, 32, 2, 4, 16, 3, 0.1, None],
     [(0, None), (5, None), (7, 0), (8, 0), (9, 3), (9, 66), (10, 0), (11, 96), (12, 0), (13, 0), (14, 0), (15, 12), (16, 0), (16, 4097), (17, float("nan")), (17, float("inf")), (6, P + 2), (13, 1 << 27)]),
    ("ssdk_select_spans", [P] * 6 + [2, 1, 4, 2, 64, 32, 2, 4, 16, 3, 1, 1, None],
     [(0, None), (4, None), (5, None), (6, 0), (7, 0), (8, 3), (9, 0), (10, 96), (11, 0), (12, 0), (13, 0), (14, 20), (15, 0), (15, 4097), (16, -1), (17, -1), (17, 3), (1, P + 4), (12, 20000), (7, 3000)]),
])
def test_refusals_of_the_entry_points(name, good, bad):
    from ssd_b200 import lib
    so = lib.load()
    types = lib.SIGNATURES[name][1]
    assert len(good) == len(types)
    for at, value in bad:
        args = list(good)
        args[at] = value
        assert getattr(so, name)(*args) < 0, (name, at, value)
        text = so.ssdk_last_error().decode()
        assert name.replace("ssdk_", "").split("_store")[0] in text, text
