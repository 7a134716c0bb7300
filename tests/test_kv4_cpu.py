"""The paged cache held in 4 bits without a GPU: the sources of kv4_store_kernel and kv4_load_kernel on host threads (AddressSanitizer watches the ends of the arrays) against
their definitions, rows that are hard to quantise and slots and positions outside among them, and the refusals of all entry points."""
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from tests import kv4_plain as plain
from tests.cache_ops_util import BF, angles, gen, within
from tests.test_kv4_gpu import NAN, awkward, same_bits

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "emu", "run_kv4.cpp")
BIN = os.path.join(ROOT, "tests", "emu", "_build", "run_kv4")
needs_gxx = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++ (C++20)")


def _run(mode, parts, tmp_path):
    deps = [SRC] + [os.path.join(ROOT, "tests", "emu", f) for f in ("cuda_emu.h", "pairs_emu.h")] + [os.path.join(ROOT, "ssd_b200", "csrc", f) for f in ("kv4.cuh", "paged.cuh", "common.cuh")]
    if not os.path.exists(BIN) or any(os.path.getmtime(BIN) < os.path.getmtime(d) for d in deps):
        os.makedirs(os.path.dirname(BIN), exist_ok=True)
        subprocess.run(["g++", "-std=c++20", "-O1", "-ffp-contract=off", "-fsanitize=address", "-pthread", "-Wno-unknown-pragmas", "-Wno-attributes", "-o", BIN, SRC], check=True)
    inp, out = tmp_path / "in", tmp_path / "out"
    with open(inp, "wb") as f:
        for a in parts:
            a = a.contiguous().view(torch.int16).numpy() if isinstance(a, torch.Tensor) and a.dtype == BF else np.ascontiguousarray(a)
            a.tofile(f)
    res = subprocess.run([BIN, mode, str(inp), str(out)], capture_output=True, text=True, timeout=1800, env={**os.environ, "ASAN_OPTIONS": "detect_leaks=0"})
    assert res.returncode == 0, res.stderr[-2000:]
    return out.read_bytes()


def _take(data, *shapes):
    out, at = [], 0
    for dtype, shape in shapes:
        n = int(np.prod(shape))
        raw = np.frombuffer(data, dtype=np.int16 if dtype is BF else np.uint8, count=n, offset=at).copy()
        at += raw.nbytes
        t = torch.from_numpy(raw).reshape(shape)
        out.append(t.view(BF) if dtype is BF else t)
    assert at == len(data)
    return out


def i32(v):
    return np.asarray(v, dtype=np.int32)


@needs_gxx
@pytest.mark.parametrize("M,KV,hd,S,values,warps", [(25, 3, 64, 16, 1, 8), (24, 1, 128, 16, 1, 3), (7, 5, 128, 16, 0, 100), (1, 8, 64, 32, 1, 4)])
def test_store_source(tmp_path, M, KV, hd, S, values, warps):
    g = gen(M, KV, hd)
    pages = M // S + 2
    x = torch.cat([awkward(g, M, KV, hd), awkward(g, M, KV, hd)], 1)
    slots = torch.randperm(pages * S, generator=g)[:M].to(torch.int32)
    if M > 6:
        slots[4], slots[5], slots[6] = -1, pages * S, 2147483647
    kc, vc = plain.empty(pages, S, KV, hd, 7), plain.empty(pages, S, KV, hd, 9)
    data = _run("store", [i32([M, 0, KV, hd, 0, 0, S, pages, 0, values, warps]), np.float32([0]), np.zeros(M, np.int64), slots, torch.zeros(2 * hd, dtype=BF), x, kc, vc], tmp_path)
    want = [plain.rounded(plain.put(c, hd, y, slots)) for c, y in ((kc, x[:, :KV]), (vc, x[:, KV:]))]
    got = _take(data, (torch.uint8, kc.shape), (torch.uint8, vc.shape), *[(BF, (M, KV, hd))] * (2 * values))
    for a, b in zip(got, (kc, vc, *want)):
        same_bits(a, b)
    data = _run("load", [i32([M, KV, hd, S, pages, 1 + M % 3]), kc, vc, slots], tmp_path)
    out = (slots < 0) | (slots >= pages * S)
    for a, b in zip(_take(data, *[(BF, (M, KV, hd))] * 2), want):
        same_bits(a, b.masked_fill(out[:, None, None], 0.0))


@needs_gxx
@pytest.mark.parametrize("H,KV,hd,rot,norm,values,warps", [(2, 1, 64, 64, 0, 1, 1), (6, 2, 128, 128, 1, 0, 4), (5, 1, 128, 64, 1, 1, 7), (4, 2, 64, 32, 0, 0, 100), (1, 1, 128, 16, 1, 1, 2), (20, 5, 64, 48, 1, 1, 3)])
def test_rope_store_source(tmp_path, H, KV, hd, rot, norm, values, warps):
    g = gen(H, hd, rot)
    M, top, pages, S, eps = 7, 40, 2, 16, 1e-6
    qkv = torch.randn(M, (H + 2 * KV) * hd, generator=g).to(BF)
    positions = torch.randint(0, top, (M,), generator=g)
    positions[4], positions[5], positions[6] = top, -1, 1 << 40   # outside the table
    bad = torch.tensor([False] * 4 + [True] * 3)
    slots = torch.tensor([3, pages * S, -1, 0, 5, 6, 7], dtype=torch.int32)
    qn, kn = (1 + 0.2 * torch.randn(2, hd, generator=g)).to(BF)
    table = angles(top, rot)
    kc, vc = plain.empty(pages, S, KV, hd, 7), plain.empty(pages, S, KV, hd, 9)
    data = _run("rope", [i32([M, H, KV, hd, rot, top, S, pages, norm, values, warps]), np.float32([eps]), positions.numpy(), slots, table, qn, kn, qkv, kc, vc], tmp_path)
    x, safe = qkv.view(M, -1, hd), positions.masked_fill(bad, 0)
    wq, size = plain.turned(x[:, :H], safe, table, qn if norm else None, eps)
    k = plain.rounded(plain.turned(x[:, H:H + KV], safe, table, kn if norm else None, eps)[0])
    want = [plain.rounded(plain.put(c, hd, y, slots.masked_fill(bad, -1))).masked_fill(bad[:, None, None], NAN) for c, y in ((kc, k), (vc, x[:, H + KV:]))]
    got = _take(data, (BF, (M, H, hd)), (torch.uint8, kc.shape), (torch.uint8, vc.shape), *[(BF, (M, KV, hd))] * (2 * values))
    within(got[0], wq.masked_fill(bad[:, None, None], NAN), wq.abs() * 2 ** -8 + size * 2 ** -19)
    for a, b in zip(got[1:], (kc, vc, *want)):
        same_bits(a, b)


def test_every_quotient():
    """The definition's code is the nearest of the values that can stand there, the upper one of two equally near: scales of all mantissas, values on and beside every border."""
    s = torch.arange(128, 256, dtype=torch.float64)[:, None, None] / 128
    at = (torch.arange(15, dtype=torch.float64) + 0.5)[None, :, None] * s
    x = at * (1 + torch.tensor([-2.0 ** -20, 0.0, 2.0 ** -20], dtype=torch.float64))
    codes = torch.floor(x / s + 0.5)
    assert torch.equal(codes, torch.arange(15.0, dtype=torch.float64)[None, :, None] + torch.tensor([0.0, 1.0, 1.0], dtype=torch.float64).expand(128, 15, 3))


# ---------------------------------------------------------------------------------------------------- refusals
def _args(**change):
    a = dict(qkv=torch.zeros(3, 4 * 64, dtype=BF), positions=torch.zeros(3, dtype=torch.int64), slot_mapping=torch.zeros(3, dtype=torch.int32), rope_table=torch.zeros(10, 64),
             k_cache=torch.zeros(2, 1, 16 * 36, dtype=torch.uint8), v_cache=torch.zeros(2, 1, 16 * 36, dtype=torch.uint8), heads=2, kv_heads=1, head_dim=64)
    return {**a, **change}


def _rows(**change):
    a = _args()
    return {**{n: a[n] for n in ("slot_mapping", "k_cache", "v_cache")}, "k": torch.zeros(3, 1, 64, dtype=BF), "v": torch.zeros(3, 1, 64, dtype=BF), **change}


def _attn(**change):
    a = _args()
    return {**{n: a[n] for n in ("k_cache", "v_cache")}, "q": torch.zeros(4, 2, 64, dtype=BF), "block_tables": torch.zeros(2, 3, dtype=torch.int32),
            "context_lens": torch.ones(2, dtype=torch.int32), "q_len": 2, "scale": 1.0, **change}


def test_refusals_of_types_and_shapes():
    from ssd_b200 import ops
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    for change, error, match in [({"positions": torch.zeros(3, dtype=torch.int32)}, TypeError, "positions"), ({"qkv": torch.zeros(3, 5 * 64, dtype=BF)}, ValueError, "qkv"),
                                 ({"k_cache": torch.zeros(2, 1, 16 * 36)}, TypeError, "k_cache"), ({"k_cache": u8(2, 1, 16 * 36 + 4)}, ValueError, "k_cache"),
                                 ({"v_cache": u8(3, 1, 16 * 36)}, ValueError, "v_cache"), ({"k_cache": u8(2, 2, 16 * 36)}, ValueError, "k_cache"), ({"k_cache": u8(2, 16 * 36)}, ValueError, "k_cache"),
                                 ({"head_dim": 96}, ValueError, "96"), ({"k_norm_w": torch.zeros(64)}, TypeError, "k_norm_w"), ({"slot_mapping": torch.zeros(4, dtype=torch.int32)}, ValueError, "slot_mapping"),
                                 ({"rope_table": torch.zeros(64)}, ValueError, "rope_table"), ({"k_cache": u8(2, 1, 36 * 32)[..., ::2]}, ValueError, "contiguous")]:
        with pytest.raises(error, match=match):
            ops.rope_store_kv4(**_args(**change))
    rows = torch.zeros(3, 2, 64, dtype=BF)
    for change, error, match in [({"k": torch.zeros(3, 64, dtype=BF)}, ValueError, "heads"), ({"v": torch.zeros(3, 1, 64)}, TypeError, "v"), ({"v": torch.zeros(4, 1, 64, dtype=BF)}, ValueError, "v"),
                                 ({"k": rows.transpose(0, 1), "v": rows.transpose(0, 1)}, ValueError, "contiguous"),
                                 ({"k": torch.zeros(3, 64, 2, dtype=BF)[:, :, :1].transpose(1, 2)}, ValueError, "contiguous")]:
        with pytest.raises(error, match=match):
            ops.store_kv4(**_rows(**change))
    with pytest.raises(ValueError, match="k_cache"):
        ops.load_kv4(u8(2, 1, 16 * 36), u8(2, 1, 16 * 36), torch.zeros(3, dtype=torch.int32), 128)
    with pytest.raises(TypeError, match="slot_mapping"):
        ops.load_kv4(u8(2, 1, 16 * 36), u8(2, 1, 16 * 36), torch.zeros(3, dtype=torch.int64), 64)
    for change, error, match in [({"q": torch.zeros(4, 2, 32, dtype=BF)}, ValueError, "32"), ({"q_len": 3}, ValueError, "q"), ({"context_lens": torch.ones(2, dtype=torch.int64)}, TypeError, "context_lens"),
                                 ({"block_tables": torch.zeros(3, 3, dtype=torch.int32)}, ValueError, "block_tables"), ({"q": torch.zeros(4, 128, dtype=BF)}, ValueError, "heads")]:
        with pytest.raises(error, match=match):
            ops.paged_attention_kv4(**_attn(**change))
    for bad in [(0, 16, 1, 64), (2, 8, 1, 64), (2, 24, 1, 64), (2, 16, 0, 64), (2, 16, 1, 96)]:
        with pytest.raises(ValueError, match="kv4_caches"):
            ops.kv4_caches(*bad, device="cpu")
    k, v = ops.kv4_caches(2, 16, 1, 64, device="cpu")
    assert k.shape == v.shape == (2, 1, 16 * 36) and k.dtype is torch.uint8


def test_no_cpu_path():
    from ssd_b200 import ops
    a = _args()
    for call in (lambda: ops.rope_store_kv4(**a), lambda: ops.store_kv4(**_rows()), lambda: ops.load_kv4(a["k_cache"], a["v_cache"], a["slot_mapping"], 64), lambda: ops.paged_attention_kv4(**_attn())):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


P = 1 << 20   # addresses that no call below gets to use
ROPE = [P * i for i in range(1, 5)] + [100, 64, None, None, 1e-6] + [P * i for i in range(5, 10)] + [2, 16, 3, 2, 1, 64, None]
STORE = [P, 2 * P, 64, 64] + [P * i for i in range(3, 8)] + [2, 16, 3, 1, 64, None]
LOAD = [P * i for i in range(1, 6)] + [2, 16, 3, 1, 64, None]
ATTN = [P * i for i in range(1, 7)] + [None, 2, 1, 2, 1, 64, 16, 3, 2, 1.0, None]


@pytest.mark.parametrize("name,good,bad", [
    ("ssdk_rope_store_kv4", ROPE, [(0, 0), (0, P + 2), (1, 0), (3, 0), (3, 4 * P + 4), (4, 0), (5, 8), (5, 24), (5, 80), (6, 2), (9, 0), (9, 7 * P), (10, 6 * P + 8), (11, 0), (12, 0), (12, 6 * P), (13, P),
                                   (14, 0), (14, 1 << 28), (15, 8), (15, 24), (15, 65552), (16, 0), (17, 0), (17, 65536), (18, 0), (18, 65536), (19, 96), (19, 256)]),
    ("ssdk_store_kv4", STORE, [(0, 0), (1, 2 * P + 2), (2, -64), (2, 4), (3, 1 << 31), (4, 0), (5, 5 * P), (6, 0), (6, 2 * P), (7, 0), (8, 0), (8, 6 * P), (9, 0), (9, 1 << 40), (10, 0), (11, 0), (11, -1), (12, 0), (13, 32)]),
    ("ssdk_load_kv4", LOAD, [(0, 0), (1, 8), (2, 0), (3, 0), (3, 5 * P), (4, 2 * P), (4, 5 * P + 4), (5, 0), (6, 20), (7, 0), (7, (1 << 30) + 1), (8, 0), (9, 96)]),
    ("ssdk_paged_attn_kv4", ATTN, [(0, 0), (0, P + 2), (1, 0), (2, 8), (3, 0), (4, 0), (5, 0), (5, P), (5, 3 * P), (6, 8), (7, 0), (7, 65536), (8, 0), (8, 1 << 30), (9, 0), (9, 33), (10, 0), (10, 3), (11, 80), (12, 8),
                                   (13, 0), (13, 1 << 27), (14, 0), (14, 1 << 27), (15, float("inf")), (15, float("nan")), (15, 3e38)]),
])
def test_refusals_of_the_entry_points(name, good, bad):
    from ssd_b200 import lib
    so = lib.load()
    for i, value in bad:
        args = list(good)
        args[i] = value
        assert getattr(so, name)(*args) != 0, (name, i, value)
        assert so.ssdk_last_error().decode().startswith(name.split("_", 1)[1].replace("ssdk_", "")), (name, i, value, so.ssdk_last_error())
