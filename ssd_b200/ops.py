"""Tensor-level wrappers over the stand-alone ops of libssdk (same names/argument meaning as the
reference's layers so the parity tests read like tests of ssd.layers.*).

PyTorch is plumbing here: it owns the device memory and the stream; every op runs in the
hand-written sm_100a kernels behind the C-ABI.  All functions require CUDA tensors and raise if
the extension is missing — there is no eager fallback.
"""
from __future__ import annotations

import functools

import torch

from . import lib as _L


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _req(t: torch.Tensor, dtype, name: str):
    if not t.is_cuda:
        raise RuntimeError(f"{name}: CUDA tensor required (libssdk has no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")


def linear(x: torch.Tensor, weight: torch.Tensor, split_k: int = 0) -> torch.Tensor:
    """F.linear(x, weight) for M = x.shape[0] <= 64 tokens (layers/linear.py:98,196).

    x [M, K] bf16, weight [N, K] bf16 -> [M, N] bf16 (fp32 accumulate, one bf16 rounding)."""
    _req(x, torch.bfloat16, "x")
    _req(weight, torch.bfloat16, "weight")
    M, K = x.shape
    N = weight.shape[0]
    assert weight.shape[1] == K
    y = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
    nkb = K // 64
    if split_k == 1:
        parts = None
    else:
        if split_k == 0:  # same bound as auto_splits() in csrc/engine.cu
            tiles = (N + 127) // 128
            sms = torch.cuda.get_device_properties(x.device).multi_processor_count
            s_bound = max(1, min(max(1, nkb // 4), (2 * sms + tiles - 1) // tiles))
        else:
            s_bound = min(split_k, nkb)
        parts = torch.empty(s_bound * M * N, dtype=torch.float32, device=x.device)
    lib = _L.load()
    _L.check(lib.ssdk_gemm_small_m(_ptr(x), _ptr(weight), _ptr(y), _ptr(parts), M, N, K, N, split_k, _stream()),
             "ssdk_gemm_small_m")
    return y


def gate_up_silu(x: torch.Tensor, w_gate_up: torch.Tensor) -> torch.Tensor:
    """SiluAndMul(MergedColumnParallelLinear(x)) fused (models/llama3.py:130-133).
    w_gate_up [2*ffn, K] gate rows then up rows -> [M, ffn]."""
    _req(x, torch.bfloat16, "x")
    _req(w_gate_up, torch.bfloat16, "w_gate_up")
    M, K = x.shape
    ffn = w_gate_up.shape[0] // 2
    h = torch.empty(M, ffn, dtype=torch.bfloat16, device=x.device)
    lib = _L.load()
    _L.check(lib.ssdk_gemm_gate_up_silu(_ptr(x), _ptr(w_gate_up), _ptr(h), M, ffn, K, _stream()), "ssdk_gemm_gate_up_silu")
    return h


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None):
    """RMSDNorm.forward (layers/layernorm.py:90-98).  Returns y if residual is None else (y, new_residual)."""
    _req(x, torch.bfloat16, "x")
    _req(weight, torch.bfloat16, "weight")
    M, d = x.shape
    y = torch.empty_like(x)
    res_out = torch.empty_like(x) if residual is not None else None
    if residual is not None:
        _req(residual, torch.bfloat16, "residual")
    lib = _L.load()
    _L.check(lib.ssdk_rmsnorm(_ptr(x), _ptr(residual), _ptr(weight), float(eps), _ptr(y), _ptr(res_out), M, d, _stream()),
             "ssdk_rmsnorm")
    return y if residual is None else (y, res_out)


def rope_store_kv(qkv: torch.Tensor, positions: torch.Tensor, slot_mapping: torch.Tensor, rope_table: torch.Tensor,
                  k_cache: torch.Tensor, v_cache: torch.Tensor, heads: int, kv_heads: int, head_dim: int,
                  q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None,
                  norm_eps: float = 1e-6) -> torch.Tensor:
    """[q/k RMSHeadNorm +] RotaryEmbedding.forward + store_kvcache (qwen3.py:97-105, rotary_embedding.py:40-60,
    attention.py:35-41).  Returns q [M, H*hd]; k (rotated) and v are written into the caches."""
    _req(qkv, torch.bfloat16, "qkv")
    _req(positions, torch.int64, "positions")
    _req(slot_mapping, torch.int32, "slot_mapping")
    _req(rope_table, torch.float32, "rope_table")
    M = qkv.shape[0]
    q = torch.empty(M, heads * head_dim, dtype=torch.bfloat16, device=qkv.device)
    lib = _L.load()
    _L.check(lib.ssdk_rope_store_kv(_ptr(qkv), _ptr(positions), _ptr(slot_mapping), _ptr(rope_table), _ptr(q_norm_w),
                                    _ptr(k_norm_w), float(norm_eps), _ptr(q), _ptr(k_cache), _ptr(v_cache), M, heads,
                                    kv_heads, head_dim, _stream()), "ssdk_rope_store_kv")
    return q


def silu_and_mul(x: torch.Tensor) -> torch.Tensor:
    """SiluAndMul.forward (layers/activation.py:11-14)."""
    _req(x, torch.bfloat16, "x")
    M, two_ffn = x.shape
    out = torch.empty(M, two_ffn // 2, dtype=torch.bfloat16, device=x.device)
    lib = _L.load()
    _L.check(lib.ssdk_silu_mul(_ptr(x), _ptr(out), M, two_ffn // 2, _stream()), "ssdk_silu_mul")
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                    context_lens: torch.Tensor, q_len: int, scale: float) -> torch.Tensor:
    """flash_attn_with_kvcache(q, k_cache, v_cache, cache_seqlens=context_lens, page_table=block_tables,
    causal=True[, cu_seqlens_q]) as called at layers/attention.py:107-111,128-131.

    q [B*q_len, H, hd]; caches [num_blocks, block_size, KV, hd]; returns [B*q_len, H*hd]."""
    _req(q, torch.bfloat16, "q")
    _req(k_cache, torch.bfloat16, "k_cache")
    _req(v_cache, torch.bfloat16, "v_cache")
    _req(block_tables, torch.int32, "block_tables")
    _req(context_lens, torch.int32, "context_lens")
    Mq, H, hd = q.shape
    B = Mq // q_len
    num_blocks, block_size, KV, _ = k_cache.shape
    max_blocks = block_tables.shape[1]
    lib = _L.load()
    nbytes = lib.ssdk_paged_attn_scratch_bytes(B, q_len, H, hd, max_blocks * block_size)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    out = torch.empty(Mq, H * hd, dtype=torch.bfloat16, device=q.device)
    _L.check(lib.ssdk_paged_attn_pages(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables), _ptr(context_lens), _ptr(out),
                                       _ptr(scratch), B, q_len, H, KV, hd, block_size, max_blocks, num_blocks, float(scale), _stream()),
             "ssdk_paged_attn_pages")
    return out


def sample(logits: torch.Tensor, temperatures: torch.Tensor, seed: int = 0, step_id: int = 0) -> torch.Tensor:
    """Sampler.forward (layers/sampler.py:14-36) — logits [B, V] bf16, temperatures [B] fp32 -> int64 [B]."""
    _req(logits, torch.bfloat16, "logits")
    _req(temperatures, torch.float32, "temperatures")
    B, V = logits.shape
    out = torch.empty(B, dtype=torch.int64, device=logits.device)
    lib = _L.load()
    _L.check(lib.ssdk_sample(_ptr(logits), V, _ptr(temperatures), B, V, seed, step_id, _ptr(out), _stream()), "ssdk_sample")
    return out


def verify(logits_p: torch.Tensor, logits_q: torch.Tensor, speculations: torch.Tensor, temperatures_target: torch.Tensor,
           temperatures_draft: torch.Tensor, cache_hits: torch.Tensor | None = None, jit_speculate: bool = False,
           seed: int = 0, step_id: int = 0):
    """ssd.utils.verify.verify (utils/verify.py:5-181), device-resident results:
    returns (n_accept int32 [B], recovery int64 [B]); the accepted suffix of row b is
    speculations[b, :1 + n_accept[b]]."""
    _req(logits_p, torch.bfloat16, "logits_p")
    _req(logits_q, torch.bfloat16, "logits_q")
    _req(speculations, torch.int64, "speculations")
    _req(temperatures_target, torch.float32, "temperatures_target")
    _req(temperatures_draft, torch.float32, "temperatures_draft")
    B, Kp1, V = logits_p.shape
    K = Kp1 - 1
    hits = None
    if cache_hits is not None:
        hits = cache_hits.to(torch.int32).contiguous()
    lib = _L.load()
    scratch = torch.empty(lib.ssdk_verify_scratch_bytes(B, K), dtype=torch.uint8, device=logits_p.device)
    n_acc = torch.empty(B, dtype=torch.int32, device=logits_p.device)
    rec = torch.empty(B, dtype=torch.int64, device=logits_p.device)
    _L.check(lib.ssdk_verify(_ptr(logits_p), _ptr(logits_q), _ptr(speculations), _ptr(temperatures_target),
                             _ptr(temperatures_draft), _ptr(hits), int(jit_speculate), B, K, V, seed, step_id, _ptr(n_acc),
                             _ptr(rec), _ptr(scratch), _stream()), "ssdk_verify")
    return n_acc, rec


# ---- around a long paged cache: places of a step's tokens, positions with several axes, attention over selected spans ----
_BF, _I32, _I64, _F32 = torch.bfloat16, torch.int32, torch.int64, torch.float32
_TOP = 1 << 31   # numbers from here on, and below -_TOP, would be cut to 32 bits without a word
# private functions, since small calls are bound by the host; a PyTorch that lacks them (one without CUDA does) takes the public ones
_gpu_now = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", lambda gpu: torch.cuda.current_stream(gpu).cuda_stream)


def _check(name: str, *args) -> int:
    """(tensor, its name, dtype, shape) of every argument; returns the index of their GPU.  (Small calls are bound by the host: one test
    per argument, and the reason only where it fails.)"""
    gpu = args[0][0].get_device()
    for t, what, dtype, shape in args:
        if t.dtype is dtype and t.shape == shape and t.get_device() == gpu and t.is_contiguous():
            continue
        if t.dtype is not dtype:
            raise TypeError(f"{name}: {what}: expected {dtype}, got {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"{name}: {what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{name}: {what}: must be contiguous")
        raise ValueError(f"{name}: {what}: on {t.device}, {args[0][1]} on {args[0][0].device}")
    if gpu < 0:
        raise RuntimeError(f"{name}: CUDA tensors required (libssdk has no CPU path)")
    return gpu


def _past_32_bits(name: str, *values: int):
    raise ValueError(f"{name}: {max(values, key=abs)} passes 32 bits")


def _last(t: torch.Tensor, dims: int) -> int:
    """The last size of a tensor that is to have `dims` of them, else one that fits no tensor."""
    return t.shape[-1] if t.dim() == dims else -1


def _launch(name: str, gpu: int, *args):
    """One entry point of libssdk on the tensors' GPU and its current stream."""
    fn = getattr(_L._lib or _L.load(), name)
    if gpu == _gpu_now():
        rc = fn(*args, _stream_of(gpu))
    else:
        with torch.cuda.device(gpu):
            rc = fn(*args, _stream_of(gpu))
    if rc:
        _L.check(rc, name)


def place_tokens(context_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, free_blocks: torch.Tensor,
                 free_used: torch.Tensor, rows: int, block_size: int, num_blocks: int):
    """Pages, positions and slots of a step's tokens from the lengths of its requests, without the host (BlockManager and
    prepare_decode / prepare_prefill: engine/block_manager.py, engine/helpers/runner_helpers.py:50-121).

    context_lens, new_lens int32 [B]: tokens in the cache, and tokens to come; block_tables int32 [B, max_blocks], completed in
    place; free_blocks int32 [F]: pages to hand out, the first free_used (int32 [1]) of which are gone; rows: room for new tokens.
    Returns positions int64 [rows], slot_mapping int32 [rows], row_seqs int32 [rows] (rows behind the last token: 0, -1, -1),
    cu_rows int32 [B + 1], lens int32 [B] (context_lens + new_lens; sequences that found no pages or rows: context_lens) and the
    new free_used.  Sequences are served in order, each as a whole: see ssdk_place_tokens (include/ssdk.h)."""
    B, width, F = _last(context_lens, 1), _last(block_tables, 2), _last(free_blocks, 1)
    if not (-_TOP <= rows < _TOP and -_TOP <= block_size < _TOP):
        _past_32_bits("place_tokens", rows, block_size)
    gpu = _check("place_tokens", (context_lens, "context_lens", _I32, (B,)), (new_lens, "new_lens", _I32, (B,)),
                 (block_tables, "block_tables", _I32, (B, width)), (free_blocks, "free_blocks", _I32, (F,)), (free_used, "free_used", _I32, (1,)))
    if rows < 1:
        raise ValueError(f"place_tokens: {rows} rows")
    positions = context_lens.new_empty(rows, dtype=_I64)
    slots, seqs, cu, lens, used = torch.unsafe_split_with_sizes(context_lens.new_empty(2 * rows + 2 * B + 2), (rows, rows, B + 1, B, 1))
    _launch("ssdk_place_tokens", gpu, context_lens.data_ptr(), new_lens.data_ptr(), block_tables.data_ptr(), free_blocks.data_ptr(), free_used.data_ptr(),
            positions.data_ptr(), slots.data_ptr(), seqs.data_ptr(), cu.data_ptr(), lens.data_ptr(), used.data_ptr(), B, width, F, rows, block_size, num_blocks)
    return positions, slots, seqs, cu, lens, used


def rope_axes_store_kv(qkv: torch.Tensor, positions: torch.Tensor, axis_of, slot_mapping: torch.Tensor, rope_table: torch.Tensor,
                       k_cache: torch.Tensor, v_cache: torch.Tensor, heads: int, kv_heads: int, head_dim: int,
                       q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None, norm_eps: float = 1e-6) -> torch.Tensor:
    """rope_store_kv with positions on several axes (time, height and width of images and video).

    positions int64 [axes, M], 1 to 4 axes; axis_of: the axis that each frequency turns by (rot_dim / 2 whole numbers, e.g.
    [0] * 16 + [1] * 24 + [2] * 24); rope_table fp32 [max_pos, rot_dim] cos | sin: the first rot_dim channels of a head turn.
    Norms and rotation in fp32 with one rounding.  Returns q [M, heads * head_dim]; keys and values are in their slots.  A row with a position
    outside the table has NaN queries and stores nothing; slots are distinct, those outside the cache store nothing."""
    M, axes = qkv.shape[0], positions.shape[0]
    top, rot = rope_table.shape if rope_table.dim() == 2 else (-1, -1)
    num_blocks, block_size, _, _ = k_cache.shape if k_cache.dim() == 4 else (-1,) * 4
    cache = (num_blocks, block_size, kv_heads, head_dim)
    axis_of = bytes(axis_of if type(axis_of) in (list, tuple, bytes) else list(axis_of))
    if len(axis_of) * 2 != rot:
        raise ValueError(f"rope_axes_store_kv: axis_of has {len(axis_of)} frequencies, rope_table {rot / 2}")
    args = [(qkv, "qkv", _BF, (M, (heads + 2 * kv_heads) * head_dim)), (positions, "positions", _I64, (axes, M)), (slot_mapping, "slot_mapping", _I32, (M,)),
            (rope_table, "rope_table", _F32, (top, rot)), (k_cache, "k_cache", _BF, cache), (v_cache, "v_cache", _BF, cache)]
    for w, what in ((q_norm_w, "q_norm_w"), (k_norm_w, "k_norm_w")):
        if w is not None:
            args.append((w, what, _BF, (head_dim,)))
    gpu = _check("rope_axes_store_kv", *args)
    q = qkv.new_empty(M, heads * head_dim)
    _launch("ssdk_rope_axes_store_kv", gpu, qkv.data_ptr(), positions.data_ptr(), axes, axis_of, slot_mapping.data_ptr(), rope_table.data_ptr(),
            top, rot, _ptr(q_norm_w), _ptr(k_norm_w), norm_eps, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), num_blocks * block_size, M,
            heads, kv_heads, head_dim)
    return q


def span_bounds(bounds: torch.Tensor, k_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, new_tokens: int) -> torch.Tensor:
    """Smallest and largest value of every channel over the keys of a span, for the spans that hold one of the last new_tokens
    tokens of each sequence (at least the tokens stored since the last call; more costs time only).

    bounds [num_blocks, block_size / span, KV, 2, hd] bf16, in place: its second size says how many spans a page has; k_cache
    [num_blocks, block_size, KV, hd]; context_lens int32 [B] with the new tokens.  Sequences that share a page have the same number of its tokens in the context (shared prefixes
    of whole pages do).  Returns bounds."""
    n, block_size, KV, hd = k_cache.shape if k_cache.dim() == 4 else (-1,) * 4
    subs = bounds.shape[1] if bounds.dim() == 5 else -1
    B, width = _last(context_lens, 1), _last(block_tables, 2)
    if not -_TOP <= new_tokens < _TOP:
        if new_tokens < 0:
            _past_32_bits("span_bounds", new_tokens)
        new_tokens = _TOP - 1
    if subs == 0 or block_size % subs:
        raise ValueError(f"span_bounds: pages of {block_size} tokens in {subs} spans")
    gpu = _check("span_bounds", (bounds, "bounds", _BF, (n, subs, KV, 2, hd)), (k_cache, "k_cache", _BF, (n, block_size, KV, hd)),
                 (block_tables, "block_tables", _I32, (B, width)), (context_lens, "context_lens", _I32, (B,)))
    _launch("ssdk_span_bounds", gpu, k_cache.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), bounds.data_ptr(), B, new_tokens, KV, hd,
            block_size, width, n, block_size // subs)
    return bounds


@functools.lru_cache(maxsize=256)
def _select_scratch(*sizes: int) -> int:
    return _L.load().ssdk_select_spans_scratch_bytes(*sizes) // 2


def select_spans(q: torch.Tensor, bounds: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, q_len: int, block_size: int,
                 count: int, first: int = 1, last: int | None = None) -> torch.Tensor:
    """The `count` spans of each sequence's cache that its queries are to read, per key head: the first `first` and the last
    `last` ones (None: as many as q_len tokens can lie in, if count has room), then those that a query of the group can score highest with,
    max over its rows of sum_d max(q_d lo_d, q_d hi_d).

    q [B * q_len, H, hd] bf16 (rotated); bounds as span_bounds keeps them.  Returns int32 [B, KV, count], ascending, -1 behind the
    last: what span_attention takes.  The rows of a sequence share their spans."""
    n, subs, KV, _, hd = bounds.shape if bounds.dim() == 5 else (-1,) * 5
    B, width, H = _last(context_lens, 1), _last(block_tables, 2), q.shape[1] if q.dim() == 3 else -1
    if not (-_TOP <= block_size < _TOP and -_TOP <= count < _TOP and -_TOP <= first < _TOP and (last is None or -_TOP <= last < _TOP)):
        _past_32_bits("select_spans", block_size, count, first, last or 0)
    if subs == 0 or block_size % subs:
        raise ValueError(f"select_spans: pages of {block_size} tokens in {subs} spans")
    gpu = _check("select_spans", (q, "q", _BF, (B * q_len, H, hd)), (bounds, "bounds", _BF, (n, subs, KV, 2, hd)),
                 (block_tables, "block_tables", _I32, (B, width)), (context_lens, "context_lens", _I32, (B,)))
    span = block_size // subs
    if last is None:
        last = min((q_len + span - 2) // span + 1, count - first)
    out = context_lens.new_empty(B, KV, max(count, 0))
    scratch = q.new_empty(_select_scratch(B, KV, block_size, width, span))
    _launch("ssdk_select_spans", gpu, q.data_ptr(), bounds.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), out.data_ptr(),
            scratch.data_ptr(), B, q_len, H, KV, hd, block_size, width, n, span, count, first, last)
    return out


def span_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                   spans: torch.Tensor, span: int, q_len: int, scale: float) -> torch.Tensor:
    """paged_attention over the keys of the listed spans only: spans int32 [B, KV, count] (select_spans), `span` tokens each.

    q [B * q_len, H, hd]; returns [B * q_len, H * hd].  Entries outside the context are passed over, a span listed twice counts twice, a row
    that sees no key, or whose scores are all minus infinity, is zero (as in paged_attention)."""
    n, block_size, KV, hd = cache = k_cache.shape if k_cache.dim() == 4 else (-1,) * 4
    B, width, H, count = _last(context_lens, 1), _last(block_tables, 2), q.shape[1] if q.dim() == 3 else -1, _last(spans, 3)
    if not -_TOP <= span < _TOP:
        _past_32_bits("span_attention", span)
    gpu = _check("span_attention", (q, "q", _BF, (B * q_len, H, hd)), (k_cache, "k_cache", _BF, cache), (v_cache, "v_cache", _BF, cache),
                 (block_tables, "block_tables", _I32, (B, width)), (context_lens, "context_lens", _I32, (B,)), (spans, "spans", _I32, (B, KV, count)))
    out = q.new_empty(B * q_len, H * hd)
    _launch("ssdk_span_attn", gpu, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), spans.data_ptr(),
            out.data_ptr(), B, q_len, H, KV, hd, block_size, width, n, span, count, scale)
    return out


# ---- a paged cache whose keys and values are held in 4 bits ----
_U8 = torch.uint8


def kv4_caches(num_blocks: int, block_size: int, kv_heads: int, head_dim: int, device="cuda"):
    """(k_cache, v_cache) of zeros: uint8 [num_blocks, kv_heads, block_size * (head_dim / 2 + 4)], the codes of a page's tokens and behind them their scales and
    minima (include/ssdk.h has the format).  17 bytes where the bf16 cache has 64 (heads of 128); a page of one head is one piece, so pages are copied as they are."""
    if head_dim not in (64, 128) or not 16 <= block_size <= 65536 or block_size % 16 or num_blocks < 1 or num_blocks * block_size >= _TOP or not 1 <= kv_heads <= 65535:
        raise ValueError(f"kv4_caches: {num_blocks} pages of {block_size} tokens (a multiple of 16 up to 65536, fewer than 2^31 in all), {kv_heads} heads (at most 65535) of {head_dim} (64 or 128)")
    return tuple(torch.zeros(2, num_blocks, kv_heads, block_size * (head_dim // 2 + 4), dtype=_U8, device=device).unbind(0))


def _kv4(name: str, k_cache: torch.Tensor, head_dim: int):
    """Shape of the caches, and the tokens of a page."""
    row = 68 if head_dim == 128 else 36
    if k_cache.dim() == 3 and (head_dim == 128 or head_dim == 64):
        shape = k_cache.shape
        block_size, rest = divmod(shape[2], row)
        if not rest and 0 < block_size < _TOP:
            return shape, block_size
    if not (head_dim == 64 or head_dim == 128):
        raise ValueError(f"{name}: heads of {head_dim} (64 or 128)")
    raise ValueError(f"{name}: k_cache: {tuple(k_cache.shape)} is not [num_blocks, KV, block_size * {row}]")


def rope_store_kv4(qkv: torch.Tensor, positions: torch.Tensor, slot_mapping: torch.Tensor, rope_table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   heads: int, kv_heads: int, head_dim: int, q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None, norm_eps: float = 1e-6,
                   values: bool = False):
    """rope_store_kv into a cache of 4 bits (kv4_caches).

    qkv [M, (heads + 2 kv_heads) * head_dim] bf16; positions int64 [M]; slot_mapping int32 [M], distinct (outside the cache: stores nothing); rope_table fp32
    [max_pos, rot_dim] cos | sin: the first rot_dim channels of a head turn.  Returns q [M, heads * head_dim], and with `values` (q, k, v): k, v [M, kv_heads, head_dim] are
    what then stands in the cache, for attention among the new tokens.  A row with a position outside the table has NaN queries and stores nothing."""
    M = qkv.shape[0]
    top, rot = rope_table.shape if rope_table.dim() == 2 else (-1, -1)
    cache, block_size = _kv4("rope_store_kv4", k_cache, head_dim)
    cache = (cache[0], kv_heads, cache[2])
    args = [(qkv, "qkv", _BF, (M, (heads + 2 * kv_heads) * head_dim)), (positions, "positions", _I64, (M,)), (slot_mapping, "slot_mapping", _I32, (M,)),
            (rope_table, "rope_table", _F32, (top, rot)), (k_cache, "k_cache", _U8, cache), (v_cache, "v_cache", _U8, cache)]
    for w, what in ((q_norm_w, "q_norm_w"), (k_norm_w, "k_norm_w")):
        if w is not None:
            args.append((w, what, _BF, (head_dim,)))
    gpu = _check("rope_store_kv4", *args)
    q = qkv.new_empty(M, heads * head_dim)
    k, v = (qkv.new_empty(M, kv_heads, head_dim), qkv.new_empty(M, kv_heads, head_dim)) if values else (None, None)
    _launch("ssdk_rope_store_kv4", gpu, qkv.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(), rope_table.data_ptr(), top, rot, _ptr(q_norm_w), _ptr(k_norm_w),
            norm_eps, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _ptr(k), _ptr(v), cache[0], block_size, M, heads, kv_heads, head_dim)
    return (q, k, v) if values else q


def store_kv4(k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, values: bool = False):
    """Rows of keys and values as they are, into a cache of 4 bits (kv4_caches): a model without rotation, pages of an unquantised cache that is taken over.

    k, v [M, KV, head_dim] bf16; their rows may lie apart (views of a projection's output: heads and channels contiguous, rows at multiples of 8 elements); slot_mapping int32
    [M], distinct (outside the cache: stores nothing).  With `values` returns (k, v) as they then stand in the cache."""
    M, KV, hd = shape = k.shape if k.dim() == 3 else (-1,) * 3
    cache, block_size = _kv4("store_kv4", k_cache, hd)
    cache = (cache[0], KV, cache[2])
    plain = k.dtype is _BF and v.dtype is _BF and v.shape == shape and k.get_device() == v.get_device() == slot_mapping.get_device() and k.is_contiguous() and v.is_contiguous()
    if not plain:
        for t, what in ((k, "k"), (v, "v")):
            if t.dtype is not _BF:
                raise TypeError(f"store_kv4: {what}: expected {_BF}, got {t.dtype}")
            if t.shape != shape:
                raise ValueError(f"store_kv4: {what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
            if t.get_device() != slot_mapping.get_device():
                raise ValueError(f"store_kv4: {what}: on {t.device}, slot_mapping on {slot_mapping.device}")
            if t.stride(2) != 1 or (KV > 1 and t.stride(1) != hd):
                raise ValueError(f"store_kv4: {what}: heads and channels of a row must be contiguous")
    gpu = _check("store_kv4", (slot_mapping, "slot_mapping", _I32, (M,)), (k_cache, "k_cache", _U8, cache), (v_cache, "v_cache", _U8, cache))
    k_row, v_row = (KV * hd, KV * hd) if plain else (k.stride(0) if M > 1 else 0, v.stride(0) if M > 1 else 0)
    a, b = both = (k.new_empty(M, KV, hd), k.new_empty(M, KV, hd)) if values else (None, None)
    _launch("ssdk_store_kv4", gpu, k.data_ptr(), v.data_ptr(), k_row, v_row, slot_mapping.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _ptr(a), _ptr(b), cache[0], block_size, M, KV, hd)
    return both if values else None


def load_kv4(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, head_dim: int):
    """Rows of a cache of 4 bits read back: (k, v) bf16 [M, KV, head_dim] of the slots (int32 [M], any order; outside the cache: zeros)."""
    M = _last(slot_mapping, 1)
    cache, block_size = _kv4("load_kv4", k_cache, head_dim)
    gpu = _check("load_kv4", (k_cache, "k_cache", _U8, cache), (v_cache, "v_cache", _U8, cache), (slot_mapping, "slot_mapping", _I32, (M,)))
    k, v = both = k_cache.new_empty(M, cache[1], head_dim, dtype=_BF), k_cache.new_empty(M, cache[1], head_dim, dtype=_BF)
    _launch("ssdk_load_kv4", gpu, k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), k.data_ptr(), v.data_ptr(), cache[0], block_size, M, cache[1], head_dim)
    return both


@functools.lru_cache(maxsize=256)
def _kv4_scratch(*sizes: int) -> int:
    return _L.load().ssdk_paged_attn_kv4_scratch_bytes(*sizes) // 2


def paged_attention_kv4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, q_len: int,
                        scale: float) -> torch.Tensor:
    """paged_attention over a cache of 4 bits (kv4_caches): q [B * q_len, H, hd] bf16, block_tables int32 [B, max_blocks], context_lens int32 [B] with the new tokens.

    Returns [B * q_len, H * hd].  Keys and values are scale * code + minimum, not rounded up to sixteen rows (H / KV * q_len) to a key head, in bf16 as load_kv4 gives them with
    more.  At most 32 query heads to a key head.  Pages outside the cache are passed over, a row that sees no key is zero, a NaN row of the cache makes NaN of the rows that see it."""
    B, width, H, hd = _last(context_lens, 1), _last(block_tables, 2), *(q.shape[1:] if q.dim() == 3 else (-1, -1))
    cache, block_size = _kv4("paged_attention_kv4", k_cache, hd)
    gpu = _check("paged_attention_kv4", (q, "q", _BF, (B * q_len, H, hd)), (k_cache, "k_cache", _U8, cache), (v_cache, "v_cache", _U8, cache),
                 (block_tables, "block_tables", _I32, (B, width)), (context_lens, "context_lens", _I32, (B,)))
    out, scratch = q.new_empty(B * q_len, H * hd), _kv4_scratch(B, q_len, H, cache[1], hd, block_size, width)
    if scratch:
        scratch = (room := q.new_empty(scratch)).data_ptr()
    _launch("ssdk_paged_attn_kv4", gpu, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), out.data_ptr(), scratch or None, B, q_len, H, cache[1],
            hd, block_size, width, cache[0], scale)
    return out
