"""A key/value cache of 4 bits for heads of 128: its store, its attention and its read-back, bound through the C ABI.

A cache is a pair of byte tensors ``[pages, kv_heads, block_size * 72]``, one for keys and one for values; a token and head take 72
bytes in each where 16-bit types take 256 (include/nqb200.h states the layout and how values are quantised: groups of 64, an offset and a scale
of the model's type each).  Activations are float16 or bfloat16, and a cache is read in the type that it was written in.  Cache row
r is row ``r % block_size`` of page ``r // block_size``, as for the 16-bit caches.

The reference has no cache; what the store and the decode step compute ahead of it is its QK-norm and rotary embedding
(nanoquantization/models/qwen3_quantized.py:88, layers/rope.py:24-45), here in 32 bits and rounded once.

A page, cache row or position outside its buffer is never followed: the kernels take zeros in its place and record it, and
``_lib.check_cache_status()`` (the engine calls it after every step) raises."""
from __future__ import annotations

from typing import Sequence

import torch

from .. import _lib

DIM, TOKEN = 128, 72
SPLIT_KEYS = 4096   # decode steps of tables for fewer keys need no scratch
TILE = 128          # keys of a tile of prompt_attention, which take 512 bytes each per key/value head while it runs
MOST_SEQUENCES, MOST_TILES = 65535, 1 << 24      # of a call of the library; more are taken in several goes
MOST_SCRATCH = 1 << 30      # where they go into tiles, more sequences than fit are taken in several goes (one alone may take more)


def new_cache(num_blocks: int, block_size: int, kv_heads: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values, zero-filled (every value reads back as 0)."""
    if block_size % 16:
        raise ValueError(f"a 4-bit cache takes blocks of a multiple of 16 tokens, got {block_size}")
    return tuple(torch.zeros(num_blocks, kv_heads, block_size * TOKEN, dtype=torch.uint8, device=device) for _ in range(2))


# Checks are written for few Python operations: a call of a few microseconds on the GPU is made as often as the host can make it.
def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> _lib.Kv4:
    if k_cache.dtype is not torch.uint8 or v_cache.dtype is not torch.uint8:
        raise TypeError("a 4-bit cache is a pair of byte tensors")
    shape = k_cache.shape
    if len(shape) != 3 or v_cache.shape != shape or shape[2] % (16 * TOKEN) or not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError(f"a 4-bit cache is two contiguous tensors [pages, kv_heads, block_size * {TOKEN}] with blocks of a multiple of 16 tokens, got "
                         f"{tuple(shape)} and {tuple(v_cache.shape)}")
    return _lib.Kv4(k_cache.data_ptr(), v_cache.data_ptr(), shape[0], shape[1], shape[2] // TOKEN)


def _ints(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")


def _on_one_gpu(device: int, tensors: tuple) -> None:
    for t in tensors:
        if t.get_device() != device or device < 0:
            _lib.require_cuda(*tensors)        # says what is wrong


def _projections(qkv, q_weight, k_weight, cos_sin, positions, num_q_heads, kv_heads, rows, cache):
    """Checks of what a step's tokens come with; the type's code."""
    dtype, shape = qkv.dtype, qkv.shape
    if cache.kv_heads != kv_heads or num_q_heads % kv_heads:
        raise ValueError(f"{num_q_heads} query heads over {kv_heads} do not go with a cache of {cache.kv_heads} key/value heads")
    if len(shape) != 2 or shape[1] != (num_q_heads + 2 * kv_heads) * DIM or qkv.stride(1) != 1:
        raise ValueError(f"qkv must be [tokens, {(num_q_heads + 2 * kv_heads) * DIM}] with unit stride along a row, got {tuple(shape)}")
    if q_weight.dtype is not dtype or k_weight.dtype is not dtype or q_weight.numel() != DIM or k_weight.numel() != DIM or not (q_weight.is_contiguous() and
                                                                                                                              k_weight.is_contiguous()):
        raise ValueError(f"q_weight and k_weight must be contiguous {dtype} tensors of {DIM}")
    if cos_sin.dtype is not torch.float32 or cos_sin.shape[-1] != DIM or not cos_sin.is_contiguous():
        raise ValueError(f"cos_sin must be a contiguous float32 tensor [..., {DIM}]")
    tokens = shape[:1]
    if positions.dtype is not torch.int64 or rows.dtype is not torch.int64 or positions.shape != tokens or rows.shape != tokens or not (positions.is_contiguous() and
                                                                                                                                      rows.is_contiguous()):
        raise ValueError(f"positions and rows must be contiguous int64 tensors of {shape[0]}")
    return _lib.dtype_code(dtype)


def qknorm_rope_store(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor, num_q_heads: int,
                      num_kv_heads: int, eps: float, k_cache: torch.Tensor, v_cache: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
    """Per-head RMSNorm and rotary embedding of q and k in ``qkv [T, (Hq + 2 Hkv) * 128]`` (left as it is); k and v of token t are stored in
    cache row ``rows[t]`` (below 0: nowhere).  Returns the queries ``[T, Hq * 128]``."""
    dev = qkv.get_device()
    _on_one_gpu(dev, (qkv, q_weight, k_weight, cos_sin, positions, k_cache, v_cache, rows))
    cache = _cache(k_cache, v_cache)
    code = _projections(qkv, q_weight, k_weight, cos_sin, positions, num_q_heads, num_kv_heads, rows, cache)
    with _lib.on_device(dev) as stream:
        T = qkv.shape[0]
        out = qkv.new_empty((T, num_q_heads * DIM))
        status = _lib.load().nqb200_kv4_store(qkv.data_ptr(), qkv.stride(0), q_weight.data_ptr(), k_weight.data_ptr(), cos_sin.data_ptr(), cos_sin.numel() // DIM,
                                              positions.data_ptr(), rows.data_ptr(), cache, out.data_ptr(), T, num_q_heads, eps, code,
                                              _lib.cache_status(dev), stream)
    _lib.check(status)
    return out


def load(k_cache: torch.Tensor, v_cache: torch.Tensor, rows: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of cache rows (int64; below 0: zeros) as ``[n, kv_heads, 128]`` of ``dtype``, the type they were written in."""
    dev = k_cache.get_device()
    _on_one_gpu(dev, (k_cache, v_cache, rows))
    cache, code, n = _cache(k_cache, v_cache), _lib.dtype_code(dtype), rows.numel()
    _ints("rows", rows, torch.int64, (n,))
    with _lib.on_device(dev) as stream:
        k, v = k_cache.new_empty((2, n, cache.kv_heads, DIM), dtype=dtype).unbind()
        status = _lib.load().nqb200_kv4_load(cache, rows.data_ptr(), k.data_ptr(), v.data_ptr(), n, code, _lib.cache_status(dev), stream)
    _lib.check(status)
    return k, v


def decode_attention(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor, num_q_heads: int,
                     num_kv_heads: int, eps: float, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, ctx: torch.Tensor, rows: torch.Tensor,
                     scale: float | None = None) -> torch.Tensor:
    """One token per sequence: what ``qknorm_rope_store`` does to it, then attention over the ``ctx[b]`` keys (int32) of sequence b, its
    own among them, whose pages are ``table[b]`` (int32).  ``ctx[b] = 0``: a row without a sequence, which gets zeros.  Returns ``[B, Hq * 128]``."""
    dev = qkv.get_device()
    _on_one_gpu(dev, (qkv, q_weight, k_weight, cos_sin, positions, k_cache, v_cache, table, ctx, rows))
    cache = _cache(k_cache, v_cache)
    code = _projections(qkv, q_weight, k_weight, cos_sin, positions, num_q_heads, num_kv_heads, rows, cache)
    B, width = qkv.shape[0], table.shape[-1]
    _ints("table", table, torch.int32, (B, width))
    _ints("ctx", ctx, torch.int32, (B,))
    lib = _lib.load()
    with _lib.on_device(dev) as stream:
        out = qkv.new_empty((B, num_q_heads * DIM))
        # (asked where the answer can be other than 0: a call of a few microseconds is made as often as the host can make it)
        need = lib.nqb200_kv4_decode_scratch_bytes(width, cache.block_size, B, num_q_heads, num_kv_heads) if width * cache.block_size >= SPLIT_KEYS else 0
        scratch = k_cache.new_empty(need) if need else None
        status = lib.nqb200_kv4_decode_attention(qkv.data_ptr(), qkv.stride(0), q_weight.data_ptr(), k_weight.data_ptr(), cos_sin.data_ptr(), cos_sin.numel() // DIM,
                                                 positions.data_ptr(), rows.data_ptr(), cache, table.data_ptr(), width, ctx.data_ptr(), out.data_ptr(), B,
                                                 num_q_heads, DIM ** -0.5 if scale is None else scale, eps, code, scratch.data_ptr() if need else None, need,
                                                 _lib.cache_status(dev), stream)
    _lib.check(status)
    return out


def prompt_attention(q: torch.Tensor, num_q_heads: int, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, cu: torch.Tensor,
                     pos0: torch.Tensor, lens: Sequence[int], starts: Sequence[int], scale: float | None = None) -> torch.Tensor:
    """Causal attention of several tokens per sequence over the cache, where their own keys and values have been stored already:
    ``q [T, Hq * 128]`` (normed and rotated) holds tokens ``cu[b] .. cu[b + 1] - 1`` of sequence b, at its positions ``pos0[b] ..`` (both int32);
    ``lens`` and ``starts`` are the same on the host.  Whole prompts, later portions and drafted tokens alike; returns ``[T, Hq * 128]``."""
    dev = q.get_device()
    _on_one_gpu(dev, (q, k_cache, v_cache, table, cu, pos0))
    cache, code = _cache(k_cache, v_cache), _lib.dtype_code(q.dtype)
    B, shape, width = len(lens), q.shape, table.shape[-1]
    if len(shape) != 2 or shape[1] != num_q_heads * DIM or q.stride(1) != 1 or num_q_heads % cache.kv_heads:
        raise ValueError(f"q must be [tokens, {num_q_heads * DIM}] with unit stride along a row, the heads a multiple of the cache's {cache.kv_heads}; got {tuple(shape)}")
    T = shape[0]
    if len(starts) != B or sum(lens) != T or min(lens, default=0) < 0 or min(starts, default=0) < 0:
        raise ValueError(f"lens and starts must name the {T} tokens of q, one number each per sequence and none negative")
    _ints("table", table, torch.int32, (B, width))
    _ints("cu", cu, torch.int32, (B + 1,))
    _ints("pos0", pos0, torch.int32, (B,))
    ends = [n + s for n, s in zip(lens, starts) if n]
    max_len, max_ctx, tiles = max(lens, default=0), max(ends, default=0), sum([(e + TILE - 1) // TILE for e in ends])
    out = q.new_empty((T, num_q_heads * DIM))
    scale = DIM ** -0.5 if scale is None else scale
    with _lib.on_device(dev) as stream:
        fits = B < 2 or (B <= MOST_SEQUENCES and tiles <= MOST_TILES)
        need = _lib.load().nqb200_kv4_prompt_scratch_bytes(B, T, max_len, max_ctx, tiles, num_q_heads, cache.kv_heads) if fits else 0
        if fits and (need <= MOST_SCRATCH or B < 2):
            _prompt(q, out, num_q_heads, cache, k_cache, code, table, cu, pos0, B, max_len, max_ctx, tiles, scale, need, stream)
            return out
        room = max(1, MOST_SCRATCH // (TILE * 512 * cache.kv_heads))
        b = o = 0
        while b < B:
            e, t, n = b, 0, 0
            while e < B and e - b < MOST_SEQUENCES and (t == 0 or t + (lens[e] + starts[e] + TILE - 1) // TILE <= room):
                t += (lens[e] + starts[e] + TILE - 1) // TILE if lens[e] else 0
                n += lens[e]
                e += 1
            if n:
                max_len, max_ctx = max(lens[b:e]), max(lens[i] + starts[i] for i in range(b, e) if lens[i])
                need = _lib.load().nqb200_kv4_prompt_scratch_bytes(e - b, n, max_len, max_ctx, t, num_q_heads, cache.kv_heads)
                _prompt(q[o:o + n], out[o:o + n], num_q_heads, cache, k_cache, code, table[b:e], cu[b:e + 1] - o, pos0[b:e], e - b, max_len, max_ctx, t, scale, need, stream)
            b, o = e, o + n
    return out


def _prompt(q, out, num_q_heads, cache, k_cache, code, table, cu, pos0, B, max_len, max_ctx, tiles, scale, need, stream):
    T, width = q.shape[0], table.shape[1]
    scratch = k_cache.new_empty(need) if need else None
    _lib.check(_lib.load().nqb200_kv4_prompt_attention(q.data_ptr(), q.stride(0), cache, table.data_ptr(), width, cu.data_ptr(), pos0.data_ptr(), out.data_ptr(), B, T, max_len,
                                               max_ctx, tiles, num_q_heads, scale, code, scratch.data_ptr() if need else None, need,
                                               _lib.cache_status(q.get_device()), stream))
