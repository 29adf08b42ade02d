"""Copies of pages of a cache in all its tensors at once, bound through the C ABI.  No counterpart in the reference (it has no cache)."""
from __future__ import annotations

import ctypes
from typing import Sequence

import torch

from .. import _lib


def copy_pages(pools: Sequence[torch.Tensor], sources: Sequence[int], targets: Sequence[int]) -> None:
    """``pool[targets[i]] = pool[sources[i]]`` for every pool and i, in one launch (per 64 pools and 192 pairs).  Pools are contiguous tensors of any
    type with the same number of rows along their first dimension: keys and values of every layer, or recurrent states.  No target
    may come twice or be a source as well."""
    n = len(sources)
    if len(targets) != n:
        raise ValueError(f"{n} sources and {len(targets)} targets")
    if not pools or n == 0:
        return
    dev, rows, m = pools[0].device, pools[0].shape[0], len(pools)
    if dev.type != "cuda":
        raise RuntimeError(f"nanoquantization_b200 runs on CUDA tensors only (no CPU fallback); got a tensor on {dev}")
    for p in pools:
        if p.device != dev or p.shape[0] != rows or not p.is_contiguous():
            raise ValueError(f"pools must be contiguous tensors of {rows} rows on {dev}, got {tuple(p.shape)} on {p.device}")
    if not _in_range(sources, rows) or not _in_range(targets, rows) or len(set(targets)) < n or not set(targets).isdisjoint(sources):
        raise ValueError(f"sources and targets must be rows of 0 .. {rows - 1}, every target once and none a source as well")
    with _lib.on_device(dev) as on:
        _lib.check(_lib.load().nqb200_copy_pages((ctypes.c_void_p * m)(*[p.data_ptr() for p in pools]), (ctypes.c_int64 * m)(*[p.nbytes // rows for p in pools]), m,
                                                 rows, (ctypes.c_int32 * n)(*sources), (ctypes.c_int32 * n)(*targets), n, on.stream))


def _in_range(numbers: Sequence[int], rows: int) -> bool:
    return min(numbers) >= 0 and max(numbers) < rows
