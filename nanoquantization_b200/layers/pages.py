"""Copies of pages of a cache in all its tensors at once, bound through the C ABI.  No counterpart in the reference (it has no cache)."""
from __future__ import annotations

from array import array
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
    first, m = pools[0], len(pools)
    dev, rows = first.get_device(), first.shape[0] if first.dim() else 0
    if dev < 0:
        raise RuntimeError(f"nanoquantization_b200 runs on CUDA tensors only (no CPU fallback); got a tensor on {first.device}")
    if not all([p.dim() for p in pools]):
        raise ValueError("a pool has no rows")
    for p in pools:        # (few Python operations: a cache has dozens of pools)
        if p.get_device() != dev or not p.is_contiguous() or not rows or p.shape[0] != rows:
            raise ValueError(f"pools must be contiguous tensors of {rows} rows on {first.device}, none empty; got {tuple(p.shape)} on {p.device}")
    if min(sources) < 0 or max(sources) >= rows or min(targets) < 0 or max(targets) >= rows or len(set(targets)) < n or not set(targets).isdisjoint(sources):
        raise ValueError(f"sources and targets must be rows of 0 .. {rows - 1}, every target once and none a source as well")
    with _lib.on_device(dev) as stream:
        at, nbytes = array("Q", [p.data_ptr() for p in pools]), array("q", [p.nbytes // rows for p in pools])
        src, dst = array("i", sources), array("i", targets)
        status = _lib.load().nqb200_copy_pages(at.buffer_info()[0], nbytes.buffer_info()[0], m, rows, src.buffer_info()[0], dst.buffer_info()[0], n, stream)
    _lib.check(status)
