"""Copies of pages of a cache in all its tensors at once, bound through the C ABI.  No counterpart in the reference (it has no cache)."""
from __future__ import annotations

from array import array
from operator import attrgetter
from typing import Sequence

import torch

from .. import _lib

_T, _NBYTES = torch.Tensor, attrgetter("nbytes")


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
    # (few Python operations: a cache has dozens of pools)
    try:
        fits = rows and {p.shape[0] for p in pools} == {rows} and set(map(_T.get_device, pools)) == {dev} and all(map(_T.is_contiguous, pools))
    except IndexError:     # a tensor without dimensions
        fits = False
    if not fits:
        raise ValueError(f"pools must be contiguous tensors of {rows} rows on {first.device}, none empty; got {[(tuple(p.shape), str(p.device)) for p in pools]}")
    if min(sources) < 0 or max(sources) >= rows or min(targets) < 0 or max(targets) >= rows or len(set(targets)) < n or not set(targets).isdisjoint(sources):
        raise ValueError(f"sources and targets must be rows of 0 .. {rows - 1}, every target once and none a source as well")
    with _lib.on_device(dev) as stream:
        at, nbytes = array("Q", map(_T.data_ptr, pools)), array("q", [n // rows for n in map(_NBYTES, pools)])
        src, dst = array("i", sources), array("i", targets)
        status = _lib.load().nqb200_copy_pages(at.buffer_info()[0], nbytes.buffer_info()[0], m, rows, src.buffer_info()[0], dst.buffer_info()[0], n, stream)
    _lib.check(status)
