"""Copies of a cache without keys and values: a model of recurrent layers alone has blocks, and nothing in them."""
import torch

from nanoquantization_b200.engine.batch import CacheLayout, KVSpec
from nanoquantization_b200.engine.engine import PagedKVCache


def test_a_cache_without_pools_has_nothing_to_copy():
    PagedKVCache(CacheLayout([None, None]), 4, 4, torch.float32, "cpu").copy([(0, 1), (2, 3)])
    cache = PagedKVCache(CacheLayout([None, KVSpec(1, 2, 3)]), 4, 4, torch.float32, "cpu")
    cache.k[1].copy_(torch.randn(cache.k[1].shape)), cache.v[1].copy_(torch.randn(cache.v[1].shape))
    k, v = cache.k[1].clone(), cache.v[1].clone()
    cache.copy([(0, 1), (2, 3)])
    assert torch.equal(cache.k[1], k[[0, 0, 2, 2]]) and torch.equal(cache.v[1], v[[0, 0, 2, 2]])
