"""A scale of 0 under queries of any size: every key that a token sees has the same weight."""
import pytest
import torch

from test_gpu_kv4 import DEV, D, _cache, _close, _kernel
from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1.0, 1e-6, 1e-30, 0.0])
@pytest.mark.parametrize("n,heads,way", [(5, 4, b"rows"), (300, 32, b"tiles_tcgen05")])
@pytest.mark.parametrize("scale", [0.0, 1e-30])
@torch.no_grad()
def test_scores_of_nothing(scale, n, heads, way, size, dtype):
    from nanoquantization_b200.layers import kv4
    kv_heads, block = heads // 4, 32
    assert _kernel([n], [30], heads, kv_heads) == way
    kc, vc, table, rows = _cache([n + 30], kv_heads, block, dtype, seed=2)
    q = (torch.randn(n, heads * D, device=DEV) * size).to(dtype)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = kv4.prompt_attention(q, heads, kc, vc, table, i32(0, n), i32(30), [n], [30], scale=scale)
    v = ref.rows_of(vc, rows[0], block, dtype)
    want = v.cumsum(0)[30:] / torch.arange(31, n + 31, device=DEV)[:, None, None]
    _close(got, want.repeat_interleave(4, 1).flatten(1), dtype)
