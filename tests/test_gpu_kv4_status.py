"""What the 4-bit cache's prompt attention says of numbers on the device that are not those of the host, in both of its ways."""
import pytest
import torch

from test_gpu_kv4 import DEV, D, _cache, _kernel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,heads,way", [(5, 4, b"rows"), (300, 32, b"tiles_tcgen05")])
@torch.no_grad()
def test_other_numbers_than_the_hosts_are_reported(n, heads, way):
    """More keys than the host says, within the table; fewer tokens than none.  The sequence ahead keeps its rows."""
    from nanoquantization_b200 import _lib
    from nanoquantization_b200.layers import kv4
    lens, starts, kv_heads, block, dtype = [n, n], [30, 30], 8 if heads == 32 else 2, 32, torch.bfloat16
    assert _kernel(lens, starts, heads, kv_heads) == way
    kc, vc, table, rows = _cache([n + 30, n + 30], kv_heads, block, dtype, seed=2, width=40)
    q = torch.randn(2 * n, heads * D, device=DEV).to(dtype)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.where(table < 0, 0, table)
    run = lambda cu=i32(0, n, 2 * n), pos0=i32(30, 30): kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, lens, starts)  # noqa: E731
    good = run()
    _lib.check_cache_status()
    for kw in ({"pos0": i32(30, 31)}, {"pos0": i32(30, 500)}, {"cu": i32(0, n, n - 1)}, {"cu": i32(0, n, 0)}, {"cu": i32(0, n, -1)}, {"cu": i32(0, n, 2 * n + 1)}):
        assert torch.equal(run(**kw)[:n], good[:n])
        with pytest.raises(RuntimeError, match="outside its buffer"):
            _lib.check_cache_status()
    # fewer than the host says are no fault
    assert torch.equal(run(cu=i32(0, n, n + 2))[:n], good[:n]) and torch.equal(run(pos0=i32(30, 29))[:n], good[:n])
    _lib.check_cache_status()
