"""Which calls of the 4-bit cache's prompt attention are taken in several goes: those whose scratch is too large, and not those that need none."""
import pytest
import torch

from test_gpu_kv4 import DEV, D, _cache, _close, _kernel
from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,start,goes", [(3, 700, 1), (200, 700, 6)])
@torch.no_grad()
def test_goes(n, start, goes, monkeypatch):
    """Six sequences with room for the tiles of one and a half: drafts need no tiles, prompts are taken one at a time."""
    from nanoquantization_b200 import _lib
    from nanoquantization_b200.layers import kv4
    lens, starts, kv_heads, heads, block, dtype = [n] * 6, [start] * 6, 8, 32, 64, torch.bfloat16
    assert _kernel(lens, starts, heads, kv_heads) == (b"rows" if goes == 1 else b"tiles_tcgen05")
    kc, vc, table, rows = _cache([n + start] * 6, kv_heads, block, dtype, seed=4)
    q = torch.randn(6 * n, heads * D, device=DEV).to(dtype)
    cu, pos0 = torch.arange(0, 6 * n + 1, n, device=DEV).int(), torch.tensor(starts, dtype=torch.int32, device=DEV)
    calls, one = [], kv4._prompt
    monkeypatch.setattr(kv4, "_prompt", lambda *args: (calls.append(args), one(*args)))
    monkeypatch.setattr(kv4, "MOST_SCRATCH", -(-(n + start) // 128) * 3 // 2 * 128 * 512 * kv_heads)
    got = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, lens, starts)
    assert len(calls) == goes
    for b in range(6):
        k, v = (ref.rows_of(c, rows[b], block, dtype) for c in (kc, vc))
        at = slice(b * n, (b + 1) * n)
        _close(got[at], ref.attend(q[at].double().view(n, heads, D), k, v, start).flatten(1), dtype)
    _lib.check_cache_status()


@torch.no_grad()
def test_one_sequence_alone_may_take_more(monkeypatch):
    from nanoquantization_b200.layers import kv4
    n, start, kv_heads, heads, block, dtype = 300, 900, 8, 32, 64, torch.float16
    kc, vc, table, rows = _cache([n + start], kv_heads, block, dtype, seed=5)
    q = torch.randn(n, heads * D, device=DEV).to(dtype)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    want = kv4.prompt_attention(q, heads, kc, vc, table, i32(0, n), i32(start), [n], [start])
    monkeypatch.setattr(kv4, "MOST_SCRATCH", 1)
    assert torch.equal(kv4.prompt_attention(q, heads, kc, vc, table, i32(0, n), i32(start), [n], [start]), want)
