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


@torch.no_grad()
def test_more_sequences_than_a_launch_takes():
    """70000 of one token, all over the same page, some of them empty: each sees the keys up to its position."""
    from nanoquantization_b200 import _lib
    from nanoquantization_b200.layers import kv4
    B, block, dtype = 70000, 16, torch.float16
    kc, vc, _, rows = _cache([block], 1, block, dtype, seed=6, spare=0)
    lens, starts = [int(b % 7 > 0) for b in range(B)], [b % 16 for b in range(B)]
    live = [b for b in range(B) if lens[b]]
    q = torch.zeros(len(live), D, device=DEV, dtype=dtype)
    cu = torch.tensor([0, *lens], device=DEV).cumsum(0).int()
    got = kv4.prompt_attention(q, 1, kc, vc, torch.zeros(B, 1, dtype=torch.int32, device=DEV), cu, torch.tensor(starts, dtype=torch.int32, device=DEV), lens, starts)
    v = ref.rows_of(vc, rows[0], block, dtype)[:, 0]
    means = v.cumsum(0) / torch.arange(1, 17, device=DEV)[:, None]
    _close(got, means[torch.tensor([starts[b] for b in live], device=DEV)], dtype)
    _lib.check_cache_status()


@pytest.mark.parametrize("sequences,tiles,goes", [(4, 1 << 24, 2), (65535, 13, 3), (65535, 18, 2), (65535, 1 << 24, 1)])
@torch.no_grad()
def test_limits_of_a_call(sequences, tiles, goes, monkeypatch):
    """Six sequences of six tiles, with smaller limits in the library's place."""
    from nanoquantization_b200.layers import kv4
    n, start, kv_heads, heads, block, dtype = 3, 700, 8, 32, 64, torch.bfloat16
    kc, vc, table, rows = _cache([n + start] * 6, kv_heads, block, dtype, seed=4)
    q = torch.randn(6 * n, heads * D, device=DEV).to(dtype)
    cu, pos0 = torch.arange(0, 6 * n + 1, n, device=DEV).int(), torch.full((6,), start, dtype=torch.int32, device=DEV)
    calls, one = [], kv4._prompt
    monkeypatch.setattr(kv4, "_prompt", lambda *args: (calls.append(args), one(*args)))
    monkeypatch.setattr(kv4, "MOST_SEQUENCES", sequences)
    monkeypatch.setattr(kv4, "MOST_TILES", tiles)
    monkeypatch.setattr(kv4, "MOST_SCRATCH", (tiles if tiles < 100 else 1 << 20) * 128 * 512 * kv_heads)
    got = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [n] * 6, [start] * 6)
    assert len(calls) == goes
    for b in range(6):
        k, v = (ref.rows_of(c, rows[b], block, dtype) for c in (kc, vc))
        at = slice(b * n, (b + 1) * n)
        _close(got[at], ref.attend(q[at].double().view(n, heads, D), k, v, start).flatten(1), dtype)
