"""The 4-bit key/value cache against its description in 64 bits: store, read-back, decode and prompt attention, and chains of them, at
the edges of tiles, pages and lengths.

Tolerances count roundings, u = half of the type's eps each.  Attention is compared over the cache as it lies, so that
quantisation takes no part: queries, stored values where a kernel reads them in 16 bits, weights and the result are rounded once each, and
a score of a few units turns a rounding of its factors into an error of its weight of that size: 4 u in the 2-norm, as for the 16-bit caches."""
import pytest
import torch

from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu
DEV, D = "cuda", 128
TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def _no_status_left():
    from nanoquantization_b200 import _lib
    yield
    torch.cuda.synchronize()
    _lib.check_cache_status()


def _close(got, want, dtype, units=4):
    assert torch.isfinite(got).all()
    err = float((got.double() - want).norm() / want.norm())
    assert err <= units * ref.unit(dtype), err


def _cache(ends, kv_heads, block, dtype, seed=0, spare=2, width=0):
    """Pages in shuffled order with rows 0 .. ends[b] - 1 of every sequence; all other rows, and the pages of nobody, hold NaN.
    Returns (k, v, table, cache rows of every sequence)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // block) for n in ends]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    caches = [torch.full((len(order), kv_heads, block * ref.TOKEN), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]
    table = torch.full((len(ends), max(width, max(need, default=0), 1)), -1, dtype=torch.int32)
    rows = []
    for b, n in enumerate(ends):
        pages = [order.pop() for _ in range(need[b])]
        table[b, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        rows.append([pages[i // block] * block + i % block for i in range(n)])
        if n:
            for i, c in enumerate(caches):
                x = torch.randn(n, kv_heads, D, generator=g, device=DEV, dtype=torch.float64)
                x[..., 3] += 2 - 4 * i
                ref.set_rows(c, rows[-1], x, block, dtype)
    return (*caches, table.to(DEV), rows)


def _projections(T, heads, kv_heads, dtype, seed=1, pad=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    qkv = torch.randn(T, (heads + 2 * kv_heads) * D + pad, generator=g, device=DEV).to(dtype)
    qw, kw = ((torch.rand(D, generator=g, device=DEV) + 0.5).to(dtype) for _ in range(2))
    return qkv[:, :(heads + 2 * kv_heads) * D], qw, kw


def _rows(values):
    return torch.tensor(values, dtype=torch.int64, device=DEV)


# ------------------------------------------------------------------ store and read-back
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,heads,kv_heads,block,pad", [(1, 1, 1, 16, 0), (3, 2, 1, 16, 8), (37, 16, 8, 48, 0), (600, 12, 4, 256, 8), (5, 7, 7, 32, 4)], ids=str)
@torch.no_grad()
def test_store(T, heads, kv_heads, block, pad, dtype):
    from nanoquantization_b200.layers import kv4
    qkv, qw, kw = _projections(T, heads, kv_heads, dtype, pad=pad)
    pages = -(-T // block) + 1
    kc, vc = kv4.new_cache(pages, block, kv_heads, DEV)
    kc.fill_(7), vc.fill_(9)
    rows = torch.randperm(pages * block, generator=torch.Generator().manual_seed(T))[:T].to(DEV)
    if T > 2:
        rows[1] = -1
    positions = torch.arange(T, device=DEV) * 3 % 900
    cs = ref.angles(1000, DEV)
    before = qkv.clone()
    q = kv4.qknorm_rope_store(qkv, qw, kw, cs, positions, heads, kv_heads, 1e-6, kc, vc, rows)
    assert torch.equal(qkv, before)
    x = qkv.double().reshape(T, -1, D)
    want = ref.norm_rope(x[:, :heads], qw, cs, positions)
    # one rounding, and a few in float where a value comes from a difference
    assert ((q.double().view_as(want) - want).abs() <= ref.unit(dtype) * want.abs() + 1e-5).all()
    live = rows >= 0
    key, value = ref.norm_rope(x[:, heads:heads + kv_heads], kw, cs, positions)[live], x[:, heads + kv_heads:][live]
    for c, y, got in zip((kc, vc), (key, value), kv4.load(kc, vc, rows, dtype)):
        stored = ref.rows_of(c, rows[live].tolist(), block, dtype)
        # half a step, and what the parameters' roundings move the levels by
        s, lo = ref.params_of(y, dtype)
        edge = (0.5 * s + ref.unit(dtype) * (lo.abs() + 15 * s) + 1e-5).expand(*s.shape[:-1], 64).flatten(-2)
        assert ((stored - y).abs() <= edge).all()
        # parameters and levels are the definition's but where a float's rounding decides
        assert float(((stored - ref.quantised(y, dtype)).abs() > 1e-5).double().mean()) <= 5e-3
        assert ((got[live].double() - stored).abs() <= ref.unit(dtype) * stored.abs() + 1e-7).all()
        assert not got[~live].any()
    # nothing else is touched
    for c, byte in ((kc, 7), (vc, 9)):
        used = torch.zeros(pages * block, dtype=torch.bool, device=DEV)
        used[rows[live]] = True
        free = (~used).view(pages, 1, block, 1).expand(-1, kv_heads, -1, -1)
        assert (c[..., :block * 64].unflatten(-1, (block, 64)).masked_select(free) == byte).all()
        assert (c[..., block * 64:].unflatten(-1, (block, 8)).masked_select(free) == byte).all()


@pytest.mark.parametrize("dtype", TYPES)
@torch.no_grad()
def test_store_of_special_rows(dtype):
    """Constant rows are exact; rows with an infinity or a NaN read back as NaN in their group and nowhere else; ranges at the type's limits."""
    from nanoquantization_b200.layers import kv4
    top = torch.finfo(dtype).max
    v = torch.randn(9, D, device=DEV)
    v[0], v[1], v[2] = 0.0, -3.25, 0.0
    v[2, 64:] = 1.5
    v[3, 5], v[4, 70], v[5, 127] = float("inf"), float("nan"), -float("inf")
    v[6] = torch.tensor([-1.0, 1.0], device=DEV).repeat(64) * (top if dtype == torch.float16 else top / 4)
    v[7] *= 1e-5 if dtype == torch.float16 else 1e-30
    v[8, :64] = top
    qkv = torch.zeros(9, 3 * D, device=DEV)
    qkv[:, 2 * D:] = v
    qkv = qkv.to(dtype)
    kc, vc = kv4.new_cache(1, 16, 1, DEV)
    w, rows = torch.ones(D, device=DEV).to(dtype), torch.arange(9, device=DEV)
    kv4.qknorm_rope_store(qkv, w, w, ref.angles(16, DEV), rows, 1, 1, 1e-6, kc, vc, rows)
    got = kv4.load(kc, vc, rows, dtype)[1][:, 0]
    x = qkv[:, 2 * D:]
    for i in (0, 1, 2):
        assert torch.equal(got[i], x[i])
    for i, bad in ((3, 0), (4, 1), (5, 1)):
        assert got[i].unflatten(0, (2, 64)).isnan().all(-1).tolist() == [bad == 0, bad == 1]
        assert torch.isfinite(got[i].unflatten(0, (2, 64))[1 - bad]).all()
    y = x[6:].double()
    s, lo = ref.params_of(y, dtype)
    edge = (0.5 * s + ref.unit(dtype) * (3 * lo.abs() + 45 * s) + 15 * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).expand(3, 2, 64).flatten(-2)
    assert torch.isfinite(got[6:]).all() and ((got[6:].double() - y).abs() <= edge).all()


@pytest.mark.parametrize("dtype", TYPES)
@torch.no_grad()
def test_values_far_from_zero_with_a_small_range(dtype):
    """Ranges below the offset's rounding: the offset alone stands for them, in every way of reading."""
    from nanoquantization_b200.layers import kv4
    n, cs = 20, ref.angles(32, DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    qkv = torch.zeros(n, 3 * D, device=DEV)
    qkv[:, :D] = torch.randn(n, D, generator=g, device=DEV)
    qkv[:, D:2 * D] = 100 + torch.rand(n, D, generator=g, device=DEV) * 0.01      # after its norm, 1 and little around it
    qkv[:, 2 * D:] = 100 + torch.rand(n, D, generator=g, device=DEV) * 0.01
    qkv = qkv.to(dtype)
    w, rows, i32 = torch.ones(D, device=DEV).to(dtype), torch.arange(n, device=DEV), lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    w = (w + 0.001 * torch.arange(D, device=DEV) / D).to(dtype)
    kc, vc = kv4.new_cache(2, 16, 1, DEV)
    q = kv4.qknorm_rope_store(qkv, w, w, cs, torch.zeros(n, dtype=torch.int64, device=DEV), 1, 1, 1e-6, kc, vc, rows)
    k, v = (ref.rows_of(c, rows.tolist(), 16, dtype) for c in (kc, vc))
    assert (ref.rows_of(kc, rows.tolist(), 16, dtype) - ref.norm_rope(qkv.double()[:, None, D:2 * D], w, cs, torch.zeros(n, dtype=torch.int64, device=DEV))).abs().max() <= 2 * ref.unit(dtype)
    scales = torch.stack([c[..., 16 * 64:].unflatten(-1, (16, 8)).contiguous().view(dtype)[..., ::2].float() for c in (kc, vc)])
    assert (scales >= 0).all()
    table = i32(0, 1)[None]
    _close(kv4.prompt_attention(q, 1, kc, vc, table, i32(0, n), i32(0), [n], [0]), ref.attend(q.double().view(n, 1, D), k, v, 0).flatten(1), dtype)
    got = kv4.decode_attention(qkv[n - 1:], w, w, cs, torch.zeros(1, dtype=torch.int64, device=DEV), 1, 1, 1e-6, kc, vc, table, i32(n), rows[n - 1:])
    _close(got, ref.attend(q[n - 1:].double().view(1, 1, D), k, v, n - 1).flatten(1), dtype)


# ------------------------------------------------------------------ decode
# edges of tiles and pages, groups of heads below, at and above eight, long ones alone, many at once
DECODE = [((1,), 1, 1, 16), ((2, 16, 17, 64, 65), 2, 8, 16), ((5, 500, 1025), 2, 2, 256), ((129, 3, 31, 32, 33), 3, 48, 48), ((33,) * 70, 8, 32, 256),
          ((2048,), 8, 16, 256), ((4321,), 1, 4, 256), (tuple(1900 - 31 * i for i in range(16)), 8, 16, 256), (tuple(1500 - 8 * i for i in range(48)), 2, 10, 16),
          ((9000, 0, 1), 1, 17, 64), ((40000,), 1, 3, 256), ((100, 0, 16384, 5000), 2, 24, 32)]


def _decode_inputs(ctx, kv_heads, heads, block, dtype, seed=0, width=0):
    kc, vc, table, rows = _cache(ctx, kv_heads, block, dtype, seed, width=width)
    qkv, qw, kw = _projections(len(ctx), heads, kv_heads, dtype, seed + 1, pad=8)
    cs = ref.angles(max(ctx) + 1, DEV)
    at = _rows([r[-1] if r else -1 for r in rows])
    positions = _rows([max(n - 1, 0) for n in ctx])
    for c in (kc, vc):      # the token's own row is not there yet
        for r in at[at >= 0].tolist():
            c[..., :block * 64].unflatten(-1, (block, 64))[r // block, :, r % block] = 255
            c[..., block * 64:].unflatten(-1, (block, 8))[r // block, :, r % block] = 255
    return kc, vc, table, rows, qkv, qw, kw, cs, at, positions


def _decode_check(got, ctx, kv_heads, heads, block, dtype, kc, vc, rows, qkv, qw, kw, cs, positions):
    """Over the caches as the call left them; the token's own rows against a store of their own."""
    from nanoquantization_b200.layers import kv4
    live = [b for b, n in enumerate(ctx) if n]
    own = _rows([rows[b][-1] for b in live])
    k2, v2 = kv4.new_cache(len(live), 16, kv_heads, DEV)
    kv4.qknorm_rope_store(qkv[live].contiguous(), qw, kw, cs, positions[live], heads, kv_heads, 1e-6, k2, v2, torch.arange(len(live), device=DEV) * 16)
    for a, b in zip(kv4.load(kc, vc, own, dtype), kv4.load(k2, v2, torch.arange(len(live), device=DEV) * 16, dtype)):
        assert float((a != b).double().mean()) <= 2e-3 and float((a.double() - b.double()).norm() / b.double().norm()) <= 0.01
    x = qkv.double().reshape(len(ctx), -1, D)
    q = ref.norm_rope(x[:, :heads], qw, cs, positions)
    for b, n in enumerate(ctx):
        if n == 0:
            assert not got[b].any()
            continue
        k, v = (ref.rows_of(c, rows[b], block, dtype) for c in (kc, vc))
        _close(got[b], ref.attend(q[b:b + 1], k, v, n - 1).flatten(), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ctx,kv_heads,heads,block", DECODE, ids=str)
@torch.no_grad()
def test_decode(ctx, kv_heads, heads, block, dtype):
    from nanoquantization_b200.layers import kv4
    kc, vc, table, rows, qkv, qw, kw, cs, at, positions = _decode_inputs(ctx, kv_heads, heads, block, dtype, width=3)
    before = [c.clone() for c in (kc, vc)]
    got = kv4.decode_attention(qkv, qw, kw, cs, positions, heads, kv_heads, 1e-6, kc, vc, table, torch.tensor(ctx, dtype=torch.int32, device=DEV), at)
    _decode_check(got, ctx, kv_heads, heads, block, dtype, kc, vc, rows, qkv, qw, kw, cs, positions)
    for c, old in zip((kc, vc), before):     # the token's rows and nothing else
        changed = (c[..., :block * 64] != old[..., :block * 64]).unflatten(-1, (block, 64)).any(-1).any(1).flatten().nonzero().flatten()
        assert sorted(changed.tolist()) == sorted(at[at >= 0].tolist())


@pytest.mark.parametrize("dtype", TYPES)
@torch.no_grad()
def test_decode_of_extreme_values(dtype):
    """Scores far apart, values of very different and very small scales, a value that is not finite."""
    from nanoquantization_b200.layers import kv4
    ctx, kv_heads, heads, block = (700, 300), 2, 8, 32
    kc, vc, table, rows, qkv, qw, kw, cs, at, positions = _decode_inputs(ctx, kv_heads, heads, block, dtype)
    g = torch.Generator(device=DEV).manual_seed(5)
    for b, n in enumerate(ctx):
        size = (2.0 ** -(torch.arange(n, device=DEV) % 11) * (3e-4 if b else 200.0))[:, None, None]
        ref.set_rows(vc, rows[b][:-1], (torch.randn(n, kv_heads, D, generator=g, device=DEV, dtype=torch.float64) * size)[:-1], block, dtype)
        ref.set_rows(kc, rows[b][:-1], (20 * torch.randn(n, kv_heads, D, generator=g, device=DEV, dtype=torch.float64))[:-1], block, dtype)
    args = (qkv, qw, kw, cs, positions, heads, kv_heads, 1e-6, kc, vc, table, torch.tensor(ctx, dtype=torch.int32, device=DEV), at)
    got = kv4.decode_attention(*args, scale=2e-3)
    q = ref.norm_rope(qkv.double().reshape(2, -1, D)[:, :heads], qw, cs, positions)
    for b, n in enumerate(ctx):
        k, v = (ref.rows_of(c, rows[b], block, dtype) for c in (kc, vc))
        _close(got[b], ref.attend(q[b:b + 1], k, v, n - 1, 2e-3).flatten(), dtype)
    bad = rows[1][17]
    vc[..., block * 64:].unflatten(-1, (block, 8))[bad // block, 1, bad % block, 4:6] = 255       # the second group's scale of head 1
    got = kv4.decode_attention(*args, scale=2e-3).view(2, 2, 4, 2, 64).isnan()
    assert got[1, 1, :, 1].all() and int(got.sum()) == 4 * 64


# ------------------------------------------------------------------ prompts
# (lens, starts, kv_heads, heads, block): single tokens, tiles' edges, portions far into a sequence, sequences without tokens, groups that do not divide a tile
PROMPTS = [((1,), (0,), 1, 1, 16), ((2, 1, 5), (0, 7, 130), 2, 8, 16), ((128, 127, 129), (0, 0, 0), 1, 2, 256), ((64,), (0,), 8, 32, 256), ((33, 0, 31), (100, 5, 0), 2, 12, 48),
           ((300, 7), (0, 1000), 4, 16, 256), ((1000,), (513,), 1, 4, 32), ((5, 5, 5, 5), (3001, 2990, 64, 0), 8, 32, 256), ((17,), (9000,), 1, 8, 64),
           ((200, 1, 77), (0, 40, 3), 3, 9, 16), ((257,), (127,), 2, 14, 128), ((513, 100), (0, 255), 1, 1, 256), ((40,), (0,), 1, 64, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,starts,kv_heads,heads,block", PROMPTS, ids=str)
@torch.no_grad()
def test_prompt(lens, starts, kv_heads, heads, block, dtype):
    from nanoquantization_b200.layers import kv4
    ends = [n + s if n else 0 for n, s in zip(lens, starts)]
    kc, vc, table, rows = _cache(ends, kv_heads, block, dtype, seed=3, width=2)
    T = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(4)
    wide = torch.randn(T, heads * D + 16, generator=g, device=DEV).to(dtype)
    q = wide[:, 8:-8]
    cu = torch.tensor([0, *lens], device=DEV).cumsum(0).int()
    got = kv4.prompt_attention(q, heads, kc, vc, table, cu, torch.tensor(starts, dtype=torch.int32, device=DEV), lens, starts)
    assert got.shape == (T, heads * D)
    o = 0
    for b, n in enumerate(lens):
        if n:
            k, v = (ref.rows_of(c, rows[b], block, dtype) for c in (kc, vc))
            want = ref.attend(q[o:o + n].double().reshape(n, heads, D), k, v, starts[b])
            _close(got[o:o + n], want.flatten(1), dtype)
            for i in {0, n // 2, n - 1}:
                _close(got[o + i], want[i].flatten(), dtype)
        o += n


# what the tensor cores' tiles of 256 rows and 128 keys take: ragged prompts, groups that do not divide a tile, keys dealt to several CTAs, edges
MANY = [((300,) * 8, (0,) * 8, 8, 32, 256), ((257, 40, 700, 1), (0, 1500, 127, 9), 8, 64, 48), ((64,), (16000,), 2, 32, 256), ((1030,), (0,), 4, 12, 32), ((90, 500), (5000, 3), 4, 28, 64),
        ((520, 130), (0, 0), 8, 40, 16), ((256, 512), (0, 128), 16, 64, 128), ((1500,), (513,), 8, 8, 256)]


def _kernel(lens, starts, heads, kv_heads):
    from nanoquantization_b200 import _lib
    ends = [n + s for n, s in zip(lens, starts) if n]
    return _lib.load().nqb200_kv4_prompt_kernel_name(len(lens), sum(lens), max(lens), max(ends), sum(-(-e // 128) for e in ends), heads, kv_heads)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,starts,kv_heads,heads,block", MANY, ids=str)
@torch.no_grad()
def test_prompt_of_many_rows(lens, starts, kv_heads, heads, block, dtype):
    from nanoquantization_b200.layers import kv4
    assert _kernel(lens, starts, heads, kv_heads) == b"tiles_tcgen05"
    ends = [n + s for n, s in zip(lens, starts)]
    kc, vc, table, rows = _cache(ends, kv_heads, block, dtype, seed=5, width=2)
    T = sum(lens)
    q = torch.randn(T, heads * D, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV).to(dtype)
    cu = torch.tensor([0, *lens], device=DEV).cumsum(0).int()
    got = kv4.prompt_attention(q, heads, kc, vc, table, cu, torch.tensor(starts, dtype=torch.int32, device=DEV), lens, starts)
    again = kv4.prompt_attention(q, heads, kc, vc, table, cu, torch.tensor(starts, dtype=torch.int32, device=DEV), lens, starts)
    assert torch.equal(got, again)
    R, o = heads // kv_heads, 0
    for b, n in enumerate(lens):
        k, v = (ref.rows_of(c, rows[b], block, dtype) for c in (kc, vc))
        x = q[o:o + n].double().view(n, heads, D)
        seen = torch.arange(ends[b], device=DEV) <= starts[b] + torch.arange(n, device=DEV)[:, None]
        for h in {0, R - 1, heads // 2, heads - 1}:
            w = torch.softmax((x[:, h] @ k[:, h // R].T * D ** -0.5).masked_fill(~seen, float("-inf")), -1)
            want, mine = w @ v[:, h // R], got[o:o + n].view(n, heads, D)[:, h]
            _close(mine, want, dtype)
            worst = (mine.double() - want).norm(dim=-1) / want.norm(dim=-1)
            assert float(worst.max()) <= 4 * ref.unit(dtype), (b, h, int(worst.argmax()))
        o += n


@pytest.mark.parametrize("dtype", TYPES)
@torch.no_grad()
def test_prompt_of_many_rows_with_values_that_are_not_finite(dtype):
    """As below, for the tiles: also where the keys are dealt to several CTAs."""
    from nanoquantization_b200.layers import kv4
    for n, start, kv_heads, heads in ((700, 50, 8, 32), (64, 9000, 2, 32)):
        assert _kernel([n], [start], heads, kv_heads) == b"tiles_tcgen05"
        block, R = 64, heads // kv_heads
        kc, vc, table, rows = _cache([start + n], kv_heads, block, dtype, seed=8)
        q = torch.randn(n, heads * D, device=DEV).to(dtype)
        cu, pos0 = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.tensor([start], dtype=torch.int32, device=DEV)
        run = lambda: kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [n], [start])  # noqa: E731
        want, i = run(), n // 2
        r = rows[0][start + i]
        vc[..., block * 64:].unflatten(-1, (block, 8))[r // block, 1, r % block, 4:6] = 255             # the second group's scale of head 1
        got = run()
        nan = torch.zeros(n, kv_heads, R, 2, 64, dtype=torch.bool, device=DEV)
        nan[i:, 1, :, 1] = True
        nan = nan.view(n, -1)
        assert got[nan].isnan().all() and torch.equal(got[~nan], want[~nan])
        kc[..., block * 64:].unflatten(-1, (block, 8))[r // block, 0, r % block, 2:4] = 255             # the first group's offset of head 0
        got = run().view(n, kv_heads, -1)
        assert got[i:, 0].isnan().all() and torch.equal(got[:i], want.view(n, kv_heads, -1)[:i])


@torch.no_grad()
def test_prompts_that_are_taken_in_several_goes(monkeypatch):
    from nanoquantization_b200.layers import kv4
    lens, starts, kv_heads, heads, block, dtype = [200, 1, 0, 400, 90, 30, 700], [0, 900, 7, 100, 0, 0, 300], 4, 16, 32, torch.bfloat16
    kc, vc, table, rows = _cache([n + s if n else 0 for n, s in zip(lens, starts)], kv_heads, block, dtype, seed=4)
    q = torch.randn(sum(lens), heads * D, device=DEV).to(dtype)
    cu, pos0 = torch.tensor([0, *lens], device=DEV).cumsum(0).int(), torch.tensor(starts, dtype=torch.int32, device=DEV)
    want = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, lens, starts)
    for tiles in (1, 5, 9, 12):
        monkeypatch.setattr(kv4, "MOST_SCRATCH", tiles * 128 * 512 * kv_heads)
        _close(kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, lens, starts), want.double(), dtype)


@torch.no_grad()
def test_prompt_bad_pages_of_many_rows():
    from nanoquantization_b200 import _lib
    from nanoquantization_b200.layers import kv4
    lens, starts, kv_heads, heads, block, dtype = [300, 300], [0, 400], 8, 32, 32, torch.bfloat16
    assert _kernel(lens, starts, heads, kv_heads) == b"tiles_tcgen05"
    kc, vc, table, rows = _cache([300, 700], kv_heads, block, dtype, seed=2)
    q = torch.randn(600, heads * D, device=DEV).to(dtype)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    run = lambda t=table, cu=i32(0, 300, 600), pos0=i32(*starts): kv4.prompt_attention(q, heads, kc, vc, t, cu, pos0, lens, starts)  # noqa: E731
    good = run()
    _lib.check_cache_status()
    for at, page in ((3, -1), (0, len(kc)), (21, 1 << 30)):
        t = table.clone()
        t[1, at] = page
        got = run(t)
        assert torch.equal(got[:300], good[:300])
        with pytest.raises(RuntimeError, match="outside its buffer"):
            _lib.check_cache_status()
    # numbers on the device that are not those of the host: more keys, more tokens, tokens that are none of q's
    for kw in ({"pos0": i32(0, 30000)}, {"pos0": i32(0, -3)}, {"cu": i32(0, 300, 700)}, {"cu": i32(0, 300, 100)}, {"cu": i32(0, 300, 1 << 30)}):
        got = run(**kw)
        assert torch.equal(got[:300], good[:300])
        with pytest.raises(RuntimeError, match="outside its buffer"):
            _lib.check_cache_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 70, 400])
@torch.no_grad()
def test_prompt_with_values_that_are_not_finite(n, dtype):
    """A value that is no number reaches the tokens that see it, in its group of dimensions, and no other; a key that is none, their whole rows."""
    from nanoquantization_b200.layers import kv4
    kv_heads, heads, block, start = 2, 6, 32, 50
    kc, vc, table, rows = _cache([start + n], kv_heads, block, dtype, seed=8)
    q = torch.randn(n, heads * D, device=DEV).to(dtype)
    cu, pos0 = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.tensor([start], dtype=torch.int32, device=DEV)
    want = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [n], [start])
    i = n // 2
    r = rows[0][start + i]
    vc[..., block * 64:].unflatten(-1, (block, 8))[r // block, 1, r % block, 0:2] = 255             # the first group's scale of head 1
    got = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [n], [start])
    nan = torch.zeros(n, 2, heads // 2, 2, 64, dtype=torch.bool, device=DEV)
    nan[i:, 1, :, 0] = True
    nan = nan.view(n, -1)
    assert got[nan].isnan().all() and torch.equal(got[~nan], want[~nan])
    kc[..., block * 64:].unflatten(-1, (block, 8))[r // block, 0, r % block, 6:8] = 255             # the second group's offset of head 0
    got = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [n], [start]).view(n, 2, -1)
    assert got[i:, 0].isnan().all() and torch.equal(got[:i], want.view(n, 2, -1)[:i])


@pytest.mark.parametrize("dtype", TYPES)
@torch.no_grad()
def test_prompt_of_extreme_values(dtype):
    from nanoquantization_b200.layers import kv4
    n, kv_heads, heads, block = 333, 1, 4, 64
    kc, vc, table, rows = _cache([n], kv_heads, block, dtype, seed=9)
    g = torch.Generator(device=DEV).manual_seed(6)
    size = (2.0 ** -(torch.arange(n, device=DEV) % 11) * 200.0)[:, None, None]
    ref.set_rows(vc, rows[0], torch.randn(n, kv_heads, D, generator=g, device=DEV, dtype=torch.float64) * size, block, dtype)
    ref.set_rows(kc, rows[0], 20 * torch.randn(n, kv_heads, D, generator=g, device=DEV, dtype=torch.float64), block, dtype)
    q = torch.randn(n, heads * D, generator=g, device=DEV).to(dtype)
    cu, pos0 = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    got = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [n], [0], scale=2e-3)
    k, v = (ref.rows_of(c, rows[0], block, dtype) for c in (kc, vc))
    _close(got, ref.attend(q.double().view(n, heads, D), k, v, 0, 2e-3).flatten(1), dtype)
    # scores hundreds apart: a row's weight lies on one key, up to ties; finite, and inside the values' range
    got = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [n], [0], scale=10.0)
    assert torch.isfinite(got).all() and float(got.abs().max()) <= float(v.abs().max()) * (1 + 4 * ref.unit(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,start", [(5, 300), (400, 0), (90, 700)])
@torch.no_grad()
def test_prompt_of_values_far_from_one(n, start, dtype):
    """Tiles of very large and very small keys and values beside ordinary ones, and queries of any size: what a type holds, the result holds."""
    from nanoquantization_b200.layers import kv4
    kv_heads, heads, block, total = 2, 8, 32, n + start
    kc, vc, table, rows = _cache([total], kv_heads, block, dtype, seed=12)
    g = torch.Generator(device=DEV).manual_seed(7)
    big = 4e4 if dtype == torch.float16 else 1e20
    for c, sizes in ((kc, (1e-4, 1.0, big / 20)), (vc, (big / 20, 1e-5, 1.0))):
        for h in range(kv_heads):          # runs of 100 keys; the second head's are ten times as small
            size = torch.tensor(sizes, device=DEV, dtype=torch.float64)[torch.arange(total, device=DEV) // 100 % 3][:, None, None] * 10.0 ** -h
            x = torch.randn(total, kv_heads, D, generator=g, device=DEV, dtype=torch.float64) * size
            both = ref.rows_of(c, rows[0], block, dtype)
            both[:, h] = x[:, h]
            ref.set_rows(c, rows[0], both, block, dtype)
    k, v = (ref.rows_of(c, rows[0], block, dtype) for c in (kc, vc))
    q = torch.randn(n, heads * D, generator=g, device=DEV)
    q[:, ::2] *= 1e-3
    q = (q * (1e-3 if dtype == torch.float16 else 1e-9)).to(dtype)
    scale = 0.5 / float((q.double().view(n, kv_heads, -1, D).norm(dim=-1).amax()) * k.norm(dim=-1).amax())       # scores of one at most
    cu, pos0 = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.tensor([start], dtype=torch.int32, device=DEV)
    got = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [n], [start], scale=scale * 8)
    want = ref.attend(q.double().view(n, heads, D), k, v, start, scale * 8).flatten(1)
    _close(got, want, dtype)
    small = kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [n], [start], scale=-scale)
    _close(small, ref.attend(q.double().view(n, heads, D), k, v, start, -scale).flatten(1), dtype)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", TYPES)
@torch.no_grad()
def test_a_sequence_through_all_of_them(dtype):
    """A prompt in portions, drafted tokens and single ones: every token's result is that of the whole sequence at once."""
    from nanoquantization_b200.layers import kv4
    heads, kv_heads, block, cuts = 8, 2, 32, (0, 150, 151, 156, 200, 201, 202)
    n = cuts[-1]
    qkv, qw, kw = _projections(n, heads, kv_heads, dtype)
    cs, order = ref.angles(n, DEV), torch.tensor([5, 1, 6, 0, 3, 2, 4], dtype=torch.int32, device=DEV)
    rows = (order[torch.arange(n, device=DEV) // block].long() * block + torch.arange(n, device=DEV) % block)
    table, positions = order[None].contiguous(), torch.arange(n, device=DEV)
    whole = kv4.new_cache(7, block, kv_heads, DEV)
    q = kv4.qknorm_rope_store(qkv, qw, kw, cs, positions, heads, kv_heads, 1e-6, *whole, rows)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    want = kv4.prompt_attention(q, heads, *whole, table, i32(0, n), i32(0), [n], [0])
    kc, vc = kv4.new_cache(7, block, kv_heads, DEV)
    for a, b in zip(cuts, cuts[1:]):
        if b - a == 1:
            got = kv4.decode_attention(qkv[a:b], qw, kw, cs, positions[a:b], heads, kv_heads, 1e-6, kc, vc, table, i32(b), rows[a:b])
        else:
            q = kv4.qknorm_rope_store(qkv[a:b], qw, kw, cs, positions[a:b], heads, kv_heads, 1e-6, kc, vc, rows[a:b])
            got = kv4.prompt_attention(q, heads, kc, vc, table, i32(0, b - a), i32(a), [b - a], [a])
        _close(got, want[a:b].double(), dtype, 8)      # two results, each within four units
    assert float((kc != whole[0]).double().mean()) <= 1e-3 and float((vc != whole[1]).double().mean()) <= 1e-3


@torch.no_grad()
def test_a_cache_of_more_than_four_gigabytes():
    from nanoquantization_b200.layers import kv4
    heads, kv_heads, block, pages, dtype = 8, 8, 256, 33000, torch.bfloat16
    kc, vc = kv4.new_cache(pages, block, kv_heads, DEV)
    assert kc.numel() > 1 << 32
    qkv, qw, kw = _projections(300, heads, kv_heads, dtype)
    cs, at = ref.angles(300, DEV), torch.arange(300, device=DEV)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=DEV)
    rows = table[0, at // block].long() * block + at % block
    q = kv4.qknorm_rope_store(qkv, qw, kw, cs, at, heads, kv_heads, 1e-6, kc, vc, rows)
    k, v = (ref.rows_of(c[pages - 2:], (rows - (pages - 2) * block).tolist(), block, dtype) for c in (kc, vc))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = kv4.prompt_attention(q, heads, kc, vc, table, i32(0, 300), i32(0), [300], [0])
    _close(got, ref.attend(q.double().view(300, heads, D), k, v, 0).flatten(1), dtype)
    got = kv4.decode_attention(qkv[299:], qw, kw, cs, at[299:], heads, kv_heads, 1e-6, kc, vc, table, i32(300), rows[299:])
    _close(got, ref.attend(q[299:].double().view(1, heads, D), k, v, 299).flatten(1), dtype, 8)
    for x, y in zip(kv4.load(kc, vc, rows, dtype), (k, v)):
        _close(x, y, dtype, 1)


# ------------------------------------------------------------------ bad indexes, streams, graphs
@torch.no_grad()
def test_bad_indexes_are_reported_and_not_followed():
    from nanoquantization_b200 import _lib
    from nanoquantization_b200.layers import kv4
    dtype, heads, kv_heads, block, ctx = torch.float16, 4, 2, 16, (40, 40)
    kc, vc, table, rows, qkv, qw, kw, cs, at, positions = _decode_inputs(ctx, kv_heads, heads, block, dtype)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    n32 = i32(*ctx)

    def reported():
        with pytest.raises(RuntimeError, match="outside its buffer"):
            _lib.check_cache_status()
        _lib.check_cache_status()      # cleared
    decode = lambda **kw_: kv4.decode_attention(kw_.get("qkv", qkv), qw, kw, cs, kw_.get("positions", positions), heads, kv_heads, 1e-6, kc, vc,  # noqa: E731
                                                kw_.get("table", table), kw_.get("ctx", n32), kw_.get("rows", at))
    good = decode()
    _lib.check_cache_status()
    for page in (len(kc), -1, -5, 1 << 30):
        t = table.clone()
        t[1, 0] = page
        assert torch.equal(decode(table=t)[0], good[0])
        reported()
    assert torch.equal(decode(ctx=i32(40, 10000))[0], good[0])
    reported()
    before = kc.clone()
    assert torch.equal(decode(rows=_rows([at[0], len(kc) * block]))[0], good[0])
    reported()
    decode(positions=_rows([positions[0], 1 << 40]))
    reported()
    decode()
    assert torch.equal(kc, before)
    q = torch.randn(10, heads * D, device=DEV).to(dtype)
    prompt = lambda t=table, cu=i32(0, 5, 10), pos0=i32(30, 30): kv4.prompt_attention(q, heads, kc, vc, t, cu, pos0, [5, 5], [30, 30])  # noqa: E731
    good = prompt()
    _lib.check_cache_status()
    t = table.clone()
    t[1, 1] = len(kc)
    assert torch.equal(prompt(t)[:5], good[:5])
    reported()
    assert torch.equal(prompt(pos0=i32(30, 500))[:5], good[:5])      # more keys than the table has
    reported()
    rows3 = _rows([0, -1, len(kc) * block])
    k, v = kv4.load(kc, vc, rows3, dtype)
    assert not k[1:].any() and not v[1:].any() and k[0].any()
    reported()
    before = kc.clone(), vc.clone()
    kv4.qknorm_rope_store(qkv, qw, kw, cs, _rows([0, -7]), heads, kv_heads, 1e-6, kc, vc, _rows([-1, 1 << 40]))
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    reported()


@torch.no_grad()
def test_streams_and_graphs():
    """Captured and replayed with new contents, two graphs at once on two streams, beside eager calls."""
    from nanoquantization_b200.layers import kv4
    dtype, heads, kv_heads, block = torch.bfloat16, 8, 1, 64
    sets = []
    for seed, ctx in ((1, (9000, 70)), (2, (12000, 50))):
        kc, vc, table, rows, qkv, qw, kw, cs, at, positions = _decode_inputs(ctx, kv_heads, heads, block, dtype, seed, width=200)
        n32 = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        q = torch.randn(90, heads * D, device=DEV).to(dtype)
        cu, pos0 = torch.tensor([0, 60, 90], dtype=torch.int32, device=DEV), torch.tensor([ctx[0] - 60, 0], dtype=torch.int32, device=DEV)
        run = lambda kc=kc, vc=vc, table=table, qkv=qkv, qw=qw, kw=kw, cs=cs, at=at, positions=positions, n32=n32, q=q, cu=cu, pos0=pos0, s=ctx[0] - 60: (  # noqa: E731
            kv4.decode_attention(qkv, qw, kw, cs, positions, heads, kv_heads, 1e-6, kc, vc, table, n32, at), kv4.prompt_attention(q, heads, kc, vc, table, cu, pos0, [60, 30], [s, 0]))
        sets.append((run, qkv, q, [x.clone() for x in run()]))
    torch.cuda.synchronize()
    graphs = []
    for run, *_ in sets:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            run()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = run()
        graphs.append((g, side, out))
    for turn in range(3):
        for g, side, _ in graphs:
            with torch.cuda.stream(side):
                g.replay()
        eager = [run() for run, *_ in sets]
        torch.cuda.synchronize()
        for (_, _, out), (_, _, _, want), mine in zip(graphs, sets, eager):
            for a, b, c in zip(out, want, mine):
                assert torch.equal(a, b) and torch.equal(c, b)
    for (run, qkv, q, _), (g, side, out) in zip(sets, graphs):
        qkv.neg_(), q.neg_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, run()):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ copies
@pytest.mark.parametrize("n_pools,rows,n_pairs,shape,dtype", [(1, 2, 1, (3,), torch.uint8), (3, 9, 4, (8, 16 * 72), torch.uint8), (70, 5, 2, (33,), torch.float32),
                                                               (2, 500, 230, (7, 3), torch.float16), (2, 4, 1, (256, 8, 128), torch.bfloat16), (1, 3, 1, (1 << 22, 5), torch.uint8)], ids=str)
@torch.no_grad()
def test_copies_of_pages(n_pools, rows, n_pairs, shape, dtype):
    from nanoquantization_b200.layers.pages import copy_pages
    pools = [(torch.randint(0, 256, (rows, *shape), dtype=torch.uint8, device=DEV) if dtype == torch.uint8 else torch.randn(rows, *shape, device=DEV).to(dtype)) for _ in range(n_pools)]
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(rows)).tolist()
    src, dst = [order[i % (rows - n_pairs)] for i in range(n_pairs)], order[rows - n_pairs:]
    want = [p.clone() for p in pools]
    for p in want:
        p[dst] = p[src]
    copy_pages(pools, src, dst)
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


@torch.no_grad()
def test_copies_of_pools_that_start_anywhere():
    """Pools that are parts of a tensor: any alignment, and nothing beside them is touched."""
    from nanoquantization_b200.layers.pages import copy_pages
    base = torch.randint(0, 256, (1000,), dtype=torch.uint8, device=DEV)
    for at, nbytes in ((1, 48), (4, 48), (16, 48), (3, 7), (8, 12)):
        mine = base.clone()
        pool = mine[at:at + 5 * nbytes].view(5, nbytes)
        copy_pages([pool], [0, 0], [3, 1])
        want = base.clone()
        want[at:at + 5 * nbytes].view(5, nbytes)[[3, 1]] = base[at:at + nbytes]
        assert torch.equal(mine, want)


@torch.no_grad()
def test_copies_of_pools_that_do_not_fit():
    from nanoquantization_b200.layers.pages import copy_pages
    a = torch.zeros(4, 6, device=DEV)
    for pools in ([a, torch.zeros(5, 6, device=DEV)], [a, a.T], [a, torch.zeros(4, 6)], [a, torch.zeros((), device=DEV)], [torch.zeros((), device=DEV)], [torch.zeros(0, 6, device=DEV)]):
        with pytest.raises((ValueError, RuntimeError), match="pools must be|CUDA tensors only"):
            copy_pages(pools, [0], [1])
    for src, dst in (([0], [4]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([1 << 33], [0])):
        with pytest.raises(ValueError, match="every target once"):
            copy_pages([a], src, dst)
    with pytest.raises(RuntimeError, match="bad shape"):
        copy_pages([torch.zeros(4, 0, device=DEV)], [0], [1])


# rings that wrap with remainders for every number of CTAs on an SM: 192, 256, 360, 512 and 640 units of key/value heads
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,keys,kv_heads,heads", [(24, 700, 8, 16), (32, 600, 8, 8), (45, 500, 8, 32), (64, 400, 8, 64), (80, 300, 8, 24)], ids=str)
@torch.no_grad()
def test_decode_of_many_sequences(B, keys, kv_heads, heads, dtype):
    from nanoquantization_b200.layers import kv4
    ctx, block = tuple(keys - 7 * i % (keys - 1) for i in range(B)), 64
    kc, vc, table, rows, qkv, qw, kw, cs, at, positions = _decode_inputs(ctx, kv_heads, heads, block, dtype)
    got = kv4.decode_attention(qkv, qw, kw, cs, positions, heads, kv_heads, 1e-6, kc, vc, table, torch.tensor(ctx, dtype=torch.int32, device=DEV), at)
    _decode_check(got, ctx, kv_heads, heads, block, dtype, kc, vc, rows, qkv, qw, kw, cs, positions)
