"""Attention over the 4-bit cache where keys and values of one head are of very different sizes: what a token sees decides how exact its result is, and
not what stands beside it in a tile, behind it, or in the sequence with a weight of nearly nothing.

Every token and head by itself.  Values are random about zero and independent of the weights, so the roundings of values and weights (half a step
u each, independent from key to key) add up as the values themselves do and are 2 u of the result in the 2-norm; the result's own rounding is one u
more, and scores, of two units at most beside an offset that every type holds, move weights by another: 4 u.  float16 results below its smallest normal number are off
by half of its spacing there, 2^-25 an element, whatever computes them."""
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


def _each_close(got, want, dtype):
    """``[tokens, heads, 128]``."""
    assert torch.isfinite(got).all()
    err = (got.double() - want).norm(dim=-1)
    left = D ** 0.5 * 2.0 ** -25 if dtype == torch.float16 else 0.0
    allowed = 4 * ref.unit(dtype) * want.norm(dim=-1) + left
    worst = int((err / allowed).argmax())
    assert (err <= allowed).all(), (divmod(worst, want.shape[1]), float(err.flatten()[worst] / want.norm(dim=-1).flatten()[worst]))


def _sizes(what, total, dtype):
    """Largest magnitude of every position's values, and which keys nearly all of a token's weight lies on (where it sees one of them)."""
    j = torch.arange(total, device=DEV)
    all_, half = torch.ones(total, dtype=torch.bool, device=DEV), dtype == torch.float16
    big = torch.tensor(3e4 if half else 1e6, device=DEV, dtype=torch.float64)
    far = torch.tensor(6e4 if half else 1e20, device=DEV, dtype=torch.float64)
    one = torch.ones(total, device=DEV, dtype=torch.float64)
    return {"first tile above 1/64": lambda: (torch.where(j < 128, 0.017 * one, 0.0155), all_),
            "last tile above 1/64": lambda: (torch.where(j >= total - 100, 0.017 * one, 0.0155), all_),
            "all below 1/64": lambda: (0.0155 * one, all_),
            "steps of eight": lambda: (0.5 * 2.0 ** -(3 * (j // 128 % 5)) * one, all_),
            "weight on the small tiles": lambda: (torch.where(j // 128 % 2 == 0, one, 2.0 ** -11), j // 128 % 2 == 1),
            "large ones without weight": lambda: (torch.where(j % 128 == 77, big, 0.05), j % 128 != 77),
            "large ones at the end": lambda: (torch.where(j >= total - 3, far, 1.0), all_),
            "large ones at the start without weight": lambda: (torch.where(j < 2, far, 1.0), j >= 2),
            "a large tile in the middle": lambda: (torch.where((j >= 256) & (j < 384), far, 1.0), all_),
            "very small ones": lambda: (torch.where((j >= 256) & (j < 384), 1e-3 * one, 1e-4 if half else 1e-20), all_),
            "near the type's end": lambda: (torch.where(j % 200 < 100, (6.5e4 if half else 1e35) * one, 1.0), all_)}[what]()


VALUES = ["first tile above 1/64", "last tile above 1/64", "all below 1/64", "steps of eight", "weight on the small tiles", "large ones without weight", "large ones at the end",
          "large ones at the start without weight", "a large tile in the middle", "very small ones", "near the type's end"]


def _filled(total, kv_heads, block, dtype, sizes, heavy, key_size=None, seed=0):
    """Caches with one sequence: values of those sizes; keys random in their first half, 1 or 0 in the second, which the quantisation keeps."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = -(-total // block)
    order = torch.randperm(need + 1, generator=torch.Generator().manual_seed(seed))[:need]
    rows = (order[torch.arange(total) // block] * block + torch.arange(total) % block).tolist()
    caches = [torch.full((need + 1, kv_heads, block * ref.TOKEN), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]
    k = torch.randn(total, kv_heads, D, generator=g, device=DEV, dtype=torch.float64)
    if key_size is None:
        k[..., 64:] = heavy[:, None, None].double()
    else:
        k = (2 * torch.rand(total, kv_heads, D, generator=g, device=DEV, dtype=torch.float64) - 1) * key_size[:, None, None]
    v = (2 * torch.rand(total, kv_heads, D, generator=g, device=DEV, dtype=torch.float64) - 1) * sizes[:, None, None]
    ref.set_rows(caches[0], rows, k, block, dtype)
    ref.set_rows(caches[1], rows, v, block, dtype)
    return (*caches, order.int()[None].to(DEV), rows, g)


def _queries(n, heads, dtype, g, far):
    """Scores of the keys with a 1 in them are 64 * 2.25 / sqrt(128) = 12.7 above the others', or 51."""
    q = torch.randn(n, heads, D, generator=g, device=DEV)
    q[..., 64:] = 9.0 if far else 2.25
    return q.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", VALUES)
@pytest.mark.parametrize("n,start,kv_heads,heads,way", [(500, 500, 4, 16, b"tiles_tcgen05"), (64, 6000, 2, 32, b"tiles_tcgen05"), (900, 0, 8, 32, b"tiles_tcgen05"),
                                                        (5, 900, 2, 8, b"rows"), (40, 500, 1, 3, b"rows")])
@torch.no_grad()
def test_prompt_values(n, start, kv_heads, heads, way, what, dtype):
    from nanoquantization_b200 import _lib
    from nanoquantization_b200.layers import kv4
    total, block = n + start, 64
    assert _lib.load().nqb200_kv4_prompt_kernel_name(1, n, n, total, -(-total // 128), heads, kv_heads) == way
    sizes, heavy = _sizes(what, total, dtype)
    kc, vc, table, rows, g = _filled(total, kv_heads, block, dtype, sizes, heavy)
    q = _queries(n, heads, dtype, g, "start without" in what)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = kv4.prompt_attention(q.flatten(1), heads, kc, vc, table, i32(0, n), i32(start), [n], [start])
    k, v = (ref.rows_of(c, rows, block, dtype) for c in (kc, vc))
    _each_close(got.view(n, heads, D), ref.attend(q.double(), k, v, start), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", VALUES)
@pytest.mark.parametrize("total,kv_heads,heads", [(1000, 2, 8), (5000, 1, 8), (300, 8, 16)])
@torch.no_grad()
def test_decode_values(total, kv_heads, heads, what, dtype):
    from nanoquantization_b200.layers import kv4
    block = 64
    sizes, heavy = _sizes(what, total, dtype)
    kc, vc, table, rows, g = _filled(total, kv_heads, block, dtype, sizes, heavy)
    qkv = torch.randn(1, heads + 2 * kv_heads, D, generator=g, device=DEV)
    qkv[:, :heads, 64:] = 2.25
    qkv[:, heads:heads + kv_heads, 64:] = 1.0
    qkv[:, heads + kv_heads:] = qkv[:, heads + kv_heads:].clamp(-1, 1) * sizes[-1].float()
    qkv = qkv.flatten(1).to(dtype)
    w, first = torch.ones(D, device=DEV).to(dtype), torch.zeros(1, dtype=torch.int64, device=DEV)
    cs = ref.angles(2, DEV)                            # position 0 turns nothing
    scale = 0.6 if "start without" in what else 0.15   # of queries of 1.3 in the second half, 12.4 or 50 between the keys' scores
    got = kv4.decode_attention(qkv, w, w, cs, first, heads, kv_heads, 1e-6, kc, vc, table, torch.tensor([total], dtype=torch.int32, device=DEV),
                               torch.tensor(rows[-1:], device=DEV), scale=scale)
    k, v = (ref.rows_of(c, rows, block, dtype) for c in (kc, vc))
    q = ref.norm_rope(qkv.double().view(1, -1, D)[:, :heads], w, cs, first)
    _each_close(got.view(1, heads, D), ref.attend(q, k, v, total - 1, scale), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [0.0155, 1e-3, "first", "last"])
@pytest.mark.parametrize("n,start,kv_heads,heads", [(500, 500, 4, 16), (64, 6000, 2, 32)])
@torch.no_grad()
def test_prompt_keys(n, start, kv_heads, heads, size, dtype):
    """Small keys, all of a head's or of some of its tiles, under queries as large as make scores of a unit."""
    from nanoquantization_b200 import _lib
    from nanoquantization_b200.layers import kv4
    total, block = n + start, 64
    assert _lib.load().nqb200_kv4_prompt_kernel_name(1, n, n, total, -(-total // 128), heads, kv_heads) == b"tiles_tcgen05"
    j = torch.arange(total, device=DEV)
    key_size = {"first": torch.where(j < 128, 0.017, 0.0155), "last": torch.where(j >= total - 128, 0.017, 0.0155)}.get(size, torch.full((total,), 0.0155 if isinstance(size, str) else size, device=DEV)).double()
    kc, vc, table, rows, g = _filled(total, kv_heads, block, dtype, torch.ones(total, device=DEV, dtype=torch.float64), None, key_size)
    q = (torch.randn(n, heads, D, generator=g, device=DEV) * float(2 / key_size.max())).to(dtype)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = kv4.prompt_attention(q.flatten(1), heads, kc, vc, table, i32(0, n), i32(start), [n], [start])
    k, v = (ref.rows_of(c, rows, block, dtype) for c in (kc, vc))
    _each_close(got.view(n, heads, D), ref.attend(q.double(), k, v, start), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [-40.0, 40.0])
@pytest.mark.parametrize("n,start,kv_heads,heads", [(500, 500, 4, 16), (64, 6000, 2, 32), (5, 900, 2, 8)])
@torch.no_grad()
def test_scores_far_from_zero(n, start, kv_heads, heads, shift, dtype):
    """All scores 226 below or above zero, which moves no weight: 326 in log2 units, beyond float's own range as a power."""
    from nanoquantization_b200.layers import kv4
    total, block = n + start, 64
    sizes, heavy = _sizes("all below 1/64", total, dtype)
    kc, vc, table, rows, g = _filled(total, kv_heads, block, dtype, sizes, heavy)
    q = torch.randn(n, heads, D, generator=g, device=DEV)
    q[..., 64:] = shift
    q = q.to(dtype)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = kv4.prompt_attention(q.flatten(1), heads, kc, vc, table, i32(0, n), i32(start), [n], [start])
    k, v = (ref.rows_of(c, rows, block, dtype) for c in (kc, vc))
    _each_close(got.view(n, heads, D), ref.attend(q.double(), k, v, start), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@torch.no_grad()
def test_sequences_and_heads_of_different_sizes_in_one_call(dtype):
    """Ordinary ones beside such of very large and very small values and keys, one with a value that is no number: each as by itself."""
    from nanoquantization_b200 import _lib
    from nanoquantization_b200.layers import kv4
    lens, starts, kv_heads, heads, block = [300, 200, 260, 1], [40, 500, 0, 130], 2, 16, 64
    far, near = (6e4, 1e-5) if dtype == torch.float16 else (1e30, 1e-12)
    # of keys and values, by sequence and head
    sizes = [((1.0, 1.0), (1.0, far)), ((1.0, 0.01), (near, 1.0)), ((1e-4, 1.0), (1.0, 0.0155)), ((1.0, 1.0), (far, near))]
    assert _lib.load().nqb200_kv4_prompt_kernel_name(4, 761, 300, 700, 3 + 6 + 3 + 2, heads, kv_heads) == b"tiles_tcgen05"
    g = torch.Generator(device=DEV).manual_seed(3)
    need = [-(-(n + s) // block) for n, s in zip(lens, starts)]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(3))
    caches = [torch.full((sum(need), kv_heads, block * ref.TOKEN), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]
    table, rows, at = torch.full((4, max(need)), -1, dtype=torch.int32), [], 0
    for b, (n, s) in enumerate(zip(lens, starts)):
        pages = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = pages.int()
        rows.append((pages[torch.arange(n + s) // block] * block + torch.arange(n + s) % block).tolist())
        for c, by in zip(caches, sizes[b]):
            x = 2 * torch.rand(n + s, kv_heads, D, generator=g, device=DEV, dtype=torch.float64) - 1
            ref.set_rows(c, rows[b], x * torch.tensor(by, device=DEV, dtype=torch.float64)[:, None], block, dtype)
    bad = rows[1][600]
    caches[1][..., block * 64:].unflatten(-1, (block, 8))[bad // block, 0, bad % block, 0:2] = 255            # the first group's scale, of small values
    q = torch.randn(sum(lens), heads, D, generator=g, device=DEV).to(dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cu = [0, 300, 500, 760, 761]
    got = kv4.prompt_attention(q.flatten(1), heads, *caches, table.to(DEV), i32(cu), i32(starts), lens, starts).view(-1, heads, D)
    for b, s in enumerate(starts):
        k, v = (ref.rows_of(c, rows[b], block, dtype) for c in caches)
        v = v.nan_to_num(0.0)
        mine, want = got[cu[b]:cu[b + 1]].clone(), ref.attend(q[cu[b]:cu[b + 1]].double(), k, v, s)
        if b == 1:
            assert mine[100:, :8, :64].isnan().all() and int(mine.isnan().sum()) == 100 * 8 * 64
            mine[100:, :8, :64] = want[100:, :8, :64].to(dtype)
        _each_close(mine, want, dtype)
