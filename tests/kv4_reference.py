"""The 4-bit key/value cache from its description, in 64 bits: quantisation, layout, norm and rotation, attention."""
import torch

D, TOKEN = 128, 72


def unit(dtype):
    """The largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def params_of(x, dtype):
    """Scale and offset of the groups of ``x [..., 128]`` (double), each ``[..., 2, 1]``."""
    g = x.unflatten(-1, (2, 64))
    lo = g.amin(-1, keepdim=True).to(dtype).double()
    return ((g.amax(-1, keepdim=True) - lo) / 15).to(dtype).double(), lo


def quantised(x, dtype):
    """The values that rows ``x [..., 128]`` (double, finite) are stored as."""
    s, lo = params_of(x, dtype)
    n = torch.where(s > 0, (x.unflatten(-1, (2, 64)) - lo) / s.clamp(min=1e-300), 0).round().clamp(0, 15)
    return (lo + n * s).flatten(-2)


def pack(x, dtype):
    """Rows ``x [n, 128]`` (double, finite) as bytes: ``[n, 64]`` of nibbles and ``[n, 8]`` of parameters."""
    s, lo = params_of(x, dtype)
    n = torch.where(s > 0, (x.unflatten(-1, (2, 64)) - lo) / s.clamp(min=1e-300), 0).round().clamp(0, 15).long().flatten(-2)
    word = torch.zeros(x.shape[0], 16, dtype=torch.int64, device=x.device)
    for d in range(D):
        j, m, e = d // 64, d % 64 // 8, d % 8
        word[:, 2 * m + j] |= n[:, d] << (4 * (e // 2 + 4 * (e % 2)))
    data = torch.stack([word >> (8 * i) & 255 for i in range(4)], -1).flatten(1).to(torch.uint8)
    return data, torch.cat([s, lo], -1).flatten(1).to(dtype).contiguous().view(torch.uint8)


def unpack(data, params, dtype):
    """Bytes ``[n, 64]`` and ``[n, 8]`` as values (double)."""
    out = torch.empty(data.shape[0], D, dtype=torch.float64, device=data.device)
    p = params.contiguous().view(dtype).double()
    for d in range(D):
        j, m, e = d // 64, d % 64 // 8, d % 8
        place = 4 * (2 * m + j) * 2 + e // 2 + 4 * (e % 2)                  # of nibbles, low one of a byte first
        out[:, d] = p[:, 2 * j + 1] + (data[:, place // 2].long() >> (4 * (place % 2)) & 15).double() * p[:, 2 * j]
    return out


def rows_of(cache, rows, block, dtype):
    """Values of cache rows (a list), ``[n, kv_heads, 128]``."""
    r = torch.as_tensor(rows, device=cache.device).long()
    data = cache[..., :block * 64].unflatten(-1, (block, 64))[r // block, :, r % block]
    params = cache[..., block * 64:].unflatten(-1, (block, 8))[r // block, :, r % block]
    return unpack(data.reshape(-1, 64), params.reshape(-1, 8), dtype).view(len(r), cache.shape[1], D)


def set_rows(cache, rows, x, block, dtype):
    """Stores ``x [n, kv_heads, 128]`` (double, finite)."""
    r = torch.as_tensor(rows, device=cache.device).long()
    data, params = pack(x.reshape(-1, D), dtype)
    cache[..., :block * 64].unflatten(-1, (block, 64))[r // block, :, r % block] = data.view(len(r), cache.shape[1], 64)
    cache[..., block * 64:].unflatten(-1, (block, 8))[r // block, :, r % block] = params.view(len(r), cache.shape[1], 8)


def norm_rope(x, w, cos_sin, positions, eps=1e-6):
    """``x [T, heads, 128]`` (double)."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    c, s = cos_sin.view(-1, D)[positions].double()[:, None].chunk(2, -1)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def attend(q, k, v, first, scale=D ** -0.5):
    """``q [n, heads, 128]`` at positions ``first ..`` over ``k`` and ``v [keys, kv_heads, 128]``, causal, double."""
    R = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(R, 1), v.repeat_interleave(R, 1)
    s = torch.einsum("nhd,khd->hnk", q, k) * scale
    seen = torch.arange(k.shape[0], device=q.device) <= first + torch.arange(q.shape[0], device=q.device)[:, None]
    w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
    # what a query does not see has no part in its result, whatever it holds
    return torch.stack([torch.einsum("hk,khd->hd", w[:, i, :first + i + 1], v[:first + i + 1]) for i in range(q.shape[0])])


def angles(positions, device, base=1e6):
    f = base ** (-torch.arange(0, D, 2, device=device, dtype=torch.float64) / D)
    a = torch.outer(torch.arange(positions, device=device, dtype=torch.float64), f)
    return torch.cat([a.cos(), a.sin()], -1).float()
