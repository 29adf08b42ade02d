"""The operators of the 4-bit key/value cache and of pages that sequences share, as cases whose time and outputs can be measured.

Four kinds:

* ``store``: norm, rotation and 4-bit store of the tokens of a prompt step, and the stored rows read back.
* ``decode``: one token of every sequence: norm, rotation, 4-bit store and attention over the pages, and the stored rows read back.
* ``prompt``: attention of several tokens per sequence, causal, over the 4-bit pages: fresh prompts, later portions, drafts.
* ``pages``: copies of pages (or of recurrent states) in all pools of a cache, as a fork and its copy on write make them.

Heads are those of the Qwen3 architectures (16, 32 and 64 over 8 key/value heads), of their tensor-parallel shards and of one
group that is no power of two.  Caches hold quantised normal values, a few channels of the keys larger than the others.

Layout of a page: for each key/value head ``block_size`` rows of 64 bytes, then ``block_size`` rows of four 16-bit numbers, scale and
offset of dimensions 0 to 63 and of 64 to 127.  Little-endian word ``2 m + j`` of a row holds dimensions ``64 j + 8 m ..``; dimension
``2 i`` of the eight is nibble ``i``, ``2 i + 1`` is nibble ``i + 4``."""
import math

import torch

own = False

DEV, D, GROUP, ROW = "cuda", 128, 64, 72
HEADS = [(16, 8), (32, 8), (64, 8), (8, 1), (4, 1), (24, 8)]
BASE, EPS = 1e6, 1e-6
MOST = {"store": 8192 * (32 + 16), "decode": 64 * 4000 * 8, "prompt": 8000 * 8000 // 2 * 32, "pages": 56 * 32 * 8 * 256 * ROW}


def listed():
    return [
        # a short prompt of the small model
        {"name": "store 100", "kind": "store", "tokens": 100, "prompts": 3, "start": 0, "heads": 16, "kv_heads": 8, "block": 256, "dtype": "float16"},
        # a portion of a long prompt
        {"name": "store 4096", "kind": "store", "tokens": 4096, "prompts": 2, "start": 1000, "heads": 32, "kv_heads": 8, "block": 256, "dtype": "bfloat16"},
        # one user at the start of an answer: all latency
        {"name": "decode 1 x 37", "kind": "decode", "batch": 1, "context": 37, "idle": 0, "heads": 16, "kv_heads": 8, "block": 256, "dtype": "float16"},
        # one user behind a long document
        {"name": "decode 1 x 32000", "kind": "decode", "batch": 1, "context": 32000, "idle": 0, "heads": 32, "kv_heads": 8, "block": 256, "dtype": "bfloat16"},
        # a server under load, a few rows of the step without a sequence
        {"name": "decode 45 x 1500", "kind": "decode", "batch": 45, "context": 1500, "idle": 3, "heads": 32, "kv_heads": 8, "block": 256, "dtype": "bfloat16"},
        # a full batch of long sequences of the large model, small pages
        {"name": "decode 64 x 4000", "kind": "decode", "batch": 64, "context": 4000, "idle": 0, "heads": 64, "kv_heads": 8, "block": 16, "dtype": "float16"},
        # short prompts of several users in one step
        {"name": "prompts 5 of 300", "kind": "prompt", "tokens": 300, "prompts": 5, "start": 0, "heads": 16, "kv_heads": 8, "block": 256, "dtype": "float16"},
        # drafted tokens of four sequences, to be judged in one step
        {"name": "drafts 4 x 5", "kind": "prompt", "tokens": 20, "prompts": 4, "start": 3001, "heads": 32, "kv_heads": 8, "block": 256, "dtype": "float16"},
        # a portion of a long prompt of the large model
        {"name": "portion 500 of 12500", "kind": "prompt", "tokens": 500, "prompts": 1, "start": 12000, "heads": 64, "kv_heads": 8, "block": 256, "dtype": "bfloat16"},
        # a whole long prompt: the most work
        {"name": "prompt 8000", "kind": "prompt", "tokens": 8000, "prompts": 1, "start": 0, "heads": 32, "kv_heads": 8, "block": 256, "dtype": "bfloat16"},
        # one fork: the page in which the sequence stands, of every layer of the small model
        {"name": "pages 1", "kind": "pages", "pools": 56, "pairs": 1, "spare": 6, "item": 8 * 256 * ROW, "dtype": "uint8"},
        # a batch of forks: their pages, or a compaction
        {"name": "pages 32", "kind": "pages", "pools": 56, "pairs": 32, "spare": 16, "item": 8 * 256 * ROW, "dtype": "uint8"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "prompt", "prompt", "pages"])
    while True:
        if kind == "pages":
            # pages of 16 or 4 bits, rows of recurrent states (float), an odd number of values among them
            item, dtype = rng.choice([(8 * 256 * ROW, "uint8"), (8 * 16 * ROW, "uint8"), (256 * 8 * D, "float16"), (1000 + rng.randint(0, 99), "float32"), (128 * 256, "float32")])
            c = {"kind": kind, "pools": rng.randint(2, 60), "pairs": _log_int(rng, 1, 32), "spare": rng.randint(0, 9), "item": item, "dtype": dtype}
            cost = c["pools"] * c["pairs"] * item * {"uint8": 1, "float16": 2, "float32": 4}[dtype]
        else:
            heads, kv_heads = rng.choice(HEADS)
            c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "block": rng.choice([16, 48, 256, 256]), "dtype": rng.choice(["float16", "bfloat16"])}
            if kind == "store":
                c.update(tokens=_log_int(rng, 1, 8192), prompts=rng.randint(1, 4), start=rng.choice([0, _log_int(rng, 1, 20000)]))
                cost = c["tokens"] * (heads + 2 * kv_heads)
            elif kind == "decode":
                c.update(batch=_log_int(rng, 1, 64), context=_log_int(rng, 1, 32000), idle=rng.choice([0, 0, 2]))
                cost = c["batch"] * c["context"] * kv_heads
            else:
                c.update(tokens=_log_int(rng, 2, 8000), prompts=rng.randint(1, 6), start=rng.choice([0, 0, _log_int(rng, 1, 20000)]))
                cost = heads * sum(n * s + n * n // 2 for n, s in zip(*_prompts(c)))
        if cost <= MOST[kind]:
            return c


# ------------------------------------------------------------------ sizes
def _prompts(case):
    """Tokens that each sequence brings, and the positions they start at."""
    n, k = case["tokens"], min(case["prompts"], case["tokens"])
    weights = [3 + i for i in range(k)]
    lens = [max(1, n * w // sum(weights)) for w in weights]
    lens[-1] += max(0, n - sum(lens))
    return lens, [case["start"] - (31 * i) % (case["start"] // 3 + 1) for i in range(k)]


def _contexts(case):
    """Keys that each sequence of a decode step sees, its own token among them; 0: a row without a sequence."""
    n = case["context"]
    live = [n - (37 * i) % (n // 4 + 1) for i in range(case["batch"])]
    for i in range(case["idle"]):
        live.insert(5 * i % len(live), 0)
    return live


def _visible(case):
    """Pairs of a query and a key that it sees."""
    return sum(n * s + n * (n + 1) // 2 for n, s in zip(*_prompts(case)))


def work(case):
    if case["kind"] == "pages":
        return {"bytes": 2 * case["pools"] * case["pairs"] * case["item"] * {"uint8": 1, "float16": 2, "float32": 4}[case["dtype"]], "flops": 0}
    hq, hk = case["heads"], case["kv_heads"]
    if case["kind"] == "prompt":
        lens, starts = _prompts(case)
        return {"bytes": 2 * 2 * D * hq * sum(lens) + 2 * ROW * hk * (sum(lens) + sum(starts)), "flops": 4 * D * hq * _visible(case)}
    if case["kind"] == "store":
        T = sum(_prompts(case)[0])
        keys = 0
    else:
        T = sum(n > 0 for n in _contexts(case))
        keys = sum(n - 1 for n in _contexts(case) if n)
    # projections and angles in, queries (or the attention's output) out, rows stored, and their values read back
    return {"bytes": T * (2 * D * (2 * hq + 2 * hk) + 4 * D + 2 * ROW * hk + 4 * D * hk) + 2 * ROW * hk * keys,
            "flops": T * D * 12 * (hq + 2 * hk) + 4 * D * hq * (keys + T if case["kind"] == "decode" else 0)}


# ------------------------------------------------------------------ inputs
def _angles(positions):
    f = BASE ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    a = torch.outer(torch.arange(positions, device=DEV, dtype=torch.float64), f)
    return torch.cat([a.cos(), a.sin()], -1).float()


def _random_cache(blocks, kv_heads, block, dtype, g, keys):
    x = torch.randn(blocks, kv_heads, block, D, generator=g, device=DEV, dtype=torch.float16).float()
    if keys:
        x[..., 5::32] *= 4
    else:
        x *= 0.3
    data, params = _quantise(x, dtype)
    return torch.cat([data.flatten(2), params.flatten(2)], -1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    if case["kind"] == "pages":
        places = 2 * case["pairs"] + case["spare"]
        dtype = getattr(torch, case["dtype"])
        make = lambda: (torch.randint(0, 256, (places, case["item"]), generator=g, device=DEV, dtype=torch.uint8) if dtype == torch.uint8 else  # noqa: E731
                        torch.randn(places, case["item"], generator=g, device=DEV, dtype=dtype))
        order = torch.randperm(places, generator=host)
        return {"case": case, "pools": [make() for _ in range(case["pools"])],
                "sources": order[:case["pairs"]].tolist(), "targets": order[case["pairs"]:2 * case["pairs"]].tolist()}
    dtype, hq, hk, block = getattr(torch, case["dtype"]), case["heads"], case["kv_heads"], case["block"]
    if case["kind"] == "decode":
        ends = _contexts(case)
        lens, starts = [1] * len(ends), [n - 1 for n in ends]
    else:
        lens, starts = _prompts(case)
        ends = [n + s for n, s in zip(lens, starts)]
    need = [-(-n // block) for n in ends]
    width = max(max(need), 1)
    order = torch.randperm(sum(need) + 1, generator=host)      # one page that no sequence has
    table = torch.full((len(ends), width), -1, dtype=torch.int32)
    o = 0
    for b, n in enumerate(need):
        table[b, :n] = order[o:o + n]
        o += n
    positions = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)]).clamp_(min=0)
    which = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    page = table[which, positions // block].long()
    rows = torch.where(page >= 0, page * block + positions % block, -1)
    T = sum(lens)
    s = {"case": case, "lens": lens, "starts": starts, "table": table.to(DEV), "rows": rows.to(DEV), "positions": positions.to(DEV),
         "cu": torch.tensor([0] + lens).cumsum(0).int().to(DEV), "pos0": torch.tensor(starts).clamp(min=0).int().to(DEV),
         "ctx": torch.tensor(ends).int().to(DEV)}
    s["k_cache"] = _random_cache(sum(need) + 1, hk, block, dtype, g, True)
    s["v_cache"] = _random_cache(sum(need) + 1, hk, block, dtype, g, False)
    if case["kind"] == "prompt":      # queries as the norm and the rotation leave them
        s["q"] = torch.randn(T, hq * D, generator=g, device=DEV).to(dtype)
        return s
    s["qkv"] = torch.randn(T, (hq + 2 * hk) * D, generator=g, device=DEV).to(dtype)
    s["q_weight"], s["k_weight"] = ((1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dtype) for _ in range(2))
    s["angles"] = _angles(max(ends) + 1)
    return s


# ------------------------------------------------------------------ the plain form
def _quantise(x, dtype):
    """``x [..., 128]`` (float): packed rows ``[..., 64]`` and parameters ``[..., 8]``, both bytes."""
    x = x.unflatten(-1, (2, GROUP))
    lo = x.amin(-1, keepdim=True).to(dtype).float()
    scale = ((x.amax(-1, keepdim=True) - lo) / 15).to(dtype)
    s = scale.float()
    n = torch.where(s > 0, (x - lo) / s, 0).round_().clamp_(0, 15).to(torch.int32)
    n = n.unflatten(-1, (8, 4, 2)).transpose(-1, -2).flatten(-2)           # [..., group, eight dimensions, nibble]
    n = (n << (4 * torch.arange(8, device=x.device, dtype=torch.int32))).sum(-1, dtype=torch.int32)
    data = n.transpose(-1, -2).flatten(-2).contiguous().view(torch.uint8)
    params = torch.stack([scale.squeeze(-1), lo.squeeze(-1).to(dtype)], -1).flatten(-2).contiguous().view(torch.uint8)
    return data, params


def _values(data, params, dtype):
    """What packed rows stand for, in float."""
    w = data.contiguous().view(torch.int32).unflatten(-1, (8, 2)).transpose(-1, -2)         # [..., group, eight dimensions]
    n = (w.unsqueeze(-1) >> (4 * torch.arange(8, device=w.device, dtype=torch.int32))) & 15
    n = n.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-3)              # [..., group, 64]
    p = params.contiguous().view(dtype).unflatten(-1, (2, 2)).float()
    return (p[..., 1:] + n * p[..., :1]).flatten(-2)


def _split(cache, block):
    """Views ``[pages, kv_heads, block, 64]`` and ``[pages, kv_heads, block, 8]`` of a cache."""
    return cache[..., :block * 64].unflatten(-1, (block, 64)), cache[..., block * 64:].unflatten(-1, (block, 8))


def _write(cache, rows, x, dtype, block):
    data, params = _split(cache, block)
    live = rows >= 0
    r = rows[live]
    d, p = _quantise(x[live], dtype)
    data[r // block, :, r % block] = d
    params[r // block, :, r % block] = p


def _read(cache, rows, dtype, block):
    data, params = _split(cache, block)
    r = rows.clamp(min=0)
    x = _values(data[r // block, :, r % block], params[r // block, :, r % block], dtype)
    return torch.where((rows >= 0)[:, None, None], x, 0).to(dtype)


def _gather(cache, table, dtype, block):
    """Values of all pages of a table, ``[batch, kv_heads, width * block, 128]``; pages that are not there give zeros."""
    data, params = _split(cache, block)
    t = table.clamp(min=0).long()
    x = _values(data[t], params[t], dtype).transpose(1, 2).flatten(2, 3)
    return torch.where((table >= 0).repeat_interleave(block, 1)[:, None, :, None], x, 0)


def _heads(s):
    """Queries, keys and values of a step, normed and rotated, in float."""
    c = s["case"]
    hq, hk = c["heads"], c["kv_heads"]
    x = s["qkv"].float().unflatten(-1, (-1, D))
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    cos, sin = s["angles"][s["positions"]][:, None].chunk(2, -1)

    def turn(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.float()
        a, b = y.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return turn(q, s["q_weight"]), turn(k, s["k_weight"]), v


def _attend(q, k, v, mask):
    """q ``[batch, kv_heads, queries, 128]`` over k and v ``[batch, kv_heads, keys, 128]``; mask ``[batch, queries, keys]``."""
    s = torch.matmul(q * D ** -0.5, k.transpose(-1, -2))
    s.masked_fill_(~mask[:, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    l = s.sum(-1, keepdim=True)
    return torch.where(l > 0, torch.matmul(s, v) / l, 0)


def _plain(s):
    case = s["case"]
    if case["kind"] == "pages":
        a, b = torch.tensor([s["sources"], s["targets"]]).to(DEV)
        return [p.index_copy_(0, b, p[a]) for p in s["pools"]]
    dtype, hq, hk, block = getattr(torch, case["dtype"]), case["heads"], case["kv_heads"], case["block"]
    R = hq // hk
    if case["kind"] == "prompt":
        n = max(s["lens"])
        step = torch.arange(n, device=DEV)
        at = s["cu"][:-1, None] + step                                                        # [batch, n]
        there = step < (s["cu"][1:] - s["cu"][:-1])[:, None]
        q = s["q"].float()[torch.where(there, at, 0)].unflatten(-1, (hk, R, D)).transpose(1, 2).flatten(2, 3)      # rows: token, head of the group
        k, v = _gather(s["k_cache"], s["table"], dtype, block), _gather(s["v_cache"], s["table"], dtype, block)
        pos = (s["pos0"][:, None] + step).repeat_interleave(R, 1)
        o = _attend(q, k, v, torch.arange(k.shape[2], device=DEV) <= pos[..., None])
        return o.unflatten(2, (n, R)).transpose(1, 2).flatten(2)[there].to(dtype)
    q, k, v = _heads(s)
    _write(s["k_cache"], s["rows"], k, dtype, block)
    _write(s["v_cache"], s["rows"], v, dtype, block)
    back = [_read(s[c], s["rows"], dtype, block) for c in ("k_cache", "v_cache")]
    if case["kind"] == "store":
        return [q.flatten(1).to(dtype)] + back
    k, v = _gather(s["k_cache"], s["table"], dtype, block), _gather(s["v_cache"], s["table"], dtype, block)
    o = _attend(q.unflatten(1, (hk, R)), k, v, (torch.arange(k.shape[2], device=DEV) < s["ctx"][:, None])[:, None])
    return [o.flatten(1).to(dtype)] + back


# ------------------------------------------------------------------ the framework's calls
def _framework(s):
    from nanoquantization_b200.layers import kv4, pages
    case = s["case"]
    if case["kind"] == "pages":
        pages.copy_pages(s["pools"], s["sources"], s["targets"])
        return s["pools"]
    hq, hk = case["heads"], case["kv_heads"]
    if case["kind"] == "prompt":
        return kv4.prompt_attention(s["q"], hq, s["k_cache"], s["v_cache"], s["table"], s["cu"], s["pos0"], s["lens"], s["starts"])
    if case["kind"] == "store":
        out = kv4.qknorm_rope_store(s["qkv"], s["q_weight"], s["k_weight"], s["angles"], s["positions"], hq, hk, EPS, s["k_cache"], s["v_cache"], s["rows"])
    else:
        out = kv4.decode_attention(s["qkv"], s["q_weight"], s["k_weight"], s["angles"], s["positions"], hq, hk, EPS, s["k_cache"], s["v_cache"], s["table"],
                                   s["ctx"], s["rows"])
    return [out, *kv4.load(s["k_cache"], s["v_cache"], s["rows"], s["qkv"].dtype)]


@torch.no_grad()
def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------ from the definition, in 64 bits
def _levels(x, dtype):
    """The values that quantised rows of ``x`` (double) stand for."""
    out = []
    for part in x.split(GROUP, -1):
        low = part.min(-1, keepdim=True).values.to(dtype).double()
        step = ((part.max(-1, keepdim=True).values - low) / 15).to(dtype).double()
        level = ((part - low) / step.clamp(min=1e-300)).round().clamp(0, 15)
        out.append(torch.where(step > 0, low + level * step, low))
    return torch.cat(out, -1)


def _sequence(cache, pages, n, dtype, block):
    """The first n rows of a sequence, double ``[n, kv_heads, 128]``: byte by byte, from the layout's description."""
    c = cache[pages]
    byte = c[..., :block * 64].reshape(len(pages), c.shape[1], block, 8, 2, 4)             # piece m, group j, byte of the word
    nib = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)                            # nibbles 0 .. 7 of the word
    dims = torch.empty_like(nib)
    for i in range(4):
        dims[..., 2 * i], dims[..., 2 * i + 1] = nib[..., i], nib[..., i + 4]
    level = dims.transpose(3, 4).flatten(4).double()                                     # [page, head, row, group, 64]
    par = c[..., block * 64:].contiguous().view(dtype).reshape(len(pages), c.shape[1], block, 2, 2).double()
    x = (par[..., 1:] + level * par[..., :1]).flatten(3)
    return x.transpose(1, 2).flatten(0, 1)[:n]


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "pages":
        if case["dtype"] == "uint8":
            return None
        out = []
        for p in s["pools"]:
            p = p.double()
            for a, b in zip(s["sources"], s["targets"]):
                p[b] = p[a]
            out.append(p)
        return out
    dtype, hq, hk, block = getattr(torch, case["dtype"]), case["heads"], case["kv_heads"], case["block"]
    R = hq // hk
    if case["kind"] != "prompt":
        heads = s["qkv"].double().view(-1, hq + 2 * hk, D)
        angle = s["angles"][s["positions"]].double()
        turned = []
        for x, w in ((heads[:, :hq], s["q_weight"]), (heads[:, hq:hq + hk], s["k_weight"])):
            x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            c, sn = angle[:, None, :64], angle[:, None, 64:]
            turned.append(torch.cat([x[..., :64] * c - x[..., 64:] * sn, x[..., :64] * sn + x[..., 64:] * c], -1))
        q, k, v = turned[0], _levels(turned[1], dtype), _levels(heads[:, hq + hk:], dtype)
        idle = s["rows"] < 0
        k[idle], v[idle] = 0, 0
        if case["kind"] == "store":
            return [q.flatten(1), k, v]
    else:
        q = s["q"].double().view(-1, hq, D)
    out, o = [], 0
    for b, (n, start) in enumerate(zip(s["lens"], s["starts"])):
        if start < 0:
            out.append(torch.zeros(n, hq, D, dtype=torch.float64, device=DEV))
            o += n
            continue
        pages = s["table"][b][:-(-(start + n) // block)].long()
        keys, vals = (_sequence(s[c], pages, start + n, dtype, block) for c in ("k_cache", "v_cache"))
        if case["kind"] == "decode":
            keys[-1], vals[-1] = k[o], v[o]
        seen = torch.arange(start + n, device=DEV) <= torch.arange(start, start + n, device=DEV)[:, None]
        got = []
        for h in range(hq):
            w = q[o:o + n, h] @ keys[:, h // R].T / math.sqrt(D)
            w = torch.softmax(w.masked_fill(~seen, -math.inf), -1)
            got.append(w @ vals[:, h // R])
        out.append(torch.stack(got, 1))
        o += n
    out = torch.cat(out).flatten(1)
    return out if case["kind"] == "prompt" else [out, k, v]
