"""The operators for a long stream of tokens, as measurable cases: attention with a sliding window and sinks, and the
K/V cache held in 4 bits with its append, its read and the attention over it.

Where `own` is false the operators are computed in their plain form with elementary torch operations in float32, where
it is true by the framework's own entry points (`torch.ops.rldx_amd`).  `exact` evaluates the definitions in float64,
apart from the plain form.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DEV = "cuda"


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
# window: queries [batch, seq_q] behind a past of seq_k - seq_q keys; `pad`: the batch is padded on the left to ragged
# lengths.  append: `seq` new tokens of each sequence into its pages, read back as values.  cache: `seq_q` new queries of
# each sequence, the longest of which holds `slots` tokens (the others are `ragged` or as long); window 0: every slot.
def listed():
    return [
        # One new token of a robot's stream, its window of 1024 tokens and the first 4.
        {"name": "window_token", "kind": "window", "batch": 1, "seq_q": 1, "seq_k": 4096, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "window": 1024, "sinks": 4, "pad": False},
        # The tokens of one more camera image behind a stream (the backbone's prompt of one image: 169 tokens).
        {"name": "window_image", "kind": "window", "batch": 1, "seq_q": 169, "seq_k": 1449, "q_heads": 28,
         "kv_heads": 4, "head_dim": 128, "window": 1000, "sinks": 16, "pad": False},
        # A prompt with several camera images, prefilled with a short window.
        {"name": "window_prompt", "kind": "window", "batch": 1, "seq_q": 1280, "seq_k": 1280, "q_heads": 28,
         "kv_heads": 4, "head_dim": 128, "window": 512, "sinks": 64, "pad": False},
        # Video history of several cameras, prefilled.
        {"name": "window_history", "kind": "window", "batch": 1, "seq_q": 8192, "seq_k": 8192, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "window": 1024, "sinks": 4, "pad": False},
        # Eight robots' streams of different lengths, padded on the left, heads of 64 without sharing.
        {"name": "window_padded", "kind": "window", "batch": 8, "seq_q": 777, "seq_k": 777, "q_heads": 24,
         "kv_heads": 24, "head_dim": 64, "window": 200, "sinks": 3, "pad": True},
        # One token of each of eight robots enters the cache and is read back.
        {"name": "append_token", "kind": "append", "batch": 8, "seq": 1, "kv_heads": 8, "head_dim": 128, "past": 1000,
         "page": 64},
        # A prompt of one image for two robots, heads of 64.
        {"name": "append_image", "kind": "append", "batch": 2, "seq": 169, "kv_heads": 24, "head_dim": 64, "past": 333,
         "page": 32},
        # A long history enters the cache at once.
        {"name": "append_history", "kind": "append", "batch": 4, "seq": 8192, "kv_heads": 8, "head_dim": 128, "past": 5,
         "page": 64},
        # One token of one robot over a short cache: latency.
        {"name": "cache_token", "kind": "cache", "batch": 1, "seq_q": 1, "slots": 1281, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "window": 0, "sinks": 0, "ragged": False, "page": 64},
        # One token of each of sixteen robots with caches of different lengths, heads of 64.
        {"name": "cache_robots", "kind": "cache", "batch": 16, "seq_q": 1, "slots": 8000, "q_heads": 24, "kv_heads": 8,
         "head_dim": 64, "window": 4096, "sinks": 16, "ragged": True, "page": 32},
        # One token over a day's long stream.
        {"name": "cache_long", "kind": "cache", "batch": 1, "seq_q": 1, "slots": 131072, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "window": 0, "sinks": 0, "ragged": False, "page": 64},
        # The tokens of a small image of each of two robots over their caches (7 query heads per KV head).
        {"name": "cache_chunk", "kind": "cache", "batch": 2, "seq_q": 49, "slots": 6000, "q_heads": 28, "kv_heads": 4,
         "head_dim": 128, "window": 0, "sinks": 0, "ragged": True, "page": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, dim = rng.choice([(32, 8, 128), (28, 4, 128), (16, 8, 128), (12, 12, 128), (24, 24, 64), (24, 8, 64)])
    kind = rng.choice(["window", "window", "append", "cache", "cache"])
    if kind == "window":
        form = rng.choice(["token", "chunk", "prefill"])
        if form == "token":
            batch, sq, sk = _log(rng, 1, 16), rng.randint(1, 4), _log(rng, 8, 32768)
        elif form == "chunk":
            batch, sq = rng.randint(1, 3), _log(rng, 5, 512)
            sk = sq + _log(rng, 1, 8192)
        else:
            sq = sk = _log(rng, 33, 8192)
            batch = rng.randint(1, max(1, min(8, 8192 // sq)))
        return {"kind": kind, "batch": batch, "seq_q": sq, "seq_k": sk, "q_heads": hq, "kv_heads": hkv, "head_dim": dim,
                "window": _log(rng, 16, 1024), "sinks": rng.choice([0, 1, 4, 16, 40]), "pad": rng.random() < 0.3}
    if kind == "append":
        batch, seq = _log(rng, 1, 16), _log(rng, 1, 8192)
        return {"kind": kind, "batch": min(batch, max(1, 32768 // seq)), "seq": seq, "kv_heads": hkv if hkv <= 8 else 8,
                "head_dim": dim, "past": rng.randint(0, 2000), "page": rng.choice([32, 64, 128, 256])}
    slots = _log(rng, 1, 131072)
    batch = _log(rng, 1, max(1, min(16, 131072 // slots)))
    sq = 1 if rng.random() < 0.6 else _log(rng, 2, max(2, min(64, slots, 1 + 600000 // (slots * batch))))
    return {"kind": kind, "batch": batch, "seq_q": min(sq, slots), "slots": slots, "q_heads": hq,
            "kv_heads": hkv if hkv <= 8 else 8 if hq % 8 == 0 else 4, "head_dim": dim,
            "window": rng.choice([0, 0, _log(rng, 16, 8192)]), "sinks": rng.choice([0, 4, 33]),
            "ragged": rng.random() < 0.5, "page": rng.choice([32, 64, 128, 256])}


# ---------------------------------------------------------------------------
# the cache's layout
# ---------------------------------------------------------------------------
# cache [pages, kv_heads, page / 32 * tile] uint8, a tile of 32 slots holding
#   K codes  [slot][head_dim] 4 bits each, the even dimension in the low half of its byte
#   V codes  [slot / 4 % 4][dim / (head_dim / 16)][slot / 16][slot % 4][dim % (head_dim / 16)], 4 bits each
#   K scales [slot][head_dim / 32] bytes, V scales [head_dim / 32][slot / 4 % 4][slot / 16][slot % 4] bytes
# Code bit 3 is the sign, the others one of 0, .5, 1, 1.5, 2, 3, 4, 6; scale byte e stands for 2^(e - 127), 255 for NaN.
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _tile_bytes(dim):
    return 32 * dim + 64 * (dim // 32)


def _nibbles(codes):
    """[..., 2 n] codes -> [..., n] bytes."""
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _quantise(x):
    """Rows [..., dim] -> codes [..., dim] and scale bytes [..., dim / 32], both uint8."""
    b = x.to(F32).unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    bits = amax.view(torch.int32)
    up = (bits & 0x7FFFFF) >= 0x600000  # amax / 2^p >= 1.75
    e = ((bits >> 23) - 129 + up.to(torch.int32)).clamp(-125, 125)
    # 2^-e in two exact factors
    h = e // 2
    y = b.abs() * torch.exp2(-h.to(F32)).unsqueeze(-1) * torch.exp2((h - e).to(F32)).unsqueeze(-1)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code = code.to(torch.uint8) | (torch.signbit(b).to(torch.uint8) << 3)
    bad = ~torch.isfinite(b).all(-1)
    return code.flatten(-2), torch.where(bad, 255, e + 127).to(torch.uint8)


def _values(codes, scales):
    """Codes [..., dim] and scale bytes [..., dim / 32] -> float32 values."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=F32, device=codes.device)
    v = grid[codes.to(torch.int32)].unflatten(-1, (-1, 32))
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.to(F32) - 127.0))
    return (v * s.unsqueeze(-1)).flatten(-2)


def _to_tiles(kc, ks, vc, vs):
    """Codes and scales [..., 32 n slots, dim] -> tiles [..., n, tile bytes]."""
    dim = kc.shape[-1]
    k = _nibbles(kc).unflatten(-2, (-1, 32)).flatten(-2)
    v = vc.unflatten(-2, (-1, 2, 4, 4)).unflatten(-1, (16, dim // 16))  # n, slot/16, slot/4%4, slot%4, group, dim
    n = v.dim()
    v = v.permute(*range(n - 5), n - 4, n - 2, n - 5, n - 3, n - 1)
    v = _nibbles(v).flatten(-5)
    s = ks.unflatten(-2, (-1, 32)).flatten(-2)
    t = vs.unflatten(-2, (-1, 2, 4, 4))  # n, slot/16, slot/4%4, slot%4, block
    n = t.dim()
    t = t.permute(*range(n - 4), n - 1, n - 3, n - 4, n - 2).flatten(-4)
    return torch.cat([k, v, s, t], -1)


def _from_tiles(tiles, dim):
    """Tiles [..., n, tile bytes] -> float32 K and V [..., 32 n slots, dim]."""
    k, v, s, t = tiles.split([16 * dim, 16 * dim, dim, dim], -1)
    spread = lambda x: torch.stack([x & 15, x >> 4], -1).flatten(-2)  # noqa: E731
    kc = spread(k).unflatten(-1, (32, dim)).flatten(-3, -2)
    vc = spread(v).unflatten(-1, (4, 16, 2, 4, dim // 16))  # slot/4%4, group, slot/16, slot%4, dim
    n = vc.dim()
    vc = vc.permute(*range(n - 5), n - 3, n - 5, n - 2, n - 4, n - 1).flatten(-2).flatten(-4, -2).flatten(-3, -2)
    ks = s.unflatten(-1, (32, dim // 32)).flatten(-3, -2)
    vs = t.unflatten(-1, (dim // 32, 4, 2, 4))
    n = vs.dim()
    vs = vs.permute(*range(n - 4), n - 2, n - 3, n - 1, n - 4).flatten(-4, -2).flatten(-3, -2)
    return _values(kc, ks), _values(vc, vs)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=F32)


def _keys(g, batch, seq, heads, dim):
    """Keys as a norm and a rotation leave them: rows of similar length, a few dimensions larger than the others."""
    wide = torch.exp(0.5 * _rand(g, 1, 1, heads, dim))
    return (_rand(g, batch, seq, heads, dim) * wide).to(BF16)


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEV)


def _pages(g, c, slots):
    """A cache with a table of its pages in any order; bytes that nobody has written hold whatever was there."""
    per = -(-slots // c["page"])
    n = c["batch"] * per
    cache = _ints(g, 0, 256, n + 3, c["kv_heads"], c["page"] // 32 * _tile_bytes(c["head_dim"])).to(torch.uint8)
    table = torch.randperm(n + 3, generator=g, device=DEV)[:n].to(torch.int32).view(c["batch"], per)
    return cache, table


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(seed)
    B, D = c["batch"], c["head_dim"]
    if c["kind"] == "window":
        s = {"q": _rand(g, B, c["seq_q"], c["q_heads"], D).to(BF16), "k": _keys(g, B, c["seq_k"], c["kv_heads"], D),
             "v": _rand(g, B, c["seq_k"], c["kv_heads"], D).to(BF16), "mask": None}
        if c["pad"]:  # sequence b's keys begin behind its padding
            first = _ints(g, 0, max(1, c["seq_k"] // 2), B, 1)
            s["mask"] = (torch.arange(c["seq_k"], device=DEV) >= first).to(F32)
    elif c["kind"] == "append":
        cache, table = _pages(g, c, c["past"] + c["seq"])
        s = {"k": _keys(g, B, c["seq"], c["kv_heads"], D), "v": _rand(g, B, c["seq"], c["kv_heads"], D).to(BF16),
             "cache": cache, "table": table, "starts": _ints(g, c["past"] // 2, c["past"] + 1, B).to(torch.int32)}
    else:
        cache, table = _pages(g, c, c["slots"])
        first = c["slots"] - c["seq_q"]
        starts = _ints(g, first // 4 if c["ragged"] else first, first + 1, B)
        starts[0] = first
        # the tokens so far, the new ones' among them, behind which nobody has written anything
        n = table.shape[1] * c["page"]
        k = _keys(g, B, n, c["kv_heads"], D).transpose(1, 2)
        v = _rand(g, B, n, c["kv_heads"], D).to(BF16).transpose(1, 2)
        tiles = _to_tiles(*_quantise(k), *_quantise(v))  # [B, heads, tiles, bytes]
        t = torch.arange(n // 32, device=DEV) * 32 < (starts + c["seq_q"])[:, None]
        per = c["page"] // 32
        old = cache[table.long()].unflatten(-1, (per, -1)).transpose(2, 3).flatten(1, 2).transpose(1, 2)
        tiles = torch.where(t[:, None, :, None], tiles, old)
        cache[table.long()] = tiles.unflatten(2, (-1, per)).transpose(1, 2).flatten(-2)
        s = {"q": _rand(g, B, c["seq_q"], c["q_heads"], D).to(BF16), "cache": cache, "table": table,
             "starts": starts.to(torch.int32)}
    return {"case": dict(c), **s}


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def _ops():
    if "rldx_amd.ops" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "rldx-1_amd"))
        import rldx_amd.ops  # noqa: F401  (registers the operators)
    return torch.ops.rldx_amd


def _attend(q, k, v, visible):
    """q [B, Sq, Hq, D], k and v [B, Hkv, S, D] in float32, visible [B, 1, Sq, S] -> bf16 [B, Sq, Hq, D]."""
    B, Sq, Hq, D = q.shape
    Hkv = k.shape[1]
    x = q.to(F32).permute(0, 2, 1, 3).reshape(B, Hkv, Hq // Hkv * Sq, D)
    s = torch.matmul(x, k.transpose(2, 3).contiguous()).view(B, Hq, Sq, -1) / math.sqrt(D)
    s = torch.where(visible, s, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p.view(B, Hkv, Hq // Hkv * Sq, -1), v).view(B, Hq, Sq, D)
    return o.permute(0, 2, 1, 3).to(BF16).contiguous()


def _in_window(at, keys, window, sinks):
    return (keys <= at) & ((keys > at - window) | (keys < sinks))


def run(state):
    c = state["case"]
    if c["kind"] == "window":
        q, k, v, mask = state["q"], state["k"], state["v"], state["mask"]
        if own:
            return _ops().window_attention(q, k, v, c["window"], c["sinks"], mask)
        at = torch.arange(c["seq_k"] - c["seq_q"], c["seq_k"], device=DEV)[:, None]
        visible = _in_window(at, torch.arange(c["seq_k"], device=DEV), c["window"], c["sinks"])[None, None]
        if mask is not None:
            visible = visible & (mask != 0)[:, None, None, :]
        return _attend(q, k.to(F32).transpose(1, 2).contiguous(), v.to(F32).transpose(1, 2).contiguous(), visible)
    table, starts, cache = state["table"], state["starts"], state["cache"]
    if c["kind"] == "append":
        k, v = state["k"], state["v"]
        if own:
            _ops().kv4_append(cache, k, v, table, starts)
            return _ops().kv4_read(cache, table, starts, c["seq"], c["head_dim"])
        return tuple(_values(*_quantise(x)).to(BF16) for x in (k, v))
    if own:
        return _ops().kv4_attention(state["q"], cache, table, starts, None, c["window"] or None, c["sinks"])
    tiles = cache[table.long()].unflatten(-1, (c["page"] // 32, -1)).transpose(2, 3).flatten(1, 2).transpose(1, 2)
    k, v = _from_tiles(tiles, c["head_dim"])
    keys = torch.arange(k.shape[2], device=DEV)
    at = starts.long()[:, None, None] + torch.arange(c["seq_q"], device=DEV)[:, None]
    visible = _in_window(at, keys, c["window"] or k.shape[2], c["sinks"])
    written = (keys < (starts + c["seq_q"])[:, None])[:, None, :, None]
    return _attend(state["q"], torch.where(written, k, 0.0), torch.where(written, v, 0.0), visible[:, None])


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _row(q, k, v, at, c, mask=None):
    """Queries q [n, G, D] at the slots `at` [n], keys k, v [S, D] of one KV head, in float64 -> [n, G, D]."""
    j = torch.arange(k.shape[0], device=DEV)
    window = c["window"] or k.shape[0]
    hidden = (j[None] > at[:, None]) | ((j[None] <= at[:, None] - window) & (j[None] >= c["sinks"]))
    if mask is not None:
        hidden = hidden | (mask == 0)[None]
    s = torch.matmul(q.flatten(0, 1), k.t().contiguous()).unflatten(0, q.shape[:2]) * q.shape[-1] ** -0.5
    s = s.masked_fill(hidden[:, None], -math.inf)
    p = torch.softmax(s, -1).masked_fill(hidden.all(-1)[:, None, None], 0.0)
    return torch.matmul(p.flatten(0, 1), v).unflatten(0, q.shape[:2])


def _stored(cache, pages, head, dim, page, n):
    """K and V [n, dim] of the first n slots of a sequence's pages, in float64, byte by byte as the layout says."""
    t, d = torch.arange(n, device=DEV), torch.arange(dim, device=DEV)
    r, w = t % 32, dim // 16
    where = t % page // 32 * _tile_bytes(dim)
    rows = cache[pages[t // page].long(), head]  # [n, page bytes]
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F64, device=DEV)
    unit = (r // 4 % 4 * 16)[:, None] + d // w
    nib = {"k": r[:, None] * dim + d, "v": 32 * dim + (unit * 8 + (r // 16 * 4 + r % 4)[:, None]) * w + d % w}
    scale = {"k": 32 * dim + r[:, None] * (dim // 32) + d // 32,
             "v": 33 * dim + (d // 32 * 4 + (r // 4 % 4)[:, None]) * 8 + (r // 16 * 4 + r % 4)[:, None]}
    got = []
    for x in ("k", "v"):
        byte = rows.gather(1, where[:, None] + nib[x] // 2).long()
        code = torch.where(nib[x] % 2 == 0, byte % 16, byte // 16)
        e = rows.gather(1, where[:, None] + scale[x]).to(F64)
        got.append(torch.where(code >= 8, -1.0, 1.0).to(F64) * grid[code % 8] * torch.pow(2.0, e - 127))
    return got


def _nearest(x):
    """[..., dim] in float64 -> the values that it stands for in 4 bits."""
    b = x.unflatten(-1, (-1, 32))
    f, p = torch.frexp(b.abs().amax(-1, keepdim=True))  # f in [0.5, 1)
    e = (p - 3 + (f >= 0.875).to(p.dtype)).clamp(-125, 125)
    e = torch.where(f == 0, -125, e).to(F64)
    y = (b * torch.pow(2.0, -e)).abs()
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F64, device=DEV)
    odd = torch.tensor([0.0, 1e-12] * 4, dtype=F64, device=DEV)  # of two as near, the even code
    best = torch.zeros_like(y)
    near = torch.full_like(y, math.inf)
    for i in range(8):
        off = (y - grid[i]).abs() + odd[i]
        best = torch.where(off < near, grid[i], best)
        near = torch.minimum(near, off)
    return (torch.where(torch.signbit(b), -best, best) * torch.pow(2.0, e)).flatten(-2)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "append":
        return tuple(_nearest(s[x].to(F64)) for x in ("k", "v"))
    q = s["q"].to(F64)
    B, Sq, Hq, D = q.shape
    G = Hq // c["kv_heads"]
    out = torch.empty(B, Sq, Hq, D, dtype=F64, device=DEV)
    for b in range(B):
        for h in range(c["kv_heads"]):
            mine = q[b, :, h * G:(h + 1) * G]
            if c["kind"] == "window":
                at = torch.arange(Sq, device=DEV) + c["seq_k"] - Sq
                k, v, m = s["k"][b, :, h].to(F64), s["v"][b, :, h].to(F64), s["mask"]
                got = _row(mine, k, v, at, c, None if m is None else m[b])
            else:
                at = torch.arange(Sq, device=DEV) + int(s["starts"][b])
                k, v = _stored(s["cache"], s["table"][b], h, D, c["page"], int(at[-1]) + 1)
                got = _row(mine, k, v, at, c)
            out[b, :, h * G:(h + 1) * G] = got
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs(first, n, window, sinks):
    """(visible pairs, keys visible to any) of queries at first .. first + n - 1."""
    pairs = 0
    for p in range(first, first + n):
        low = max(0, p - window + 1)
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, first - window + 1)
    return pairs, first + n - low + min(sinks, low)


def work(case):
    c = case
    B, D = c["batch"], c["head_dim"]
    held = 2 * (D // 2 + D // 32)  # bytes of a slot's K and V in one head
    if c["kind"] == "append":
        rows = B * c["seq"] * c["kv_heads"]
        return {"bytes": rows * (4 * D + 2 * held + 4 * D), "flops": rows * 2 * 4 * D}
    last = c["seq_k"] if c["kind"] == "window" else c["slots"]
    pairs, keys = _pairs(last - c["seq_q"], c["seq_q"], c["window"] or last, c["sinks"])
    if c["kind"] == "cache" and c["ragged"]:  # lengths are spread over a quarter to all of the longest
        pairs, keys = pairs * 0.6, keys * 0.6
    rows = B * c["seq_q"] * c["q_heads"]
    per = 4 * D if c["kind"] == "window" else held
    return {"bytes": B * keys * c["kv_heads"] * per + 4 * rows * D, "flops": 4 * D * B * pairs * c["q_heads"]}
