"""Window attention and the 4-bit K/V cache on the GPU against their definitions in 64 bits (stream_ref.attend gives the
bound of every element with the reference)."""

import pytest
import torch

import rldx_amd.ops as ops
from rldx_amd import functional as Fn
from rldx_amd import workloads as W
from stream_ref import attend, nearest, visible

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def rnd(dev, *shape, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed * 1000 + sum(shape))
    return (std * torch.randn(*shape, generator=g)).to(BF16).to(dev)


def check(o, ref, bound, what=""):
    o = o.double()
    assert torch.equal(torch.isnan(o), torch.isnan(ref)), f"{what}: NaN pattern"
    assert torch.equal(torch.isinf(o), torch.isinf(ref)), f"{what}: infinities"
    fin = torch.isfinite(ref)
    off = ((o - ref).abs() / bound)[fin]
    assert off.numel() == 0 or float(off.max()) <= 1.0, f"{what}: {float(off.max()):.3g} of the bound"


def window_ref(q, k, v, window, sinks, mask=None, scale=None):
    B, Sq, Sk = q.shape[0], q.shape[1], k.shape[1]
    at = torch.arange(Sk - Sq, Sk, device=q.device)
    got = []
    for b in range(B):
        vis = visible(at, Sk, window, sinks)
        if mask is not None:
            vis = vis & (mask if mask.dim() == 1 else mask[b if mask.shape[0] > 1 else 0])[None].ne(0)
        got.append(attend(q[b], k[b], v[b], vis, scale))
    return torch.stack([x[0] for x in got]), torch.stack([x[1] for x in got])


# ---------------------------------------------------------------------------
# window attention
# ---------------------------------------------------------------------------
SHAPES = [  # batch, Sq, Sk, Hq, Hkv, D, window, sinks
    (1, 1, 1, 4, 4, 64, 1, 0), (1, 1, 1, 8, 2, 128, 5, 3), (2, 1, 33, 8, 1, 128, 7, 2), (1, 3, 32, 7, 1, 64, 32, 0),
    (1, 2, 2000, 14, 2, 128, 100, 5), (3, 1, 4097, 32, 8, 128, 1024, 4), (2, 4, 700, 4, 4, 64, 1 << 40, 0),
    (1, 5, 5, 4, 2, 128, 1, 0), (1, 31, 31, 4, 2, 64, 8, 1), (1, 33, 33, 2, 2, 128, 33, 0), (2, 65, 65, 28, 4, 128, 17, 40),
    (1, 130, 130, 3, 1, 64, 32, 7), (1, 128, 1000, 8, 8, 128, 300, 33), (1, 257, 257, 4, 1, 128, 1 << 30, 0),
    (1, 300, 301, 6, 6, 64, 64, 1 << 40), (2, 200, 523, 28, 4, 128, 90, 64), (1, 1000, 1000, 4, 1, 128, 256, 4),
    (1, 777, 777, 5, 5, 64, 200, 3), (1, 600, 2000, 8, 2, 64, 1, 2), (5, 40, 40, 1, 1, 128, 6, 0),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_window_attention(dev, shape):
    B, Sq, Sk, Hq, Hkv, D, window, sinks = shape
    q, k, v = rnd(dev, B, Sq, Hq, D), rnd(dev, B, Sk, Hkv, D, seed=1), rnd(dev, B, Sk, Hkv, D, seed=2)
    o = torch.ops.rldx_amd.window_attention(q, k, v, window, sinks)
    check(o, *window_ref(q, k, v, window, sinks))
    assert torch.equal(o, torch.ops.rldx_amd.window_attention(q, k, v, window, sinks)), "two calls, two results"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sq", [1, 70, 190])
def test_window_attention_large_scores_and_scale(dev, D, sq):
    """Scores of hundreds: the softmax reference moves, tiles weigh nothing."""
    q, k, v = rnd(dev, 1, sq, 4, D, std=8), rnd(dev, 1, 320, 2, D, seed=1, std=8), rnd(dev, 1, 320, 2, D, seed=2)
    k[:, 200:] *= 2
    check(Fn.window_attention(q, k, v, 250, 3), *window_ref(q, k, v, 250, 3))
    check(Fn.window_attention(q, k, v, 250, 3, scale=0.013), *window_ref(q, k, v, 250, 3, scale=0.013))


@pytest.mark.parametrize("sq,sk,D", [(1, 100, 128), (100, 100, 64), (150, 400, 128)])
def test_window_attention_strides(dev, sq, sk, D):
    """Packed QKV rows, head-major tensors, one K/V for a batch, an output inside a wider one."""
    Hq, Hkv = 6, 2
    qkv = rnd(dev, 2, sk, (Hq + 2 * Hkv) * D)
    q = qkv[:, sk - sq:, : Hq * D].unflatten(2, (Hq, D))
    k, v = (qkv[:, :, (Hq + i * Hkv) * D: (Hq + (i + 1) * Hkv) * D].unflatten(2, (Hkv, D)) for i in (0, 1))
    ref = window_ref(q, k, v, 60, 2)
    o = Fn.window_attention(q, k, v, 60, 2)
    check(o, *ref, "packed")
    h = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(Fn.window_attention(*h, 60, 2), o)
    wide = torch.full((2, sq, Hq + 3, D + 8), 7.0, dtype=BF16, device=dev)
    Fn.window_attention(q, k, v, 60, 2, out=wide[:, :, 1: Hq + 1, :D])
    assert torch.equal(wide[:, :, 1: Hq + 1, :D], o)
    wide[:, :, 1: Hq + 1, :D] = 7.0
    assert (wide == 7.0).all(), "written beside the output"
    one = [t[:1].expand(2, -1, -1, -1) for t in (k, v)]
    check(Fn.window_attention(q, *one, 60, 2), *window_ref(q, *one, 60, 2), "broadcast")


@pytest.mark.parametrize("sq,sk,D,Hq,Hkv", [(1, 90, 128, 8, 2), (90, 90, 64, 4, 4), (333, 400, 128, 7, 1)])
def test_window_attention_key_mask(dev, sq, sk, D, Hq, Hkv):
    """Padding on the left, holes, a sequence of nothing but padding (rows of zeros), 1-D and shared masks."""
    q, k, v = rnd(dev, 4, sq, Hq, D), rnd(dev, 4, sk, Hkv, D, seed=1), rnd(dev, 4, sk, Hkv, D, seed=2)
    mask = torch.ones(4, sk, device=dev)
    mask[0, : sk // 2 + 5] = 0
    mask[1] = 0
    mask[2] = (torch.rand(sk, generator=torch.Generator().manual_seed(3)) < 0.3).float().to(dev)
    o = torch.ops.rldx_amd.window_attention(q, k, v, 50, 3, mask)
    check(o, *window_ref(q, k, v, 50, 3, mask))
    assert (o[1] == 0).all()
    check(Fn.window_attention(q, k, v, 50, 3, mask[2]), *window_ref(q, k, v, 50, 3, mask[2]), "1-D")
    check(Fn.window_attention(q, k, v, 50, 3, mask[2:3]), *window_ref(q, k, v, 50, 3, mask[2:3]), "shared")
    big = torch.where(mask == 0, 0.0, torch.finfo(torch.float32).min)  # any value but zero is visible
    assert torch.equal(Fn.window_attention(q, k, v, 50, 3, big), o)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", [(1, 300, 2500, 28, 4), (2, 49, 6000, 28, 4), (1, 500, 2049, 16, 16), (1, 41, 9000, 64, 2)], ids=str)
def test_window_attention_long_chunks(dev, case, D):
    """Chunks behind long pasts, with values that only some queries may see and a key mask."""
    B, sq, sk, Hq, Hkv = case
    q, k, v = rnd(dev, B, sq, Hq, D), rnd(dev, B, sk, Hkv, D, seed=1), rnd(dev, B, sk, Hkv, D, seed=2)
    check(Fn.window_attention(q, k, v, 1 << 30), *window_ref(q, k, v, 1 << 30, 0), "whole")
    mask = (torch.rand(B, sk, generator=torch.Generator().manual_seed(5)) < 0.9).float().to(dev)
    mask[-1, :800] = 0
    k[mask == 0], v[mask == 0] = float("nan"), float("inf")
    check(Fn.window_attention(q, k, v, 1700, 40, mask), *window_ref(q, k, v, 1700, 40, mask), "mask")
    v[:, sk - 3, 0, 5], v[:, sk - sq // 2, Hkv - 1, D - 1] = float("inf"), float("nan")
    check(Fn.window_attention(q, k, v, 1700, 40, mask), *window_ref(q, k, v, 1700, 40, mask), "infinite")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sq,window,sinks", [(1100, 1 << 30, 0), (300, 1 << 30, 0), (1100, 150, 40), (17, 600, 1)])
def test_window_attention_long_padding(dev, sq, window, sinks, D):
    """Masked keys of many tiles before, behind and between the others."""
    sk = 1100
    q, k, v = rnd(dev, 6, sq, 4, D), rnd(dev, 6, sk, 2, D, seed=1), rnd(dev, 6, sk, 2, D, seed=2)
    mask = torch.zeros(6, sk, device=dev)
    mask[0, 700:] = mask[1, :310] = mask[2, 1033] = mask[3, 0] = mask[4, 32:64] = mask[4, 600:608] = mask[4, 1099] = 1
    k[mask == 0] = float("nan")
    v[mask == 0] = float("inf")
    check(Fn.window_attention(q, k, v, window, sinks, mask), *window_ref(q, k, v, window, sinks, mask))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("sq,sk,D,G", [(1, 200, 128, 4), (3, 200, 64, 2), (64, 64, 64, 1), (150, 333, 128, 2)])
def test_window_attention_hidden_keys_may_hold_anything(dev, bad, sq, sk, D, G):
    """Masked keys, and keys outside the window of every query: the bits of zeros there."""
    q, k, v = rnd(dev, 1, sq, 2 * G, D), rnd(dev, 1, sk, 2, D, seed=1), rnd(dev, 1, sk, 2, D, seed=2)
    mask = torch.ones(sk, device=dev)
    mask[sk - 20: sk - 9] = 0
    vis = visible(torch.arange(sk - sq, sk, device=dev), sk, 30, 2).any(0) & mask.bool()
    k[:, ~vis], v[:, ~vis] = 0, 0
    o = Fn.window_attention(q, k, v, 30, 2, mask)
    k[:, ~vis], v[:, ~vis] = bad, bad
    assert torch.equal(Fn.window_attention(q, k, v, 30, 2, mask), o)
    check(o, *window_ref(q, k, v, 30, 2, mask))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("sq,D", [(3, 128), (40, 64), (200, 128), (200, 64)])
def test_window_attention_values_that_only_some_queries_see(dev, bad, sq, D):
    """An infinity or a NaN in V (single dimensions) and in K reaches the queries that see it, and no other."""
    q, k, v = rnd(dev, 1, sq, 4, D), rnd(dev, 1, sq + 30, 2, D, seed=1), rnd(dev, 1, sq + 30, 2, D, seed=2)
    for at, d in ((0, 3), (7, 0), (29, D - 1), (30 + sq // 2, 17), (sq + 29, 33)):
        v[:, at, 0, d] = bad
    ref, bound = window_ref(q, k, v, 12, 1)
    assert torch.isfinite(ref).any() and not torch.isfinite(ref).all()
    check(Fn.window_attention(q, k, v, 12, 1), ref, bound)
    v = rnd(dev, 1, sq + 30, 2, D, seed=2)
    k[:, 30 + sq // 2, 1, 5] = float("nan")
    ref, bound = window_ref(q, k, v, 12, 1)
    check(Fn.window_attention(q, k, v, 12, 1), ref, bound)


@pytest.mark.parametrize("sq,D", [(3, 128), (40, 64), (200, 128)])
def test_window_attention_largest_finite_values(dev, sq, D):
    """Values next to the infinities are values."""
    q, k, v = rnd(dev, 1, sq, 4, D), rnd(dev, 1, sq + 30, 2, D, seed=1), rnd(dev, 1, sq + 30, 2, D, seed=2)
    v[:, 5, 0, 3], v[:, 29, 1, D - 1], v[:, 30 + sq // 2, 0, 17] = 2.0 ** 121, -(2.0 ** 127), torch.finfo(torch.bfloat16).max
    check(Fn.window_attention(q, k, v, 12, 1), *window_ref(q, k, v, 12, 1))


def test_window_attention_offsets_past_32_bits(dev):
    """Rows 64 KiB apart: the last keys lie 4.5 GB behind the first."""
    n, row = 70000, 32768
    buf = torch.empty(n * row, dtype=BF16, device=dev)
    kv = buf.view(n, row)
    kv[:, :512] = rnd(dev, n, 512, std=0.5)
    k, v = kv[None, :, :256].unflatten(2, (2, 128)), kv[None, :, 256:512].unflatten(2, (2, 128))
    for sq in (1, 80):
        q = rnd(dev, 1, sq, 4, 128, seed=5)
        o = Fn.window_attention(q, k, v, 500, 8)
        keep = torch.cat([torch.arange(8), torch.arange(n - sq - 500, n)]).to(dev)
        vis = visible(torch.arange(n - sq, n, device=dev), n, 500, 8)[:, keep]
        check(o[0], *attend(q[0], k[0, keep], v[0, keep], vis), f"Sq {sq}")


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
def cache_of(dev, B, slots, H, D, page, seed=0, spare=2):
    """Pages of random bytes, and a table of them in any order."""
    g = torch.Generator().manual_seed(seed)
    per = -(-slots // page)
    c = Fn.kv4_cache(B * per + spare, H, D, page_tokens=page, device=dev)
    c.copy_(torch.randint(0, 256, c.shape, generator=g, dtype=torch.uint8))
    table = torch.randperm(B * per + spare, generator=g)[: B * per].to(torch.int32).view(B, per).to(dev)
    return c, table


def ints(dev, *v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("B,S,H,D,page", [(1, 1, 1, 64, 32), (1, 1, 8, 128, 64), (3, 37, 2, 128, 32), (2, 65, 5, 64, 128),
                                          (1, 300, 3, 128, 256), (4, 33, 1, 64, 32)])
def test_append_and_read(dev, B, S, H, D, page):
    """Values equal to the format's, at unaligned starts and with ragged counts; every other byte left as it was."""
    c, table = cache_of(dev, B, S + 70, H, D, page)
    k, v = rnd(dev, B, S, H, D, seed=1, std=3), rnd(dev, B, S, H, D, seed=2)
    k[..., :32] *= 1e-3
    starts = ints(dev, *[(7 * b) % 70 for b in range(B)])
    counts = ints(dev, *[S - b * S // (B + 1) for b in range(B)])
    total = table.shape[1] * page
    before = c.clone()
    ok, ov = torch.ops.rldx_amd.kv4_read(c, table, ints(dev, *[0] * B), total, D)
    version = c._version
    torch.ops.rldx_amd.kv4_append(c, k, v, table, starts, counts)
    assert c._version > version
    rk, rv = torch.ops.rldx_amd.kv4_read(c, table, ints(dev, *[0] * B), total, D)
    for b in range(B):
        s, n = int(starts[b]), int(counts[b])
        for got, old, src in ((rk, ok, k), (rv, ov, v)):
            assert torch.equal(got[b, s: s + n].double(), nearest(src[b, :n])), f"sequence {b}"
            out = torch.ones(total, dtype=torch.bool, device=dev)
            out[s: s + n] = False
            assert torch.equal(got[b, out].view(torch.int16), old[b, out].view(torch.int16)), "other slots changed"
    spare = torch.ones(c.shape[0], dtype=torch.bool, device=dev)
    spare[table.flatten().long()] = False
    assert torch.equal(c[spare], before[spare]), "pages of nobody changed"
    # all rows (no counts) in pieces give the same bytes as at once
    one, two = before.clone(), before.clone()
    Fn.kv4_append(one, k, v, table, starts)
    for i in range(0, S, 5):
        Fn.kv4_append(two, k[:, i: i + 5], v[:, i: i + 5], table, starts + i)
    assert torch.equal(one, two)


@pytest.mark.parametrize("D", [64, 128])
def test_append_special_values(dev, D):
    """Zeros, subnormals, the largest values, infinities and NaN, each in a block of its own."""
    c, table = cache_of(dev, 1, 64, 2, D, 64)
    k = rnd(dev, 1, 9, 2, D)
    k[0, 0] = 0
    k[0, 1] = -0.0
    k[0, 2] = 1e-40
    k[0, 3, :, 5] = 3.3e38
    k[0, 4, 0, 40] = float("inf")
    k[0, 5, 1, 3] = float("nan")
    k[0, 6, 0, :32] = float("-inf")
    k[0, 7] = torch.finfo(BF16).max
    v = k.flip(1)
    Fn.kv4_append(c, k, v, table, ints(dev, 11))
    rk, rv = Fn.kv4_read(c, table, ints(dev, 11), 9, D)
    for got, src in ((rk, k), (rv, v)):
        want = nearest(src)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        g, w = torch.nan_to_num(got.double()), torch.nan_to_num(want)
        assert torch.equal(g, w) and torch.equal(torch.signbit(g), torch.signbit(w))


def test_append_every_bf16_value(dev):
    """All 65536 values, in blocks whose largest magnitude runs over mantissas and exponents, and in blocks of their
    own, against the format in 64 bits, which the CPU tests hold the format's definition to."""
    every = torch.arange(65536, dtype=torch.int32)
    parts = [every[:, None].expand(-1, 32)]
    for top in (0x3F80, 0x3FDF, 0x3FE0, 0x3FE1, 0x3FFF, 0x0001, 0x007F, 0x0080, 0x0100, 0x7F00, 0x7F60, 0x7F7F, 0x4123):
        rows = torch.cat([every, every[: 2115 * 31 - 65536]]).view(2115, 31)
        parts.append(torch.cat([torch.full((2115, 1), top, dtype=torch.int32), rows], 1))
    x = torch.cat(parts)
    x = torch.cat([x, x[: -x.shape[0] % 8]]).to(torch.int16).view(BF16).view(1, -1, 2, 128).to(dev)
    S = x.shape[1]
    c, table = cache_of(dev, 1, S, 2, 128, 256)
    Fn.kv4_append(c, x, x.flip(1), table, ints(dev, 0))
    rk, rv = Fn.kv4_read(c, table, ints(dev, 0), S, 128)
    want = nearest(x)
    for got, w in ((rk, want), (rv, want.flip(1))):
        assert torch.equal(torch.isnan(got), torch.isnan(w))
        g, w = torch.nan_to_num(got.double()), torch.nan_to_num(w)
        assert torch.equal(g, w) and torch.equal(torch.signbit(g), torch.signbit(w))


def test_append_and_read_skip_what_is_not_there(dev):
    """Slots below 0, past the table and of pages outside the cache are not written, and read as NaN."""
    c, table = cache_of(dev, 3, 128, 2, 128, 32)
    table[1, 1], table[2, 0] = c.shape[0], -1
    k, v = rnd(dev, 3, 50, 2, 128), rnd(dev, 3, 50, 2, 128, seed=1)
    starts = ints(dev, -20, 10, 100)
    before = c.clone()
    Fn.kv4_append(c, k, v, table, starts)
    rk, rv = Fn.kv4_read(c, table, starts, 50, 128)
    for got, src in ((rk, k), (rv, v)):
        want = nearest(src)
        want[0, :20] = torch.nan  # below 0
        want[1, 22:] = torch.nan  # slots 32 .. 59: the page is missing
        want[2, 28:] = torch.nan  # past the table's 128 slots
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.double()), torch.nan_to_num(want))
    used = torch.zeros(c.shape[0], dtype=torch.bool, device=dev)
    used[[int(table[0, 0]), int(table[1, 0]), int(table[2, 3])]] = True
    assert torch.equal(c[~used], before[~used])


def kv4_ref(q, c, table, starts, counts=None, window=None, sinks=0, scale=None):
    """The reference on the values that the cache holds."""
    B, Sq, D = q.shape[0], q.shape[1], q.shape[3]
    page = c.shape[2] // (34 * D) * 32
    n = table.shape[1] * page
    k, v = Fn.kv4_read(c, table, torch.zeros_like(starts), n, D)
    got = []
    for b in range(B):
        i = torch.arange(Sq, device=q.device)
        at = i + int(starts[b])
        vis = visible(at, n, 1 << 30 if window is None else window, sinks)
        if counts is not None:
            vis = vis & (i < int(counts[b]))[:, None]
        got.append(attend(q[b], k[b], v[b], vis, scale))
    return torch.stack([x[0] for x in got]), torch.stack([x[1] for x in got])


def filled(dev, B, slots, H, D, page, upto, seed=0):
    """A cache whose sequences hold upto[b] slots; the others hold random bytes."""
    c, table = cache_of(dev, B, slots, H, D, page, seed)
    k, v = rnd(dev, B, slots, H, D, seed=seed + 1), rnd(dev, B, slots, H, D, seed=seed + 2)
    Fn.kv4_append(c, k, v, table, ints(dev, *[0] * B), ints(dev, *upto))
    return c, table


CACHES = [  # batch, Sq, Hq, Hkv, D, page, slots, window, sinks, starts
    (1, 1, 4, 4, 64, 32, 1, None, 0, (0,)), (1, 1, 8, 2, 128, 64, 40, None, 0, (39,)),
    (3, 1, 8, 1, 128, 32, 97, None, 0, (0, 31, 96)), (2, 1, 28, 4, 128, 128, 3000, None, 0, (2999, 31)),
    (4, 1, 24, 8, 64, 32, 5000, 300, 16, (4999, 4000, 310, 5)), (2, 3, 8, 2, 64, 64, 200, 40, 3, (197, 60)),
    (1, 16, 2, 2, 128, 64, 500, None, 0, (480,)), (2, 9, 14, 2, 128, 32, 700, 100, 33, (0, 650)),
    (1, 64, 8, 8, 64, 256, 64, None, 0, (0,)), (1, 49, 28, 4, 128, 64, 1000, 200, 4, (900,)),
    (2, 100, 4, 1, 64, 64, 4000, None, 0, (3900, 17)), (1, 1, 32, 8, 128, 64, 40000, None, 0, (39998,)),
    (1, 2, 64, 1, 128, 64, 600, 1, 0, (598,)), (1, 1, 17, 1, 64, 32, 300, 64, 500, (299,)),
]


@pytest.mark.parametrize("case", CACHES, ids=str)
def test_kv4_attention(dev, case):
    B, Sq, Hq, Hkv, D, page, slots, window, sinks, starts = case
    c, table = filled(dev, B, slots, Hkv, D, page, [s + Sq for s in starts])
    q, st = rnd(dev, B, Sq, Hq, D, seed=7), ints(dev, *starts)
    o = torch.ops.rldx_amd.kv4_attention(q, c, table, st, None, window, sinks)
    check(o, *kv4_ref(q, c, table, st, None, window, sinks))
    assert torch.equal(o, torch.ops.rldx_amd.kv4_attention(q, c, table, st, None, window, sinks)), "two calls, two results"
    check(Fn.kv4_attention(q, c, table, st, None, window, sinks, 0.3), *kv4_ref(q, c, table, st, None, window, sinks, 0.3))


@pytest.mark.parametrize("Sq,Hq,Hkv,D", [(6, 4, 2, 128), (40, 8, 2, 64), (3, 8, 8, 128)])
def test_kv4_attention_counts_and_negative_starts(dev, Sq, Hq, Hkv, D):
    """Rows past a sequence's count, and below slot 0, are zeros; an empty sequence has nothing but those."""
    starts, counts = ints(dev, 50, -2, 0, 20, 7), ints(dev, Sq, Sq, 0, 1, Sq - 1)
    c, table = filled(dev, 5, 128, Hkv, D, 32, [50 + Sq, Sq - 2, 0, 21, 6 + Sq])
    q = rnd(dev, 5, Sq, Hq, D)
    o = Fn.kv4_attention(q, c, table, starts, counts)
    check(o, *kv4_ref(q, c, table, starts, counts))
    assert (o[1, :2] == 0).all() and (o[2] == 0).all() and (o[3, 1:] == 0).all() and (o[4, -1] == 0).all()
    check(Fn.kv4_attention(q, c, table, starts, counts, 9, 2), *kv4_ref(q, c, table, starts, counts, 9, 2))


@pytest.mark.parametrize("Sq", [1, 30])
def test_kv4_attention_pages(dev, Sq):
    """Pages that no query sees may be missing; a query that sees a missing one, or stands past the table, gets NaN."""
    c, table = filled(dev, 2, 640, 2, 128, 64, [640, 640])
    q, st = rnd(dev, 2, Sq, 8, 128), ints(dev, 600 - Sq, 600 - Sq)
    want = Fn.kv4_attention(q, c, table, st, None, 90, 5)
    holes = table.clone()
    holes[:, 1:7] = torch.tensor([-1, 1 << 30, -(1 << 31), c.shape[0], 9999, -7], dtype=torch.int32, device=dev)
    assert torch.equal(Fn.kv4_attention(q, c, holes, st, None, 90, 5), want)
    holes[1, 9] = c.shape[0]
    o = Fn.kv4_attention(q, c, holes, st, None, 90, 5)
    assert torch.equal(o[0], want[0])
    i = torch.arange(Sq, device=dev) + 600 - Sq
    assert torch.equal(torch.isnan(o[1]).all(-1).all(-1), i >= 576) and torch.equal(o[1][i < 576], want[1][i < 576])
    o = Fn.kv4_attention(q, c, holes, st)
    assert torch.isnan(o).all()
    o = Fn.kv4_attention(q, c, table, ints(dev, 640 - Sq // 2 - 1, 2000000000), None, 90)
    past = torch.arange(Sq, device=dev) + 640 - Sq // 2 - 1 >= 640
    assert torch.equal(torch.isnan(o[0]).all(-1).all(-1), past) and torch.isnan(o[1]).all()
    assert not torch.isnan(o[0][~past]).any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 5, 40])
def test_kv4_attention_nan_blocks(dev, D, Sq):
    """A NaN in K reaches the queries that see it, one in V the 32 dimensions of its block, and nothing else."""
    n = 200
    for which in (0, 1):
        k, v = rnd(dev, 1, n, 2, D, seed=1), rnd(dev, 1, n, 2, D, seed=2)
        for at, h, d in ((n - Sq, 0, 3), (n - Sq - 25, 1, 40), (n - 1, 1, D - 1), (2, 0, 9), (100, 0, 0)):
            (k, v)[which][0, at, h, d] = float("inf")
        c, table = cache_of(dev, 1, n, 2, D, 64)
        Fn.kv4_append(c, k, v, table, ints(dev, 0))
        q, st = rnd(dev, 1, Sq, 6, D), ints(dev, n - Sq)
        for window, sinks in ((30, 2), (30, 3), (None, 0)):
            ref, bound = kv4_ref(q, c, table, st, None, window, sinks)
            check(Fn.kv4_attention(q, c, table, st, None, window, sinks), ref, bound, f"{which} {window} {sinks}")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", [  # batch, Sq, Hq, Hkv, slots, starts: one or two of each cut of the work
    (2, 1, 32, 8, 250, (249, 100)), (16, 1, 24, 8, 1300, tuple(range(1299, 3, -81))), (1, 49, 28, 4, 6000, (5940,)),
    (2, 49, 28, 4, 6000, (5951, 333)), (1, 70, 32, 8, 9000, (8900,)), (8, 300, 24, 24, 331, (31, 0, 30, 17, 1, 12, 29, 5))],
    ids=str)
def test_kv4_attention_long_chunks(dev, case, D):
    """Chunks over long caches with NaN blocks in K and V, hidden from some queries by the order and the window, rows
    past a sequence's count and a page that is missing."""
    B, Sq, Hq, Hkv, slots, starts = case
    k, v = rnd(dev, B, slots, Hkv, D, seed=1), rnd(dev, B, slots, Hkv, D, seed=2)
    for b, st in enumerate(starts):
        v[b, st + Sq - 1, Hkv - 1, D - 1] = v[b, max(st - 4, 0), 0, 3] = float("nan")
        v[b, st + Sq // 2, b % Hkv, 40] = k[b, st + Sq - 1, 1, 0] = float("inf")
        v[b, st // 3, 2, 0] = k[b, st // 2, 3, 9] = -float("inf")
    c, table = cache_of(dev, B, slots, Hkv, D, 64)
    Fn.kv4_append(c, k, v, table, ints(dev, *[0] * B))
    q, st = rnd(dev, B, Sq, Hq, D, seed=3), ints(dev, *starts)
    counts = ints(dev, *[Sq - (b % 3 == 1) for b in range(B)])
    for window, sinks in ((None, 0), (70, 33)):
        check(Fn.kv4_attention(q, c, table, st, counts, window, sinks),
              *kv4_ref(q, c, table, st, counts, window, sinks), f"{window} {sinks}")
    if starts[0] >= 250:
        want = Fn.kv4_attention(q, c, table, st, counts, 70, 33)
        table[0, 1] = -1
        assert torch.equal(torch.nan_to_num(Fn.kv4_attention(q, c, table, st, counts, 70, 33)), torch.nan_to_num(want))
        assert torch.isnan(Fn.kv4_attention(q, c, table, st, counts)[0, 0]).all()


def test_kv4_offsets_past_32_bits(dev):
    """Pages more than 2^32 bytes behind the first one."""
    H, D, page = 8, 128, 64
    c = Fn.kv4_cache((1 << 32) // (H * 2 * 34 * D) + 50, H, D, page_tokens=page, device=dev)
    table = ints(dev, *range(c.shape[0] - 1, c.shape[0] - 31, -1))[None]
    k, v = rnd(dev, 1, 1900, H, D), rnd(dev, 1, 1900, H, D, seed=1)
    Fn.kv4_append(c, k, v, table, ints(dev, 0))
    rk, rv = Fn.kv4_read(c, table, ints(dev, 0), 1900, D)
    assert torch.equal(rk.double(), nearest(k)) and torch.equal(rv.double(), nearest(v))
    for Sq in (1, 20):
        q, st = rnd(dev, 1, Sq, 16, D), ints(dev, 1900 - Sq)
        check(Fn.kv4_attention(q, c, table, st), *kv4_ref(q, c, table, st))


def test_kv4_strided_cache_and_rows(dev):
    """Pages inside a larger buffer (two layers' side by side, heads of one of them), rows of packed QKV."""
    D, H = 128, 2
    n = Fn.kv4_cache(1, 1, D, device=dev).shape[2]
    big = torch.zeros(6, 2, H + 1, n, dtype=torch.uint8, device=dev)
    c = big[:, 1, :H]
    table, st = ints(dev, 4, 1, 3)[None], ints(dev, 0)
    qkv = rnd(dev, 1, 150, (4 + 2 * H) * D)
    q, k, v = (t.unflatten(2, (-1, D)) for t in qkv.split([4 * D, H * D, H * D], 2))
    torch.ops.rldx_amd.kv4_append(c, k, v, table, st)
    assert not big[:, 0].any() and not big[:, 1, H:].any()
    rk, _ = torch.ops.rldx_amd.kv4_read(c, table, st, 150, D)
    assert torch.equal(rk.double(), nearest(k))
    o = torch.ops.rldx_amd.kv4_attention(q, c, table, st)
    check(o, *kv4_ref(q, c, table, st))
    assert torch.equal(o, Fn.kv4_attention(q.contiguous(), c.contiguous(), table, st))


# ---------------------------------------------------------------------------
# how they are called
# ---------------------------------------------------------------------------
def test_nothing_to_do(dev):
    q = torch.empty(0, 3, 4, 64, dtype=BF16, device=dev)
    k = torch.empty(0, 5, 2, 64, dtype=BF16, device=dev)
    assert torch.ops.rldx_amd.window_attention(q, k, k, 4).shape == q.shape
    q, k = torch.empty(2, 0, 4, 64, dtype=BF16, device=dev), rnd(dev, 2, 5, 2, 64)
    assert torch.ops.rldx_amd.window_attention(q, k, k, 4).shape == q.shape
    c, table = cache_of(dev, 2, 64, 2, 64, 32)
    st = ints(dev, 0, 0)
    before = c.clone()
    torch.ops.rldx_amd.kv4_append(c, k[:, :0], k[:, :0], table, st)
    assert torch.equal(c, before)
    assert torch.ops.rldx_amd.kv4_read(c, table, st, 0, 64)[0].shape == (2, 0, 2, 64)
    assert torch.ops.rldx_amd.kv4_attention(q, c, table, st).shape == q.shape
    # a table without pages: every slot is missing
    none = table[:, :0]
    assert torch.isnan(torch.ops.rldx_amd.kv4_attention(rnd(dev, 2, 1, 4, 64), c, none, st)).all()
    assert torch.isnan(torch.ops.rldx_amd.kv4_read(c, none, st, 1, 64)[0]).all()


def test_refusals(dev):
    q, k = rnd(dev, 1, 4, 4, 64), rnd(dev, 1, 9, 2, 64)
    wa = torch.ops.rldx_amd.window_attention
    for args, msg in (((q.half(), k, k, 4), "bf16"), ((q, k, k, 0), "window"), ((q, k, k, 4, -1), "sinks"),
                      ((k, q[:, :, :2], q[:, :, :2], 4), "Sq <= Sk"), ((q[:, :, :3], k, k, 4), "multiple of kv heads"),
                      ((q, k, k[:, :8], 4), "matching q"), ((q, k.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), 4), "matching q"),
                      ((q, k, k, 4, 0, torch.ones(1, 8, device=dev)), "key_mask"),
                      ((q, k, k, 4, 0, torch.ones(9, device=dev, dtype=torch.bool)), "key_mask"),
                      ((q, k, k, 4, 0, None, 0.0), "scale"), ((q, k, k, 4, 0, None, float("nan")), "scale"),
                      ((q.transpose(2, 3), k, k, 4), "head_dim"), ((q[..., :32], k[..., :32], k[..., :32], 4), "head_dim"),
                      ((rnd(dev, 1, 4, 4, 68)[..., 4:], k, k, 4), "aligned"), ((q, k.cpu(), k, 4), "ROCm device")):
        with pytest.raises(RuntimeError, match=msg):
            wa(*args)
    with pytest.raises(RuntimeError, match="overlapping"):
        Fn.window_attention(q, k, k, 4, out=q[:, :1].expand(-1, 4, -1, -1))
    c, table = cache_of(dev, 1, 64, 2, 64, 32)
    st = ints(dev, 0)
    at, ap = torch.ops.rldx_amd.kv4_attention, torch.ops.rldx_amd.kv4_append
    for args, msg in (((q, c, table, st.long()), "starts"), ((q, c, table.long(), st), "page_table"),
                      ((q, c, table, ints(dev, 0, 0)), "starts"), ((q, c, table, st, ints(dev, 1, 1)), "counts"),
                      ((rnd(dev, 1, 4, 4, 128), c, table, st), "head_dim 128"), ((q[:, :, :3], c, table, st), "multiple"),
                      ((q, c.view(torch.int8), table, st), "uint8"), ((q, c, table, st, None, 0), "window"),
                      ((q, c, table, st, None, 3, -2), "sinks"), ((q, c, table, st, None, 3, 0, -1.0), "scale"),
                      ((q, c[:1].expand(5, -1, -1), table, st), "apart")):
        with pytest.raises(RuntimeError, match=msg):
            at(*args)
    before = c.clone()
    for args, msg in (((c, k, k[:, :4], table, st), "one shape"), ((c, q, q, table, st), "kv heads"),
                      ((c, k, k, table.expand(2, -1), st), "page_table"), ((c[..., 1:], k, k, table, st), "bytes")):
        with pytest.raises(RuntimeError, match=msg):
            ap(*args)
    assert torch.equal(c, before)
    with pytest.raises(RuntimeError, match="count"):
        torch.ops.rldx_amd.kv4_read(c, table, st, -1, 64)


def test_no_backward(dev):
    """As the framework's other operators: inference only."""
    q, k = rnd(dev, 1, 4, 4, 64).requires_grad_(), rnd(dev, 1, 9, 2, 64)
    o = torch.ops.rldx_amd.window_attention(q, k, k, 4)
    with pytest.raises(RuntimeError):
        o.sum().backward()


def test_native_calls_match_python(dev):
    q, k, v = rnd(dev, 2, 40, 8, 128), rnd(dev, 2, 90, 2, 128, seed=1), rnd(dev, 2, 90, 2, 128, seed=2)
    mask = (torch.arange(90, device=dev) >= 11).float()
    o = torch.ops.rldx_amd.window_attention(q, k, v, 20, 3, mask[None], 0.1)
    assert torch.equal(o, ops.window_attention_op._init_fn(q, k, v, 20, 3, mask[None], 0.1))
    c, table = cache_of(dev, 2, 200, 2, 128, 32)
    st, ct = ints(dev, 3, 50), ints(dev, 90, 80)
    one, two = c.clone(), c.clone()
    torch.ops.rldx_amd.kv4_append(one, k, v, table, st, ct)
    ops.kv4_append_op._init_fn(two, k, v, table, st, ct)
    assert torch.equal(one, two)
    for a, b in zip(torch.ops.rldx_amd.kv4_read(one, table, st, 60, 128), ops.kv4_read_op._init_fn(one, table, st, 60, 128)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    a = torch.ops.rldx_amd.kv4_attention(q, one, table, st, ct, 33, 2, 0.2)
    # (the first slots are random bytes, which may stand for NaN: bits are compared)
    assert torch.equal(a.view(torch.int16), ops.kv4_attention_op._init_fn(q, one, table, st, ct, 33, 2, 0.2).view(torch.int16))
    with torch.inference_mode():
        o = torch.ops.rldx_amd.kv4_attention(q, one, table, st, ct, 33, 2, 0.2)
        assert torch.equal(o.view(torch.int16), a.view(torch.int16))
        three = c.clone()
        torch.ops.rldx_amd.kv4_append(three, k, v, table, st, ct)
        assert torch.equal(three, one)


def test_register_fake_matches_real_op(dev):
    q, k = rnd(dev, 1, 4, 4, 64), rnd(dev, 1, 9, 2, 64)
    c, table = cache_of(dev, 1, 64, 2, 64, 32)
    st = ints(dev, 2)
    for op, args in ((torch.ops.rldx_amd.window_attention, (q, k, k, 4, 1, torch.ones(9, device=dev))),
                     (torch.ops.rldx_amd.kv4_append, (c, k, k, table, st)), (torch.ops.rldx_amd.kv4_read, (c, table, st, 3, 64)),
                     (torch.ops.rldx_amd.kv4_attention, (q, c, table, st, None, 5, 1, 0.2))):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


def _stream_step(c, table, starts, q, k, v):
    torch.ops.rldx_amd.kv4_append(c, k, v, table, starts)
    return torch.ops.rldx_amd.kv4_attention(q, c, table, starts, None, 2000, 4)


def test_refused_token_strides(dev):
    wide = torch.empty((1 << 24) + 8 + 64, dtype=torch.bfloat16, device=dev).as_strided((1, 2, 1, 64), (0, (1 << 24) + 8, 64, 1))
    q, k = rnd(dev, 1, 2, 1, 64), rnd(dev, 1, 2, 1, 64)
    for args in ((q, wide, k, 4), (q, k, wide, 4)):
        with pytest.raises(RuntimeError, match="from token to token"):
            torch.ops.rldx_amd.window_attention(*args)


def test_tensors_off_the_current_device(dev, monkeypatch):
    """The launchers make the tensors' device the current one where it is not."""
    q, k = rnd(dev, 1, 4, 4, 64), rnd(dev, 1, 40, 2, 64)
    c, table = cache_of(dev, 1, 64, 2, 64, 32)
    st = ints(dev, 3)

    def calls():
        Fn.kv4_append(c, k, k, table, ints(dev, 0))
        return (Fn.window_attention(q, k, k, 9), *Fn.kv4_read(c, table, st, 30, 64), Fn.kv4_attention(q, c, table, st))

    class Entered(torch.cuda.device):
        at = []

        def __enter__(self):
            self.at.append(self.idx)
            return super().__enter__()

    want = calls()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "device", Entered)
    got = calls()
    monkeypatch.undo()
    assert Entered.at == [0] * 4 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once(dev):
    """Calls on two streams, nothing waiting between them: each has a workspace of its own."""
    sets = []
    for i in range(2):
        c, table = filled(dev, 2, 4000, 2, 128, 64, [3000, 1000], seed=i)
        sets.append((c, table, ints(dev, 3000, 1000), *(rnd(dev, 2, 1, h, 128, seed=9 + i) for h in (8, 2, 2))))
    want = [_stream_step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_stream_step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


def test_captured_steps_follow_their_inputs(dev):
    """One captured step (append + attention), replayed while the slots, the rows and the page table change; two graphs
    that share a memory pool; eager calls between the replays."""
    c, table = filled(dev, 2, 3000, 2, 128, 64, [2500, 60])
    eager = c.clone()
    starts = ints(dev, 2500, 60)
    q, k, v = (rnd(dev, 2, 1, h, 128, seed=4) for h in (8, 2, 2))
    x = rnd(dev, 1, 300, 4, 64)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # warm up outside the capture
        _stream_step(eager.clone(), table, starts, q, k, v)
        torch.ops.rldx_amd.window_attention(x, x, x, 40, 2)
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with Fn.record_graph(one):
        o1 = _stream_step(c, table, starts, q, k, v)
    with Fn.hold_gc(), torch.cuda.graph(two, pool=one.pool()):
        o2 = torch.ops.rldx_amd.window_attention(x, x, x, 40, 2)
    now = starts.clone()
    for step in range(4):
        for t, s in ((q, 1), (k, 2), (v, 3)):
            t.copy_(rnd(dev, *t.shape, seed=20 + 4 * step + s))
        starts.copy_(now)
        if step == 2:  # the first sequence's first pages change places, their bytes too
            table[0, [0, 1]] = table[0, [1, 0]]
            a, b = int(table[0, 0]), int(table[0, 1])
            for cc in (c, eager):
                cc[[a, b]] = cc[[b, a]]
        x.copy_(rnd(dev, *x.shape, seed=50 + step))
        one.replay()
        got = o1.clone()
        two.replay()
        assert torch.equal(got, _stream_step(eager, table, starts, q, k, v)), f"step {step}"
        assert torch.equal(o2, torch.ops.rldx_amd.window_attention(x, x, x, 40, 2)), f"step {step}"
        torch.cuda.synchronize()
        now = now + 1
    assert torch.equal(c, eager)


def test_a_stream_from_prompt_to_tokens(dev):
    """As they are used together: norm and rotation, window attention over a prompt of two sequences, its rows into the
    cache, a chunk, then single tokens over the cache with the same window and sinks."""
    B, Hq, Hkv, D, window, sinks, prompt, chunk, tokens = 2, 8, 2, 128, 70, 4, 150, 20, 5
    total = prompt + chunk + tokens
    cos, sin = W.qwen_rope_cos_sin(total, D, 1e6, BF16)
    cos, sin, w = cos.to(dev), sin.to(dev), (1 + 0.1 * rnd(dev, D)).to(BF16)
    xq, xk, v = rnd(dev, B, total, Hq, D), rnd(dev, B, total, Hkv, D, seed=1), rnd(dev, B, total, Hkv, D, seed=2)
    q, k = Fn.qk_rmsnorm_rope_half(xq, xk, w, w, cos, sin)
    o = torch.ops.rldx_amd.window_attention(q[:, :prompt], k[:, :prompt], v[:, :prompt], window, sinks)
    check(o, *window_ref(q[:, :prompt], k[:, :prompt], v[:, :prompt], window, sinks), "prompt")
    c, table = cache_of(dev, B, total, Hkv, D, 32)
    at = ints(dev, 0, 0)
    torch.ops.rldx_amd.kv4_append(c, k[:, :prompt], v[:, :prompt], table, at)
    at = at + prompt
    for n in [chunk] + [1] * tokens:
        s = int(at[0])
        torch.ops.rldx_amd.kv4_append(c, k[:, s: s + n], v[:, s: s + n], table, at)
        o = torch.ops.rldx_amd.kv4_attention(q[:, s: s + n], c, table, at, None, window, sinks)
        check(o, *kv4_ref(q[:, s: s + n], c, table, at, None, window, sinks), f"slots {s} ..")
        kq, vq = nearest(k[:, : s + n]).to(BF16), nearest(v[:, : s + n]).to(BF16)
        check(o, *window_ref(q[:, s: s + n], kq, vq, window, sinks), f"window attention on the held values, {s} ..")
        at = at + n
