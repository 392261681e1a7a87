"""CPU tests of the window attention and the 4-bit K/V cache: the format on all kinds of values, what the C ABI and the
Python launchers refuse before any GPU work, and the shapes that the operators' fakes report."""

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import rldx_amd.ops  # noqa: F401
from rldx_amd import _lib
from rldx_amd import functional as Fn
from stream_ref import GRID, nearest

INVALID = 1
BF16 = torch.bfloat16
P = 4096  # stand-in device address, 16-byte aligned: every call below must end in validation


def _encode(x):
    """[n, 32] bf16 -> float64 values by the append kernel's element functions, run on the CPU."""
    x = x.contiguous()
    codes, scales = torch.empty(x.shape[0], 16, dtype=torch.uint8), torch.empty(x.shape[0], dtype=torch.uint8)
    assert _lib.load().rldx_host_kv4_encode_bf16(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), x.shape[0]) == 0
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(1).long()
    v = torch.where(c >= 8, -1.0, 1.0).double() * GRID[c % 8] * torch.pow(2.0, scales.double() - 127)[:, None]
    return torch.where(scales[:, None] == 255, torch.nan, v), scales


def _bits(a):
    return torch.from_numpy(np.ascontiguousarray(a.astype(np.uint16)).view(np.int16)).view(BF16)


def _same(got, want):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    g, w = torch.nan_to_num(got), torch.nan_to_num(want)
    assert torch.equal(g, w) and torch.equal(torch.signbit(g), torch.signbit(w))


def test_format_every_bf16_value_beside_every_largest_one():
    """Each of the 65536 values in blocks whose largest magnitude runs over mantissas and exponents (1.75 2^p and its
    neighbours among them), itself among the largest."""
    every = np.arange(65536, dtype=np.uint32)
    for top in (0x3F80, 0x3FDF, 0x3FE0, 0x3FE1, 0x3FFF, 0x0001, 0x007F, 0x0080, 0x0100, 0x7F00, 0x7F60, 0x7F7F, 0x4123):
        rows = np.resize(every, (2115, 31))
        x = _bits(np.concatenate([np.full((rows.shape[0], 1), top, dtype=np.uint32), rows], 1))
        _same(_encode(x)[0], nearest(x))


def test_format_blocks_of_one_magnitude_and_random_ones():
    x = _bits(np.repeat(np.arange(65536, dtype=np.uint32), 32).reshape(-1, 32))
    _same(_encode(x)[0], nearest(x))
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(20000, 32, generator=g) * torch.exp2(torch.randint(-130, 120, (20000, 1), generator=g).float())).to(BF16)
    got, scales = _encode(x)
    _same(got, nearest(x))
    assert torch.isfinite(got).all() and int(scales.min()) >= 2 and int(scales.max()) <= 252
    # half a step at the most (a quarter of the value where 1.5 lies between 1 and 2, 0.25 2^e next to 0)
    e = torch.pow(2.0, scales.double() - 127)[:, None]
    assert ((got - x.double()).abs() <= torch.maximum(x.double().abs() / 4, 0.25 * e)).all()


def test_values_are_exact_in_bf16():
    x = _bits(np.repeat(np.arange(0, 65536, 7, dtype=np.uint32), 32).reshape(-1, 32))
    got = _encode(x)[0]
    back = got.to(BF16).double()
    assert torch.equal(torch.nan_to_num(back), torch.nan_to_num(got))


def test_page_bytes():
    lib = _lib.load()
    assert lib.rldx_kv4_page_bytes(64, 128) == 2 * 34 * 128 and lib.rldx_kv4_page_bytes(32, 64) == 34 * 64
    for t, d in ((0, 64), (16, 64), (48, 64), (64, 96), (-32, 64), (1 << 21, 128)):
        assert lib.rldx_kv4_page_bytes(t, d) == -1
    assert lib.rldx_host_kv4_encode_bf16(None, P, P, 1) != 0 and lib.rldx_host_kv4_encode_bf16(None, None, None, 0) == 0


def test_window_attention_abi_refuses_without_launching():
    lib = _lib.load()
    st = _lib.i64_array([8192, 1024, 128])
    base = dict(q=P, qs=st, k=P, ks=st, v=P, vs=st, o=P, os=st, batch=1, hq=8, hkv=8, sq=4, sk=64, d=128, window=16,
                sinks=2, mask=None, ms=0, scale=0.1, ws=None, wb=0, stream=None)

    def call(**kw):
        return lib.rldx_window_attention_bf16(*{**base, **kw}.values())

    for kw in (dict(d=96), dict(window=0), dict(window=-1), dict(sinks=-1), dict(sq=65), dict(hkv=3), dict(hkv=0),
               dict(batch=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")),
               dict(q=P + 8), dict(k=P + 2), dict(v=P + 8), dict(o=P + 8), dict(mask=P + 2), dict(q=None), dict(k=None),
               dict(v=None), dict(o=None), dict(qs=_lib.i64_array([8192, 1024, 12])), dict(os=None),
               dict(sk=(1 << 30) + 1), dict(batch=1 << 20)):
        assert call(**kw) == INVALID, kw
    assert call(batch=0) == 0 and call(sq=0, sk=0) == 0 and call(hq=0) == 0  # nothing to do
    # a call that needs a workspace refuses to go without, with less, or with one that is not aligned
    need = lib.rldx_window_attention_workspace_bytes(1, 8, 8, 1, 4096, 128, 4096, 0)
    assert need > 0
    for ws, wb in ((None, 0), (None, need), (P, need - 1), (P + 8, need)):
        assert call(sq=1, sk=4096, window=4096, sinks=0, ws=ws, wb=wb) == INVALID
    assert lib.rldx_window_attention_workspace_bytes(1, 8, 8, 5, 4, 128, 4, 0) == -1
    assert lib.rldx_window_attention_workspace_bytes(1, 8, 8, 5, 5, 80, 4, 0) == -1
    assert lib.rldx_window_attention_workspace_bytes(1, 8, 8, 5, 5, 64, 0, 0) == -1


def _cache(**kw):
    n = 2 * 34 * 128
    d = dict(data=P, num_pages=4, kv_heads=2, head_dim=128, page_tokens=64, page_stride=2 * n, head_stride=n, page_table=P,
             table_pages=3, page_table_stride=3)
    return _lib.Kv4Cache(*{**d, **kw}.values())


BAD_CACHES = [dict(head_dim=96), dict(page_tokens=48), dict(page_tokens=16), dict(num_pages=-1), dict(num_pages=1 << 31),
              dict(data=None), dict(data=P + 8), dict(page_stride=2 * 2 * 34 * 128 + 8), dict(page_stride=1024),
              dict(head_stride=1024), dict(head_stride=2 * 34 * 128 + 4), dict(page_table=None), dict(table_pages=-1),
              dict(table_pages=1 << 25), dict(kv_heads=-1), dict(kv_heads=1 << 17)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: "-".join(d))
def test_kv4_abi_refuses_bad_caches(bad):
    lib = _lib.load()
    st = _lib.i64_array([8192, 256, 128])
    c = _cache(**bad)
    assert lib.rldx_kv4_append_bf16(c, P, st, P, st, P, None, 1, 4, None) == INVALID
    assert lib.rldx_kv4_read_bf16(c, P, P, st, P, st, 1, 4, None) == INVALID
    assert lib.rldx_kv4_attention_bf16(P, st, c, P, None, P, st, 1, 4, 1, 64, 0, 0.1, P, 1 << 30, None) == INVALID


def test_kv4_abi_refuses_bad_arguments():
    lib = _lib.load()
    st, odd = _lib.i64_array([8192, 256, 128]), _lib.i64_array([8192, 256, 124])
    c = _cache()
    for a in ((None, P, st, P, st, P, None, 1, 4), (c, None, st, P, st, P, None, 1, 4), (c, P, st, None, st, P, None, 1, 4),
              (c, P + 8, st, P, st, P, None, 1, 4), (c, P, odd, P, st, P, None, 1, 4), (c, P, st, P, None, P, None, 1, 4),
              (c, P, st, P, st, None, None, 1, 4), (c, P, st, P, st, P, None, -1, 4), (c, P, st, P, st, P, None, 1, -4),
              (c, P, st, P, st, P, None, 1 << 17, 4)):
        assert lib.rldx_kv4_append_bf16(*a, None) == INVALID, a
    assert lib.rldx_kv4_append_bf16(c, None, st, None, st, None, None, 0, 4, None) == 0
    assert lib.rldx_kv4_read_bf16(c, None, None, st, None, st, 1, 0, None) == 0
    base = dict(q=P, qs=st, c=c, starts=P, counts=None, o=P, os=st, batch=1, hq=4, sq=1, window=64, sinks=0, scale=0.1,
                ws=None, wb=0, stream=None)
    for kw in (dict(q=None), dict(o=None), dict(starts=None), dict(c=None), dict(hq=3), dict(window=0), dict(sinks=-1),
               dict(scale=0.0), dict(q=P + 8), dict(qs=odd), dict(os=None), dict(batch=-1), dict(sq=-1)):
        assert lib.rldx_kv4_attention_bf16(*{**base, **kw}.values()) == INVALID, kw
    assert lib.rldx_kv4_attention_bf16(*{**base, "batch": 0}.values()) == 0
    need = lib.rldx_kv4_attention_workspace_bytes(1, 4, 2, 1, 128, 64, 64, 1 << 30, 0)
    assert need > 0
    big = _cache(table_pages=64)
    for ws, wb in ((None, 0), (P, need - 1), (P + 8, need)):
        assert lib.rldx_kv4_attention_bf16(*{**base, "c": big, "window": 1 << 30, "ws": ws, "wb": wb}.values()) == INVALID
    assert lib.rldx_kv4_attention_workspace_bytes(1, 4, 2, 1, 128, 48, 64, 64, 0) == -1
    assert lib.rldx_kv4_attention_workspace_bytes(1, 4, 2, 1, 128, 64, 1 << 25, 64, 0) == -1


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 2, 64, dtype=BF16)
    c = torch.zeros(2, 2, 34 * 64, dtype=torch.uint8)
    t, s = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for f in (lambda: Fn.window_attention(x, x, x, 4), lambda: Fn.kv4_append(c, x, x, t, s),
              lambda: Fn.kv4_read(c, t, s, 1, 64), lambda: Fn.kv4_attention(x, c, t, s)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            f()
    with pytest.raises(RuntimeError, match="page_tokens"):
        Fn.kv4_cache(4, 2, 64, page_tokens=48, device="cpu")
    assert Fn.kv4_cache(4, 2, 64, page_tokens=32, device="cpu").shape == (4, 2, 34 * 64)


def test_fakes():
    with FakeTensorMode():
        q, k = torch.empty(2, 5, 8, 128, dtype=BF16), torch.empty(2, 9, 2, 128, dtype=BF16)
        o = torch.ops.rldx_amd.window_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k, k, 4)
        c = torch.empty(4, 2, 34 * 128, dtype=torch.uint8)
        t, s = torch.empty(2, 3, dtype=torch.int32), torch.empty(2, dtype=torch.int32)
        assert torch.ops.rldx_amd.kv4_append(c, k, k, t, s) is None
        rk, rv = torch.ops.rldx_amd.kv4_read(c, t, s, 7, 128)
        a = torch.ops.rldx_amd.kv4_attention(q, c, t, s, None, 16, 2)
    assert o.shape == q.shape and o.is_contiguous() and o.dtype == BF16
    assert rk.shape == rv.shape == (2, 7, 2, 128) and rk.dtype == BF16
    assert a.shape == q.shape and a.dtype == BF16


def test_abi_refuses_sizes_that_the_kernels_do_not_address():
    lib = _lib.load()
    st = _lib.i64_array([8192, 256, 128])
    for seq in (-256, (1 << 24) + 8):
        bad = _lib.i64_array([8192, seq, 128])
        for ks, vs in ((bad, st), (st, bad)):
            assert lib.rldx_window_attention_bf16(P, st, P, ks, P, vs, P, st, 1, 2, 2, 4, 64, 128, 16, 0, None, 0, 0.1, None, 0,
                                                  None) == INVALID
    assert lib.rldx_kv4_append_bf16(_cache(), P, st, P, st, P, None, 1, (1 << 28) + 1, None) == INVALID
    assert lib.rldx_kv4_read_bf16(_cache(), P, P, st, P, st, 1, (1 << 28) + 1, None) == INVALID
    # more threads than a grid has
    assert lib.rldx_window_attention_workspace_bytes(1 << 15, 1 << 13, 1 << 13, 1, 40, 64, 8, 0) == -1
    assert lib.rldx_window_attention_workspace_bytes(1 << 15, 1 << 8, 1 << 8, 1, 40, 64, 8, 0) == 0
