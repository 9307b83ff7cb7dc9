"""Refusals of the serving operators (host side, no GPU): the C ABI's checks return an error before any launch, the Python
wrappers raise before they call it. Also checks the tests' own 64-bit forms against other formulations."""
import ctypes
import math

import pytest
import torch

from noise_amd import _lib, ops
from noise_amd.cache import KVCache
from tests import _serving as plain

EINVAL, ENOSPC = -1, -2


def cache(**kw):
    a = dict(keys=16, key_scales=16, values=16, value_scales=16, pages=4, page_size=64, kv_heads=8, dim=64, format=0)
    a.update(kw)
    return _lib.Cache(*a.values())


def seqs(**kw):
    a = dict(table=16, table_ld=2, table_pages=2, lengths=16, starts=None, sequences=3, rows=3)
    a.update(kw)
    return _lib.Sequences(*a.values())


BAD_CACHES = [dict(keys=None), dict(values=None), dict(key_scales=None), dict(value_scales=None), dict(keys=8), dict(values=24),
              dict(key_scales=2), dict(pages=0), dict(pages=2 ** 31), dict(page_size=0), dict(page_size=8), dict(page_size=48),
              dict(page_size=512), dict(kv_heads=0), dict(kv_heads=2048), dict(dim=32), dict(dim=96), dict(format=2)]
BAD_SEQS = [dict(table=None), dict(table_ld=-1), dict(table_pages=-1), dict(lengths=None), dict(sequences=0), dict(rows=0),
            dict(rows=4), dict(sequences=-1)]


@pytest.mark.parametrize('c,s', [(c, {}) for c in BAD_CACHES] + [({}, s) for s in BAD_SEQS])
def test_bad_caches_and_rows_are_refused(c, s):
    lib = _lib.load()
    cc, ss = cache(**c), seqs(**s)
    a, b = ctypes.addressof(cc), ctypes.addressof(ss)
    assert lib.noise_cache_write(a, b, 16, 512, 64, 16, 512, 64, 0, None) == EINVAL
    assert lib.noise_cache_read(a, b, 16, 16, 0, None) == EINVAL
    assert lib.noise_cache_attend(a, b, 16, 512, 64, 0, 8, 100, 0, 0.125, 16, 1, 16, 1 << 40, None) == EINVAL
    assert lib.noise_cache_attend_workspace_size(a, b, 8, 0, ctypes.byref(ctypes.c_size_t())) == EINVAL


def test_bad_operands_are_refused():
    lib = _lib.load()
    cc, ss = cache(), seqs()
    a, b = ctypes.addressof(cc), ctypes.addressof(ss)
    write = lambda k=16, ld=512, hs=64, t=0: lib.noise_cache_write(a, b, k, ld, hs, 16, 512, 64, t, None)  # noqa: E731
    for bad in (dict(k=None), dict(k=8), dict(ld=4), dict(hs=-8), dict(ld=-512), dict(t=3), dict(t=-1)):
        assert write(**bad) == EINVAL, bad
    assert lib.noise_cache_write(None, b, 16, 512, 64, 16, 512, 64, 0, None) == EINVAL
    assert lib.noise_cache_write(a, None, 16, 512, 64, 16, 512, 64, 0, None) == EINVAL
    assert lib.noise_cache_read(a, b, None, 16, 0, None) == EINVAL
    assert lib.noise_cache_read(a, b, 16, 24, 0, None) == EINVAL
    att = lambda q=16, ld=512, t=0, h=8, w=9, s=0, sc=0.1, y=16: lib.noise_cache_attend(  # noqa: E731
        a, b, q, ld, 64, t, h, w, s, sc, y, 1, 16, 1 << 40, None)
    for bad in (dict(q=None), dict(q=8), dict(ld=12), dict(t=2), dict(h=0), dict(h=12), dict(h=2048), dict(w=-1), dict(s=-1),
                dict(sc=-1.0), dict(sc=math.nan), dict(y=None), dict(y=8)):
        assert att(**bad) == EINVAL, bad
    sink = lambda q=16, k=16, ld=512, st=None, n=2, rows=200, T=100, h=8, kv=8, dim=64, t=0, w=9, s=0, sc=0.1, y=16: (  # noqa: E731
        lib.noise_sink_attention(q, ld, 64, k, 512, 64, 16, 512, 64, st, n, rows, T, h, kv, dim, t, w, s, sc, y, 1, None))
    for bad in (dict(q=None), dict(k=None), dict(k=8), dict(ld=4), dict(n=0), dict(rows=0), dict(rows=150), dict(T=0), dict(h=0),
                dict(h=12), dict(kv=0), dict(dim=96), dict(t=2), dict(w=-1), dict(s=-2), dict(sc=-0.1), dict(y=None), dict(y=4)):
        assert sink(**bad) == EINVAL, bad


def test_wrappers_refuse_what_the_kernels_do_not_take():
    x = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='CUDA'):
        ops.sink_attention(x, x, x, torch.tensor([0, 4], dtype=torch.int32))
    g = x.float().requires_grad_()
    with pytest.raises(RuntimeError, match='no backward'):
        ops.sink_attention(g, g, g)
    with pytest.raises(ValueError, match='CUDA'):
        KVCache.zeros(4, device='cpu')
    with pytest.raises(ValueError, match='format'):
        KVCache.zeros(4, format='int4', device='cpu')
    for bad in (dict(window=-1), dict(sinks=-1), dict(scale=math.inf), dict(scale=-1.0), dict(scale=math.nan)):
        with pytest.raises(ValueError):
            ops.mask_args(**{**dict(window=None, sinks=0, scale=None, dim=64), **bad})
    assert ops.mask_args(None, 0, None, 64) == (2 ** 31 - 1, 0, 0.125)
    assert ops.mask_args(2 ** 40, 2 ** 40, 1, 64) == (2 ** 31 - 1, 2 ** 31 - 1, 1.0)


def test_rows_are_read_in_place_where_they_can_be():
    x = torch.zeros(10, 3, 8, 64, dtype=torch.bfloat16)
    t, p, ld, hs = ops.heads_rows(x[:, 1])
    assert p == x.data_ptr() + 2 * 512 and (ld, hs) == (1536, 64) and t.data_ptr() == p
    for bad in (x[:, 1].transpose(1, 2).contiguous().transpose(1, 2), x[:, 0, :, 1:][:, :, :63].repeat(1, 1, 2)[:, :, 1:65],
                torch.zeros(10, 8 * 64 + 4, dtype=torch.bfloat16)[:, 4:].view(10, 8, 64)):
        t, p, ld, hs = ops.heads_rows(bad)
        assert (ld, hs) == (512, 64) and p % 16 == 0 and torch.equal(t, bad)
    t, p, ld, hs = ops.heads_rows(x[:1, 0, :1])  # strides of one entry are not read
    assert (ld, hs) == (0, 0)


@pytest.mark.parametrize('fmt', ['fp4', 'fp8'])
def test_plain_quantisation(fmt):
    """The plain form against another formulation of its scale, at its borders, and its error bound."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 64, generator=g).double() * torch.exp2(torch.randint(-20, 20, (200, 1), generator=g).double())
    x[0, :32] = 0
    x[1, 3] = math.inf
    x[2, :32] = torch.linspace(-6, 6, 32)
    x[3, :32] = torch.linspace(-448, 448, 32)
    codes, e, val = plain.quantise(x, fmt)
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1)
    assert int(e[0, 0]) == 0 and int(e[1, 0]) == 255 and torch.isnan(val[1, :32]).all()
    good = torch.isfinite(top) & (top > 0)
    k = (e.double() - 127)[good]
    assert torch.equal(k, torch.ceil(torch.log2(top[good] / plain.TOP[fmt])))
    # a nearest code is at most half a step off: 2^-2 of the value in e2m1, 2^-4 in e4m3, or half the smallest code
    rel, least = (0.25, 0.25) if fmt == 'fp4' else (2 ** -4, 2.0 ** -10)
    err = (val - x).abs()
    tol = torch.maximum(rel * x.abs(), least * torch.exp2(e.double() - 127).repeat_interleave(32, -1))
    fine = torch.isfinite(val)
    assert (err[fine] <= tol[fine]).all()


def test_plain_attention_masks():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(9, h, 64, generator=g).double() for h in (4, 2, 2))
    y, _ = plain.attend(q, k, v, torch.arange(9), 3, 2)
    z = torch.einsum('ihd,jhd->hij', q, k.repeat_interleave(2, 1)) / 8
    i, j = torch.arange(9)[:, None], torch.arange(9)[None]
    z = z.masked_fill(~((j <= i) & ((i - j <= 3) | (j < 2))), -math.inf)
    assert torch.allclose(y, torch.einsum('hij,jhd->ihd', z.softmax(-1), v.repeat_interleave(2, 1)), atol=1e-12)
    y, _ = plain.attend(q[:2], k, v, torch.tensor([-1, 0]), None, 0)
    assert not y[0].any() and torch.allclose(y[1], v[0].repeat_interleave(2, 0), atol=1e-12)
