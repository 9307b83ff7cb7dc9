"""Plain 64-bit forms of the serving operators, on the CPU, for their tests."""
import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
E4M3[127] = math.nan
TOP = {'fp4': 6.0, 'fp8': 448.0}


def quantise(x, fmt):
    """x [..., dim] -> (codes uint8, scale bytes uint8, values fp64) by the definition, group by group."""
    grid = torch.tensor((E2M1 if fmt == 'fp4' else E4M3)[:8 if fmt == 'fp4' else 127], dtype=torch.float64)
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    ok = torch.isfinite(g).all(-1)
    k = torch.full(top.shape, -127)
    for e in range(-127, 128):  # the smallest k with top <= MAX 2^k
        k = torch.where((k == e) & (top > TOP[fmt] * 2.0 ** e), e + 1, k)
    k = k.clamp(max=127)
    y = g.abs() * torch.pow(torch.tensor(2.0, dtype=torch.float64), -k)[..., None]
    y = torch.where(ok[..., None], y, 0.0)
    d = (y[..., None] - grid).abs() if fmt == 'fp4' else None
    if fmt == 'fp4':
        # nearest, the even code of two equally near ones
        near = d == d.amin(-1, keepdim=True)
        even = torch.arange(8) % 2 == 0
        code = torch.where((near & even).any(-1), (near & even).int().argmax(-1), near.int().argmax(-1))
    else:
        hi = torch.searchsorted(grid, y.contiguous()).clamp(1, 126)
        lo_d, hi_d = y - grid[hi - 1], grid[hi] - y
        code = torch.where((lo_d < hi_d) | ((lo_d == hi_d) & (hi % 2 == 1)), hi - 1, hi)
    minus = torch.signbit(g)
    val = grid[code] * torch.pow(torch.tensor(2.0, dtype=torch.float64), k)[..., None] * torch.where(minus, -1.0, 1.0)
    val = torch.where(ok[..., None], val, math.nan).flatten(-2)
    code = (code + minus * (8 if fmt == 'fp4' else 128)).flatten(-2)
    if fmt == 'fp4':
        code = code[..., 0::2] + 16 * code[..., 1::2]
    return code.to(torch.uint8), torch.where(ok, k + 127, 255).to(torch.uint8), val


def attend(q, k, v, pos, window, sinks, scale=None):
    """q [m, heads, dim] at positions pos over k, v [n, kv_heads, dim] at 0 .. n - 1, in fp64: (y, terms), with what the error
    bound of y takes of every row: sum of p |v| and sum of |v| over the keys it sees [m, heads, dim], the largest scale sum
    |q k| of a key and the number of keys [m, heads, 1]. Masked keys and values are taken out before any arithmetic."""
    m, heads, dim = q.shape
    n, kv = k.shape[:2]
    scale = dim ** -0.5 if scale is None else scale
    y, mag, tot = (torch.zeros(m, heads, dim, dtype=torch.float64) for _ in range(3))
    big, cnt = (torch.zeros(m, heads, 1, dtype=torch.float64) for _ in range(2))
    j = torch.arange(n)
    k, v = (x.double().repeat_interleave(heads // kv, 1).transpose(0, 1) for x in (k, v))
    for i in range(m):
        s = int(pos[i])
        see = (j <= s) & ((s - j <= window) | (j < sinks)) if window is not None else j <= s
        if s < 0 or not bool(see.any()):
            continue
        kk, vv, qq = k[:, see], v[:, see], q[i].double()[:, :, None]
        p = torch.softmax(torch.matmul(kk, qq)[..., 0] * scale, -1)[..., None]
        y[i] = (p * vv).sum(1)
        mag[i], tot[i] = (p * vv.abs()).sum(1), vv.abs().sum(1)
        big[i, :, 0] = torch.matmul(kk.abs(), qq.abs())[..., 0].amax(-1) * scale
        cnt[i] = int(see.sum())
    return y, (mag, tot, big, cnt)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention_bound(y, terms, dtype, p_dtype):
    """How far an output of `dtype` may be from y:
    - its own rounding, half a step (and fp16's smallest, 2^-25);
    - the probabilities' rounding to p_dtype (None: they stay in fp32), half a step each in the product and in the sum that
      divides it; fp16 ones below 2^-14 are off by up to 2^-25 of the largest;
    - fp32: a score's dim products and sums, its scaling and the exponential's argument, (dim + 8) half steps of sum |q k|; the
      exponential's last place and at most `cnt` additions of a sum: twice, in the product and in the divisor."""
    mag, tot, big, cnt = terms
    fp32 = 2 * 2.0 ** -24 * ((y.shape[-1] + 8) * big + cnt + 8)
    up = 0.0 if p_dtype is None else 2 * half_step(p_dtype)
    off = half_step(dtype) * y.abs() + 1.01 * (up + fp32) * mag
    if dtype == torch.float16:
        off = off + 2.0 ** -25
    if p_dtype == torch.float16:
        off = off + 2.0 ** -25 * tot
    return off + 1e-30
