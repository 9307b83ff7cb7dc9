"""The serving operators on the GPU against their 64-bit forms (tests/_serving.py): attention of whole prompts, and the
microscaled cache, written, read back and attended to."""
import math

import pytest
import torch

from noise_amd import ops
from noise_amd.cache import KVCache
from tests import _serving as plain
from tests._util import log_case

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts_of(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


def rows(gen, n, heads, dim, dtype, scale=1.0):
    x = torch.randn(n, heads, dim, generator=gen)
    x *= 1 + 4 * (torch.rand(heads, dim, generator=gen) > 0.95)
    return (x * scale).to(dtype)


def check(got, y, terms, dtype, p_dtype, what=''):
    got = got.double().cpu()
    off, tol = (got - y).abs(), plain.attention_bound(y, terms, dtype, p_dtype)
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((off / tol).max()), bad.nonzero()[:4].tolist())


# ------------------------------------------------------------------ prompts

PROMPTS = [
    # lens, heads, kv_heads, dim, dtype, window, sinks
    ([1], 8, 8, 64, BF16, None, 0),
    ([1, 2, 3, 0, 63, 64, 65], 8, 8, 64, BF16, None, 0),
    ([127, 128, 129, 0, 0, 33], 4, 1, 128, F16, None, 0),
    ([300], 8, 8, 64, F16, 100, 4),
    ([257, 1, 130], 8, 2, 64, BF16, 0, 0),
    ([257, 5], 3, 3, 64, BF16, 0, 1),
    ([400], 8, 8, 64, BF16, 64, 70),
    ([333, 200], 6, 2, 128, BF16, 37, 130),
    ([500], 2, 1, 64, F16, 1, 200),
    ([640, 90], 8, 1, 128, F16, 255, 3),
    ([1500], 2, 2, 64, BF16, 1024, 4),
    ([1100], 1, 1, 128, BF16, 10 ** 6, 0),
]


def prompt(case, seed=0):
    lens, heads, kv, dim, dtype, window, sinks = case
    g = torch.Generator().manual_seed(seed)
    n = sum(lens)
    return rows(g, n, heads, dim, dtype), rows(g, n, kv, dim, dtype), rows(g, n, kv, dim, dtype)


def prompt_reference(q, k, v, lens, window, sinks, scale=None):
    parts, s = [], 0
    for n in lens:
        parts.append(plain.attend(q[s:s + n], k[s:s + n], v[s:s + n], torch.arange(n), window, sinks, scale))
        s += n
    return torch.cat([p[0] for p in parts]), tuple(torch.cat(t) for t in zip(*[p[1] for p in parts]))


@pytest.mark.parametrize('case', PROMPTS, ids=[str(i) for i in range(len(PROMPTS))])
def test_prompts_match_the_plain_form(case):
    log_case(f'prompt {case}')
    lens, *_, dtype, window, sinks = case
    q, k, v = prompt(case)
    y, terms = prompt_reference(q, k, v, lens, window, sinks)
    got = ops.sink_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(starts_of(lens)), window=window, sinks=sinks)
    check(got, y, terms, dtype, dtype)


# (tiles of 64 queries by one group of waves, and of 128 queries: many heads)
@pytest.mark.parametrize('case', [
    ([700, 0, 301, 1], 64, 8, 64, BF16, 200, 5),
    ([900, 60], 64, 64, 64, F16, None, 0),
    ([700, 0, 501], 32, 4, 128, BF16, 200, 5),
    ([129, 0, 301, 1] + [70] * 12, 64, 8, 64, F16, 100, 5),
    ([1000, 257], 80, 16, 64, BF16, None, 0),
    ([513, 300, 64], 100, 4, 128, BF16, None, 0),
    ([30, 1, 200] + [65] * 70, 6, 2, 128, F16, 50, 2),
], ids=str)
def test_prompts_of_many_tiles(case):
    log_case(f'prompt {case}')
    lens, *_, dtype, window, sinks = case
    q, k, v = prompt(case, 5)
    y, terms = prompt_reference(q, k, v, lens, window, sinks)
    got = ops.sink_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(starts_of(lens)), window=window, sinks=sinks)
    check(got, y, terms, dtype, dtype)


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('heads', [4, 64, 128])
def test_unseen_values_in_every_kind_of_tile(heads, bad):
    """Values that come after a row, and before its window, hold NaN or infinities: rows that see none of them are what they were."""
    lens, window, n = [300, 400], 60, 700
    q, k, v = prompt((lens, heads, 1, 64, BF16, window, 0), 8)
    want = ops.sink_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(starts_of(lens)), window=window).cpu()
    v[250:300] = bad
    v[500] = bad
    got = ops.sink_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(starts_of(lens)), window=window).cpu()
    clean = torch.ones(n, dtype=torch.bool)
    clean[250:300] = False
    clean[500:500 + window + 1] = False
    assert (got[clean] - want[clean]).abs().max() <= 2 ** -7 * want.abs().max()  # (sums in another order: a rounding either way)
    assert not torch.isfinite(got[~clean]).any()


def test_prompt_batches_are_packed_sequences():
    """[batch, T, heads, dim] gives the bits of the packed call; fused and padded strides are read in place."""
    g = torch.Generator().manual_seed(3)
    B, T, H = 3, 150, 4
    fused = torch.randn(B, T, 3, H, 64, generator=g).to(BF16).to(DEV)
    q, k, v = fused.unbind(2)
    packed = [x.reshape(B * T, H, 64).contiguous() for x in (q, k, v)]
    want = ops.sink_attention(*packed, i32([0, T, 2 * T, 3 * T]), window=70, sinks=2)
    assert torch.equal(ops.sink_attention(q, k, v, window=70, sinks=2).view(B * T, H, 64), want)
    f = fused.view(B * T, 3, H, 64)
    assert torch.equal(ops.sink_attention(f[:, 0], f[:, 1], f[:, 2], i32([0, T, 2 * T, 3 * T]), window=70, sinks=2), want)
    odd = [torch.cat((torch.zeros(B * T, H, 3, device=DEV, dtype=BF16), x), -1)[:, :, 3:] for x in packed]  # not 16-byte rows
    assert torch.equal(ops.sink_attention(*odd, i32([0, T, 2 * T, 3 * T]), window=70, sinks=2), want)
    far = torch.zeros(2, 2 ** 23 + 64, device=DEV, dtype=BF16).as_strided((2, 1, 64), (2 ** 23, 64, 1))  # rows far apart
    far.copy_(packed[1][:2, :1])
    pair = ops.sink_attention(packed[0][:2], packed[1][:2, :1], packed[2][:2, :1], i32([0, 2]))
    assert torch.equal(ops.sink_attention(packed[0][:2], far, packed[2][:2, :1], i32([0, 2])), pair)
    shared = packed[1][:, :1].expand(-1, H, -1)  # one kv head broadcast to all
    one = ops.sink_attention(packed[0], packed[1][:, :1], packed[2][:, :1], i32([0, B * T]))
    assert torch.equal(ops.sink_attention(packed[0], shared, packed[2][:, :1].expand(-1, H, -1), i32([0, B * T])), one)


def test_prompt_scale_and_large_scores():
    """Scores of +-hundreds (the running maximum moves often) and a given scale."""
    g = torch.Generator().manual_seed(4)
    lens = [260, 100]
    q, k, v = (rows(g, 360, 2, 64, BF16, s) for s in (3, 3, 1))
    for scale in (1.0, 0.0):
        y, terms = prompt_reference(q, k, v, lens, 90, 5, scale)
        got = ops.sink_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(starts_of(lens)), window=90, sinks=5, scale=scale)
        check(got, y, terms, BF16, BF16, scale)


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf, 3e38])
def test_what_a_prompt_row_does_not_see_takes_no_part(bad, dim):
    """Keys and values of one position are NaN, infinite or the type's largest: rows that do not see it are as without it."""
    g = torch.Generator().manual_seed(5)
    n, window, sinks = 300, 60, 3
    q, k, v = (rows(g, n, 2, dim, BF16) for _ in range(3))
    y, terms = prompt_reference(q, k, v, [n], window, sinks)
    at = torch.arange(n)
    for where in (100, 63, 64, 1, 299):
        kb, vb = k.clone(), v.clone()
        kb[where], vb[where] = bad, bad
        got = ops.sink_attention(q.to(DEV), kb.to(DEV), vb.to(DEV), i32([0, n]), window=window, sinks=sinks).cpu()
        blind = (at < where) | ((at - where > window) & (where >= sinks))
        check(got[blind], y[blind], tuple(t[blind] for t in terms), BF16, BF16, where)
        if math.isnan(bad):
            assert torch.isnan(got[~blind]).all()


def test_an_infinite_value_shows_in_the_rows_that_see_it():
    g = torch.Generator().manual_seed(6)
    q, k, v = (rows(g, 200, 2, 64, BF16) for _ in range(3))
    v[70, 1, 5] = math.inf
    got = ops.sink_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32([0, 200]), window=40).cpu()
    sees = (torch.arange(200) >= 70) & (torch.arange(200) <= 110)
    want = torch.zeros(200, 2, 64, dtype=torch.bool)
    want[sees, 1, 5] = True
    assert torch.equal(torch.isinf(got), want) and not torch.isnan(got).any()


def test_rows_behind_the_last_prompt():
    """Rows of no sequence are zero in a fresh output and left as they were in a given one."""
    g = torch.Generator().manual_seed(7)
    q, k, v = (rows(g, 400, 2, 64, F16).to(DEV) for _ in range(3))
    q[290:] = math.nan
    k[290:] = math.nan
    v[290:] = math.nan
    st = i32([10, 150, 150, 290])
    got = ops.sink_attention(q, k, v, st, window=50)
    assert not got[:10].any() and not got[290:].any() and bool(got[10:290].any(-1).all())
    out = torch.full_like(got, 7.0)
    assert ops.sink_attention(q, k, v, st, window=50, out=out) is out
    assert (out[:10] == 7).all() and (out[290:] == 7).all() and torch.equal(out[10:290], got[10:290])
    assert not ops.sink_attention(q, k, v, i32([0]), window=50).any()
    assert ops.sink_attention(q[:0], k[:0], v[:0], i32([0, 0])).shape == (0, 2, 64)
    assert ops.sink_attention(*(x[:0].view(0, 5, 2, 64) for x in (q, k, v))).shape == (0, 5, 2, 64)


def test_many_prompts():
    """More sequences than one search round covers, many empty."""
    g = torch.Generator().manual_seed(8)
    lens = [int(x) for x in torch.randint(0, 4, (5000,), generator=g)]
    q, k, v = (rows(g, sum(lens), 1, 64, BF16) for _ in range(3))
    y, terms = prompt_reference(q, k, v, lens, None, 0)
    check(ops.sink_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(starts_of(lens))), y, terms, BF16, BF16)
    for heads in (1, 8):
        x = rows(g, 900, heads, 64, BF16).to(DEV)  # (sequences of one length, with and without starts)
        want = ops.sink_attention(x, x, x, i32(range(0, 901, 3)), window=1)
        assert torch.equal(ops.sink_attention(*[x.view(300, 3, heads, 64)] * 3, window=1).view(900, heads, 64), want)


def test_prompt_types_and_shapes_are_refused():
    x = torch.zeros(6, 4, 64, device=DEV, dtype=BF16)
    st = i32([0, 6])
    for q, k, v, s in ((x, x.half(), x, st), (x.float(), x.float(), x.float(), st), (x, x, x, None), (x, x[:5], x[:5], st),
                       (x, x[:, :3], x[:, :3], st), (x[..., :32], x[..., :32], x[..., :32], st), (x, x, x[:, :2], st),
                       (x, x, x, st.long()), (x, x, x, st[:0]), (x, x, x, st.cpu()), (x, x.cpu(), x, st)):
        with pytest.raises((ValueError, TypeError)):
            ops.sink_attention(q, k, v, s)
    for out in (x.half(), x[:5], x.transpose(0, 1).contiguous().transpose(0, 1), x.cpu()):
        with pytest.raises(ValueError):
            ops.sink_attention(x, x, x, st, out=out)
    with pytest.raises(RuntimeError, match='no backward'):
        ops.sink_attention(x.clone().requires_grad_(), x, x, st)


# ------------------------------------------------------------------ the cache


class Filled:
    """A cache with random pages for sequences of `lens` tokens, and what it holds, in fp64 on the CPU."""

    def __init__(self, lens, kv, dim, fmt, page, seed=0, spare=3, dtype=BF16):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).tolist()
        self.cols = max(1, max(need, default=0))
        table = torch.full((len(lens), self.cols), -1, dtype=torch.int32)
        self.k, self.v = [], []
        self.lens, self.page = lens, page
        self.cache = KVCache.zeros(pages, kv, dim, page, fmt)
        for b, n in enumerate(lens):
            for p in range(need[b]):
                table[b, p] = order.pop()
            self.k.append(rows(g, n, kv, dim, dtype))
            self.v.append(rows(g, n, kv, dim, dtype))
        self.table, self.lengths = table.to(DEV), i32(lens)
        self.starts = i32(starts_of(lens))
        if sum(lens):
            self.cache.write(torch.cat(self.k).to(DEV), torch.cat(self.v).to(DEV), self.table, self.lengths, self.starts)
        self.held = [tuple(plain.quantise(x[b], fmt)[2] for x in (self.k, self.v)) for b in range(len(lens))]


@pytest.mark.parametrize('fmt', ['fp4', 'fp8'])
@pytest.mark.parametrize('dtype', [BF16, F16, F32])
def test_written_codes_and_values(fmt, dtype):
    """Codes and scale bytes as the definition gives them, bit for bit, over magnitudes, ties, zeros and non-finite values; the
    values read back are theirs."""
    g = torch.Generator().manual_seed(11)
    kv, dim, page, n = 3, 64, 16, 70
    x = torch.randn(n, kv, dim, generator=g) * torch.exp2(torch.randint(-12, 12, (n, kv, 1), generator=g).float())
    x[0] = 0
    x[1, 0, :32] = torch.linspace(-6, 6, 32)
    x[1, 1] = torch.randint(-24, 25, (dim,), generator=g) / 4  # ties of every step
    x[1, 2, 32:] = torch.randint(-448, 449, (32,), generator=g).float()
    x[2, 0, 7], x[2, 1, 40], x[2, 2, 0] = math.nan, math.inf, -math.inf
    x[3, 0] = -0.0
    if dtype != F16:
        x[4] *= 2.0 ** 100
        x[5] *= 2.0 ** -110
        x[6] = torch.finfo(dtype).max
        x[7] = torch.finfo(dtype).tiny / 4  # below the smallest normal number
        x[8, 0, 0] = torch.finfo(dtype).max
    else:
        x[6] = 65504
        x[7] = 2.0 ** -24
    k = x.to(dtype)
    v = x.flip(0).to(dtype)
    cache = KVCache.zeros(8, kv, dim, page, fmt)
    table = i32([[5, 0, 7, 2, 1]])
    cache.write(k.to(DEV), v.to(DEV), table, i32([n]), i32([0, n]))
    for t, codes, scales in ((k, cache.keys, cache.key_scales), (v, cache.values, cache.value_scales)):
        c, e, val = plain.quantise(t, fmt)
        at = table[0].cpu().long()
        got_c = codes.cpu()[at].transpose(1, 2).flatten(0, 1)[:n]
        got_e = scales.cpu()[at].transpose(1, 2).flatten(0, 1)[:n]
        assert torch.equal(got_e, e)
        fine = (e != 255).repeat_interleave(c.shape[-1] // e.shape[-1], -1)
        assert torch.equal(got_c[fine], c[fine])
    assert not cache.keys.cpu()[[3, 4, 6]].any() and not cache.values.cpu()[1, :, 6:].any()
    for out in (BF16, F16, F32):
        got = cache.read(table, i32([n]), i32([0, n]), rows=n, dtype=out)
        for a, t in zip(got, (k, v)):
            want = plain.quantise(t, fmt)[2].to(out)
            assert torch.equal(a.cpu().nan_to_num(nan=123.0), want.nan_to_num(nan=123.0)), (out,)


@pytest.mark.parametrize('dim,page,kv', [(64, 16, 8), (128, 64, 2), (64, 256, 1), (128, 32, 5)])
def test_rows_go_to_their_places(dim, page, kv):
    """Prompts and steps of ragged sequences, strided rows, rows of no sequence: every other byte of the cache stays."""
    g = torch.Generator().manual_seed(12)
    lens, new = [1, 0, 100, 37, 300], [1, 0, 60, 37, 5]
    f = Filled(lens, kv, dim, 'fp4', page, seed=12)
    before = [t.clone() for t in (f.cache.keys, f.cache.key_scales, f.cache.values, f.cache.value_scales)]
    st = [2 + s for s in starts_of(new)]
    n = st[-1] + 3  # two rows before the first sequence, three behind the last
    fused = rows(g, n, 2 * kv, dim, F16)
    k, v = fused[:, :kv], fused[:, kv:]
    f.cache.write(fused.to(DEV)[:, :kv], fused.to(DEV)[:, kv:], f.table, f.lengths, i32(st))
    for b, (m, s) in enumerate(zip(new, st)):
        for i, x in enumerate((k, v)):
            f.held[b][i][lens[b] - m:] = plain.quantise(x[s:s + m], 'fp4')[2]
    whole = f.cache.read(f.table, f.lengths, f.starts, rows=sum(lens), dtype=F32)
    for i in range(2):
        want = torch.cat([h[i] for h in f.held])
        assert torch.equal(whole[i].cpu(), want.float())
    got = f.cache.read(f.table, f.lengths, i32(st), rows=n, dtype=F32)
    for i in range(2):
        assert not got[i][:2].any() and not got[i][-3:].any()
        assert torch.equal(got[i][2:-3].cpu(), torch.cat([h[i][ln - m:] for h, ln, m in zip(f.held, lens, new)]).float())
    # nothing else was written
    mine = torch.zeros(f.cache.pages, page, dtype=torch.bool)
    for b, ln in enumerate(lens):
        for p in range(ln):
            mine[int(f.table[b, p // page]), p % page] = True
    for now, was in zip((f.cache.keys, f.cache.key_scales, f.cache.values, f.cache.value_scales), before):
        same = (now == was).all(-1).all(1).cpu()
        assert bool(same[~mine].all())


def test_rows_at_no_place_and_at_bad_ones():
    """Negative positions are dropped and read as zeros; pages outside the cache, or past the table, are dropped and read as NaN."""
    kv, dim, page = 2, 64, 16
    cache = KVCache.zeros(4, kv, dim, page, 'fp8')
    x = torch.ones(6, kv, dim, device=DEV, dtype=BF16)
    table = i32([[0, 4], [-1, 1], [2, 3], [3, 3], [0, 0], [2 ** 31 - 1, -2 ** 31]])
    lengths = i32([17, 1, 0, 33, -5, 2])
    cache.write(x, x, table, lengths)  # positions 16, 0, -1, 32, -6, 1: none of them is a good place
    assert not cache.keys.any() and not cache.value_scales.any()
    for t in cache.read(table, lengths):
        assert torch.isnan(t[[0, 1, 3, 5]]).all() and not t[[2, 4]].any()
    y = cache.attend(x, table, lengths)
    assert torch.isnan(y[[0, 1, 3, 5]]).all() and not y[[2, 4]].any()
    none = table[:, :0]
    assert torch.isnan(cache.attend(x, none, i32([1] * 6))).all() and not cache.attend(x, none, i32([0] * 6)).any()
    cache.write(x, x, none, i32([1] * 6))
    assert not cache.keys.any()


def test_rows_before_and_past_the_table():
    """A sequence longer than its table: the rows at positions that the table names are attended to, the others are NaN."""
    f = Filled([128], 2, 64, 'fp4', 16, seed=13)
    q = rows(torch.Generator().manual_seed(14), 40, 4, 64, BF16)
    pos = torch.arange(95, 135)
    y, terms = plain.attend(q, *f.held[0], pos.clamp(max=127), 50, 3)
    got = f.cache.attend(q.to(DEV), f.table, i32([135]), i32([0, 40]), window=50, sinks=3).cpu()
    assert torch.isnan(got[pos > 127]).all()
    ok = pos <= 127
    check(got[ok], y[ok], tuple(t[ok] for t in terms), BF16, P_CACHE)
    x = torch.ones(40, 2, 64, device=DEV, dtype=BF16)
    f.cache.write(x, x, f.table, i32([135]), i32([0, 40]))
    k, _ = f.cache.read(f.table, i32([135]), i32([0, 40]), rows=40)
    assert (k[:33] == 1).all() and torch.isnan(k[33:]).all()


def test_nothing_is_written_or_read_for_no_rows():
    cache = KVCache.zeros(2, 1, 64, 16, 'fp4')
    x = torch.ones(3, 1, 64, device=DEV, dtype=BF16)
    none, zero = i32([]).view(0, 1), i32([])
    cache.write(x, x, none, zero, i32([0]))
    cache.write(x[:0], x[:0], none, zero)
    assert not cache.keys.any()
    k, v = cache.read(none, zero, i32([0]), rows=3)
    assert not k.any() and not v.any() and not cache.attend(x, none, zero, i32([0])).any()
    assert cache.attend(x[:0], none, zero).shape == (0, 1, 64) and cache.read(none, zero)[0].shape == (0, 1, 64)


ATTEND = [
    # lens, new (None: one row each, without starts), heads, kv_heads, dim, format, page, dtype, window, sinks
    ([1], None, 8, 8, 64, 'fp4', 64, BF16, None, 0),
    ([1, 2, 0, 15, 16, 17, 63, 64, 65, 700], None, 8, 8, 64, 'fp4', 16, BF16, None, 0),
    ([5, 129, 1000, 255], None, 8, 8, 64, 'fp8', 64, F16, None, 0),
    ([300, 50], None, 4, 2, 64, 'fp4', 32, F16, 100, 4),
    ([3000, 1, 257], None, 16, 2, 128, 'fp4', 128, BF16, None, 0),
    ([2500, 31], None, 8, 1, 128, 'fp8', 256, F16, 1024, 4),
    ([400, 0, 77], [5, 0, 1], 8, 8, 64, 'fp4', 64, BF16, 64, 70),
    ([333, 20], [3, 20], 6, 2, 128, 'fp8', 16, BF16, 37, 130),
    ([600, 10], [8, 4], 32, 4, 128, 'fp4', 64, F16, 0, 0),
    ([150], [150], 4, 4, 64, 'fp4', 64, BF16, 30, 2),
    ([40, 200], [45, 130], 4, 1, 64, 'fp8', 32, F16, None, 0),
    ([9000], None, 8, 8, 64, 'fp4', 64, BF16, None, 0),
    ([9000], None, 4, 4, 64, 'fp8', 64, BF16, 5000, 8),
    ([700, 800, 900], None, 3, 3, 128, 'fp4', 64, BF16, 1, 300),
    ([1300], None, 64, 1, 64, 'fp4', 64, F16, None, 0),
    # many sequences: shared out over the GPU, and a workgroup each; several tiles of rows on long tables
    ([(37 * i) % 300 for i in range(90)] + [2500], None, 2, 2, 64, 'fp4', 64, BF16, None, 0),
    ([(37 * i) % 300 for i in range(150)], None, 8, 8, 64, 'fp4', 32, BF16, 100, 3),
    ([3000, 0, 40, 2500], [40, 0, 3, 21], 4, 2, 64, 'fp8', 16, BF16, None, 0),
    ([3000, 2500], [30, 50], 8, 1, 128, 'fp4', 64, F16, 700, 90),
    ([4000, 900, 0], None, 4, 2, 128, 'fp8', 64, F16, None, 0),
    ([2300] * 3, [2, 1, 3], 1, 1, 128, 'fp8', 256, BF16, 2000, 4),
    # windows of more blocks than a workgroup takes alone, and of fewer on long tables
    ([4100, 3900, 10], [20, 1, 3], 4, 2, 64, 'fp4', 32, BF16, 2700, 70),
    ([4100, 3900, 10], [20, 1, 3], 16, 2, 64, 'fp8', 64, F16, 200, 70),
]
P_CACHE = BF16  # bf16 queries' probabilities are rounded to bf16 in front of the values; fp16's are two bf16 terms


def attend_reference(f, q, new, window, sinks, scale=None):
    parts, s = [], 0
    for (hk, hv), n, m in zip(f.held, f.lens, new):
        parts.append(plain.attend(q[s:s + m], hk, hv, torch.arange(n - m, n), window, sinks, scale))
        s += m
    return torch.cat([p[0] for p in parts]), tuple(torch.cat(t) for t in zip(*[p[1] for p in parts]))


@pytest.mark.parametrize('case', ATTEND, ids=[str(i) for i in range(len(ATTEND))])
def test_attention_over_the_cache(case):
    log_case(f'attend {case}')
    lens, new, heads, kv, dim, fmt, page, dtype, window, sinks = case
    f = Filled(lens, kv, dim, fmt, page, seed=len(lens))
    m = new or [1] * len(lens)
    q = rows(torch.Generator().manual_seed(9), sum(m), heads, dim, dtype)
    y, terms = attend_reference(f, q, m, window, sinks)
    st = i32(starts_of(m)) if new else None
    got = f.cache.attend(q.to(DEV), f.table, f.lengths, st, window=window, sinks=sinks)
    check(got, y, terms, dtype, P_CACHE if dtype == BF16 else None)


@pytest.mark.parametrize('step,heads,kv', [(True, 2, 2), (False, 20, 1)])
def test_many_cached_sequences(step, heads, kv):
    """More sequences than two search rounds cover, many empty; and on tables long enough for the rows to be shared out."""
    g = torch.Generator().manual_seed(50)
    for n, top, pages in ((5000, 40, 3), (300, 40, 300)):
        lens = [int(x) for x in torch.randint(0, top, (n,), generator=g)]
        new = [1] * n if step else [int(x) for x in torch.randint(0, 3, (n,), generator=g)]
        f = Filled(lens, kv, 64, 'fp8', 16, seed=51)
        q = rows(g, sum(new), heads, 64, BF16)
        y, terms = attend_reference(f, q, new, None, 0)
        table = torch.cat((f.table, torch.zeros(n, pages - f.table.shape[1], device=DEV, dtype=torch.int32)), 1)
        check(f.cache.attend(q.to(DEV), table, f.lengths, None if step else i32(starts_of(new))), y, terms, BF16, P_CACHE)


def test_cache_scale_and_large_scores():
    f = Filled([700, 90], 2, 64, 'fp8', 32, seed=21)
    q = rows(torch.Generator().manual_seed(22), 2, 4, 64, BF16, 9)
    for scale in (1.0, 0.0):
        y, terms = attend_reference(f, q, [1, 1], None, 0, scale)
        check(f.cache.attend(q.to(DEV), f.table, f.lengths, scale=scale), y, terms, BF16, P_CACHE, scale)


@pytest.mark.parametrize('heads', [2, 32])
@pytest.mark.parametrize('fmt,dim', [('fp4', 64), ('fp8', 128)])
def test_what_a_cached_row_does_not_see_takes_no_part(fmt, dim, heads):
    """Every slot that a row does not see holds NaN, and every page that it does not need is a bad one."""
    lens, new, window, sinks, page = [700, 20, 150], [4, 1, 1], 100, 5, 16
    f = Filled(lens, 2, dim, fmt, page, seed=23)
    q = rows(torch.Generator().manual_seed(24), 6, heads, dim, BF16)
    y, terms = attend_reference(f, q, new, window, sinks)
    seen = torch.zeros(f.cache.pages, page, dtype=torch.bool)
    for b, (n, m) in enumerate(zip(lens, new)):
        for p in range(n):
            if p < sinks or p >= n - m - window:
                seen[int(f.table[b, p // page]), p % page] = True
    for t in (f.cache.key_scales, f.cache.value_scales):
        t.masked_fill_(~seen.to(DEV)[:, None, :, None], 255)
    table = f.table.clone()
    for b in range(len(lens)):
        for c in range(f.cols):
            if table[b, c] < 0 or not bool(seen[int(table[b, c])].any()):
                table[b, c] = -7 if c % 2 else f.cache.pages + c
    got = f.cache.attend(q.to(DEV), table, f.lengths, i32(starts_of(new)), window=window, sinks=sinks)
    check(got, y, terms, BF16, P_CACHE)
    # drafted rows: the last token of sequence 0 is NaN, which only its last row sees
    page_of, token = int(table[0, 699 // page]), 699 % page
    f.cache.value_scales[page_of, :, token] = 255
    f.cache.key_scales[page_of, :, token] = 255
    got = f.cache.attend(q.to(DEV), table, f.lengths, i32(starts_of(new)), window=window, sinks=sinks).cpu()
    assert torch.isnan(got[3]).all()
    rest = [0, 1, 2, 4, 5]
    check(got[rest], y[rest], tuple(t[rest] for t in terms), BF16, P_CACHE)


def test_a_value_of_nan_alone_shows_where_it_is_seen():
    f = Filled([500, 500], 2, 64, 'fp4', 64, seed=25)
    q = rows(torch.Generator().manual_seed(26), 2, 4, 64, BF16).to(DEV)
    clean = f.cache.attend(q, f.table, f.lengths)
    f.cache.value_scales[int(f.table[0, 3]), 1, 9, 1] = 255  # channels 32 .. 63 of kv head 1
    got = f.cache.attend(q, f.table, f.lengths)
    assert torch.isnan(got[0, 2:, 32:]).all() and torch.equal(got[0, :2], clean[0, :2])
    assert torch.equal(got[0, 2:, :32], clean[0, 2:, :32]) and torch.equal(got[1], clean[1])


def test_rows_behind_the_last_cached_sequence():
    f = Filled([100, 30], 1, 64, 'fp4', 16, seed=27)
    q = rows(torch.Generator().manual_seed(28), 9, 2, 64, BF16).to(DEV)
    st = i32([1, 4, 6])
    got = f.cache.attend(q, f.table, f.lengths, st)
    assert not got[:1].any() and not got[6:].any() and bool(got[1:6].any(-1).all())
    out = torch.full_like(got, 3.0)
    assert f.cache.attend(q, f.table, f.lengths, st, out=out) is out
    assert (out[:1] == 3).all() and (out[6:] == 3).all() and torch.equal(out[1:6], got[1:6])


def test_far_pages():
    """Slots past 2^31 bytes of codes: the last pages of a large cache."""
    kv, dim, page = 8, 64, 256
    pages = 2 ** 31 // (kv * page * dim) + 40
    cache = KVCache.zeros(pages, kv, dim, page, 'fp8')
    g = torch.Generator().manual_seed(29)
    n = 600
    k, v = rows(g, n, kv, dim, BF16), rows(g, n, kv, dim, BF16)
    table = i32([[pages - 1, pages - 3, pages - 2]])
    cache.write(k.to(DEV), v.to(DEV), table, i32([n]), i32([0, n]))
    q = rows(g, 1, kv, dim, BF16)
    hk, hv = plain.quantise(k, 'fp8')[2], plain.quantise(v, 'fp8')[2]
    y, terms = plain.attend(q, hk, hv, torch.tensor([n - 1]), None, 0)
    check(cache.attend(q.to(DEV), table, i32([n])), y, terms, BF16, P_CACHE)
    got = cache.read(table, i32([n]), i32([0, n]), rows=n, dtype=F32)
    assert torch.equal(got[0].cpu(), hk.float()) and torch.equal(got[1].cpu(), hv.float())
    assert not cache.keys[:40].any()


def test_last_positions():
    """Positions from 2^31 - 256 on are bad places to all three, whatever the table names for them; the ones in front are not."""
    cache = KVCache.zeros(4, kv_heads=1, dim=64, page_size=256, format='fp8')
    table = torch.zeros(1, 2 ** 23, device=DEV, dtype=torch.int32)  # every position's page is page 0, but the last three
    last = 2 ** 31 - 256
    table[0, -2], table[0, -1] = 1, 2
    x = torch.full((3, 1, 64), 2., device=DEV, dtype=BF16)
    cache.write(x, x, table, i32([last + 2]), i32([0, 3]))  # the last position in front, and two behind
    assert cache.values[1, 0, 255].all() and not cache.values[2].any()
    k, v = cache.read(table, i32([last + 2]), i32([0, 3]), rows=3)
    assert torch.equal(v[0], x[0]) and torch.isnan(v[1:]).all() and torch.isnan(k[1:]).all()
    y = cache.attend(x, table, i32([last + 2]), i32([0, 3]), window=0)
    assert torch.equal(y[0], x[0]) and torch.isnan(y[1:]).all()


def test_more_rows_than_a_call_takes_are_refused():
    cache = KVCache.zeros(1, kv_heads=1, page_size=16)
    x = torch.zeros(1, 1, 64, device=DEV, dtype=BF16).expand(2 ** 31, 1, 64)
    table, lengths, st = torch.zeros(1, 1, device=DEV, dtype=torch.int32), i32([5]), i32([0, 2])
    for call in (lambda: ops.sink_attention(x, x, x, st), lambda: ops.sink_attention(*[x.unsqueeze(0)] * 3),
                 lambda: cache.write(x, x, table, lengths, st), lambda: cache.attend(x, table, lengths, st),
                 lambda: cache.read(table, lengths, st, rows=2 ** 31), lambda: cache.read(table, lengths, st, rows=-1)):
        with pytest.raises(ValueError, match='rows must lie'):
            call()


def test_cache_types_and_shapes_are_refused():
    cache = KVCache.zeros(4, 2, 64, 16, 'fp4')
    x = torch.zeros(3, 2, 64, device=DEV, dtype=BF16)
    table, lengths = i32([[0], [1], [2]]), i32([1, 1, 1])
    for k, v, t, ln, s in ((x, x.half(), table, lengths, None), (x.double(), x.double(), table, lengths, None),
                           (x[:, :1], x[:, :1], table, lengths, None), (x, x[:2], table, lengths, None),
                           (x, x, table.long(), lengths, None), (x, x, table, lengths.long(), None),
                           (x, x, table, lengths[:2], None), (x, x, table[:2], lengths[:2], None), (x, x, table[0], lengths, None),
                           (x, x, table, lengths, i32([0, 3])), (x, x, table.cpu(), lengths, None), (x.cpu(), x, table, lengths, None),
                           (x, x, i32([[0, 1, 2]]).t().expand(-1, 2).contiguous().t().contiguous().t(), lengths, None)):
        with pytest.raises((ValueError, TypeError)):
            cache.write(k, v, t, ln, s)
    for q in (x.float(), x[..., :32], x[:, :1], torch.zeros(3, 3, 64, device=DEV, dtype=BF16)):
        with pytest.raises((ValueError, TypeError)):
            cache.attend(q, table, lengths)
    with pytest.raises(ValueError, match='rows'):
        cache.read(table, lengths, i32([0, 1, 2, 3]))
    with pytest.raises(TypeError):
        cache.read(table, lengths, dtype=torch.float64)
    with pytest.raises(RuntimeError, match='no backward'):
        cache.write(x.float().requires_grad_(), x.float(), table, lengths)
    k, s = cache.keys, cache.key_scales
    for bad in ((k.float(), s, k, s), (k[:3], s, k, s), (k, s[..., :1].contiguous(), k, s), (k, s, k[..., :16].contiguous(), s),
                (k.transpose(0, 1), s, k, s), (k[:, :, :8].contiguous(), s[:, :, :8].contiguous()) * 2, (k[:0], s[:0]) * 2):
        with pytest.raises(ValueError):
            KVCache(*bad)


# ------------------------------------------------------------------ together


def test_a_prompt_and_its_steps_together():
    """A prompt's attention, its cache, then decoding steps and a drafted block, as a server runs them: every answer against the
    64-bit form over the tokens so far."""
    g = torch.Generator().manual_seed(31)
    H, dim, page, window, sinks = 8, 64, 16, 48, 4
    lens, steps, draft = [37, 1, 90], 20, 4
    cols = -(-(max(lens) + steps + draft) // page)
    cache = KVCache.zeros(3 * cols, H, dim, page, 'fp8')
    table = torch.randperm(3 * cols, generator=g).view(3, cols).to(torch.int32).to(DEV)
    lengths = i32(lens)
    q, k, v = (rows(g, sum(lens), H, dim, BF16) for _ in range(3))
    y, terms = prompt_reference(q, k, v, lens, window, sinks)
    st = i32(starts_of(lens))
    check(ops.sink_attention(q.to(DEV), k.to(DEV), v.to(DEV), st, window=window, sinks=sinks), y, terms, BF16, BF16)
    cache.write(k.to(DEV), v.to(DEV), table, lengths, st)
    held = [[plain.quantise(x[s:s + n], 'fp8')[2] for x in (k, v)] for s, n in zip(starts_of(lens), lens)]
    for step in range(steps + 1):
        m = draft if step == steps else 1
        q, k, v = (rows(g, 3 * m, H, dim, BF16) for _ in range(3))
        lengths += m
        st = None if m == 1 else i32([0, m, 2 * m, 3 * m])
        cache.write(k.to(DEV), v.to(DEV), table, lengths, st)
        got = cache.attend(q.to(DEV), table, lengths, st, window=window, sinks=sinks)
        for b in range(3):
            held[b] = [torch.cat((h, plain.quantise(x[b * m:b * m + m], 'fp8')[2])) for h, x in zip(held[b], (k, v))]
            n = len(held[b][0])
            y, terms = plain.attend(q[b * m:b * m + m], *held[b], torch.arange(n - m, n), window, sinks)
            check(got[b * m:b * m + m], y, terms, BF16, P_CACHE, (step, b))


def test_steps_replay_from_graphs():
    """A step captured once and replayed with new rows, other lengths and eager work between: every replay has the eager bits. Two
    graphs of different steps do not disturb each other."""
    f = Filled([1000, 300, 70], 4, 64, 'fp4', 64, seed=41)
    g = torch.Generator().manual_seed(42)
    q, k, v = (rows(g, 3, 4, 64, BF16).to(DEV) for _ in range(3))
    lengths = f.lengths.clone()
    x = torch.zeros(200, 4, 64, device=DEV, dtype=BF16)
    st = i32([0, 120, 200])

    def step(window):
        f.cache.write(k, v, f.table, lengths)
        return f.cache.attend(q, f.table, lengths, window=window, sinks=2), f.cache.read(f.table, lengths)[0], \
            ops.sink_attention(x, x, x, st, window=window)

    step(None), step(90)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for window in (None, 90):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(window))
        graphs.append(graph)
    for r in range(4):
        for t in (q, k, v):
            t.copy_(rows(g, 3, 4, 64, BF16))
        x.copy_(rows(g, 200, 4, 64, BF16))
        lengths.copy_(i32([1000 - 250 * r, 300 - r, 70 - 20 * r]))
        for graph in graphs:
            graph.replay()
        for out, window in zip(outs, (None, 90)):
            for a, b in zip(out, step(window)):
                assert torch.equal(a, b), (r, window)
        torch.cuda.synchronize()


def test_sequences_that_share_one_table_row():
    """A table expanded from one row, and lengths within it."""
    f = Filled([400], 2, 64, 'fp4', 16, seed=43)
    q = rows(torch.Generator().manual_seed(44), 3, 4, 64, BF16)
    lens = [400, 17, 250]
    got = f.cache.attend(q.to(DEV), f.table.expand(3, -1), i32(lens))
    for b, n in enumerate(lens):
        y, terms = plain.attend(q[b:b + 1], *f.held[0], torch.tensor([n - 1]), None, 0)
        check(got[b:b + 1], y, terms, BF16, P_CACHE)
    k, _ = f.cache.read(f.table.expand(3, -1), i32(lens), dtype=F32)
    assert torch.equal(k.cpu(), torch.stack([f.held[0][0][n - 1] for n in lens]).float())


def test_starts_that_decrease_compute_nothing_out_of_range():
    """Starts are the caller's to keep; wrong ones leave rows unwritten, and nothing else is touched."""
    f = Filled([300, 200], 2, 64, 'fp4', 64, seed=45)
    q = rows(torch.Generator().manual_seed(46), 40, 4, 64, BF16).to(DEV)
    bad = i32([0, 40, 0, 40, 7])
    table, lens = f.table[[0, 1, 0, 1]].contiguous(), i32([300, 200, 300, 200])
    out = torch.full_like(q, 5.0)
    f.cache.attend(q, table, lens, bad, out=out)
    ops.sink_attention(q, q[:, :2], q[:, :2], bad, out=out)
    wide = torch.zeros(2, 5000, dtype=torch.int32, device=DEV)  # a long table: the rows are shared out
    f.cache.attend(q, wide, i32([300, 200]), i32([0, 40, 3]), out=out)
    f.cache.read(table, lens, bad, rows=40)
    torch.cuda.synchronize()


def test_another_stream():
    f = Filled([500, 40], 2, 64, 'fp4', 64, seed=51)
    q = rows(torch.Generator().manual_seed(52), 2, 4, 64, BF16).to(DEV)
    want = f.cache.attend(q, f.table, f.lengths)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = f.cache.attend(q, f.table, f.lengths)
        got2 = ops.sink_attention(got, got[:, :2], got[:, :2], i32([0, 2]))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and torch.equal(got2, ops.sink_attention(want, want[:, :2], want[:, :2], i32([0, 2])))


def test_calls_give_the_same_bits():
    f = Filled([5000, 4000, 100], 8, 64, 'fp4', 64, seed=61)
    q = rows(torch.Generator().manual_seed(62), 3, 8, 64, BF16).to(DEV)
    a = f.cache.attend(q, f.table, f.lengths)
    for _ in range(3):
        assert torch.equal(f.cache.attend(q, f.table, f.lengths), a)
