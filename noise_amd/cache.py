"""A paged key / value cache in microscaled floating point on the HIP kernels: rows quantised as they are written, read back,
and attended to (noise_cache_write, noise_cache_read, noise_cache_attend of include/noise_hip.h).

The format is the microscaling one that gfx950 converts in hardware: every 32 channels of a head share a power-of-two scale of
one byte, the codes are e2m1 ('fp4', 4.25 bits a channel) or e4m3 ('fp8', 8.25 bits).

A call names its rows by three int32 tensors on the GPU: `table` [sequences, pages of a sequence], the page of each position of
each sequence; `lengths` [sequences], the tokens that each sequence holds, the call's own included; `starts` [sequences + 1],
the rows of each sequence in the packed tensors, nondecreasing (None: one row each). The m rows of sequence b sit at its newest positions,
lengths[b] - m .. lengths[b] - 1. One decoding step is

    lengths += 1
    cache.write(k, v, table, lengths)
    y = cache.attend(q, table, lengths)

Nothing is copied to the host. Rows of no sequence, and rows at negative positions, are at no place: they are not written, and
read back as zeros. A page outside the cache or a position past the table is a bad place: not written, and NaN to whoever reads
or sees it. Forward only.
"""
import ctypes

import torch

from . import _lib
from .ops import ROW_TYPES, _ptr, heads_rows, launch, mask_args, no_grad_rows, one_device, output_rows, row_count, sequence_starts

FORMATS = {'fp4': _lib.CACHE_FP4, 'fp8': _lib.CACHE_FP8}


class KVCache:
    """The cache's four tensors, uint8 on the GPU and contiguous: keys and values [pages, kv_heads, page_size, dim / 2 ('fp4') or
    dim ('fp8')] codes, key_scales and value_scales [pages, kv_heads, page_size, dim / 32]. dim is 64 or 128, page_size a
    power of two from 16 to 256. They are the caller's (KVCache.zeros allocates them) and are kept, not copied."""

    def __init__(self, keys, key_scales, values, value_scales):
        self.device = one_device(keys, key_scales, values, value_scales)
        for name, t, like, align in (('keys', keys, keys, 16), ('values', values, keys, 16),
                                     ('key_scales', key_scales, key_scales, 4), ('value_scales', value_scales, key_scales, 4)):
            if t.dtype != torch.uint8 or t.dim() != 4 or not t.is_contiguous() or t.shape != like.shape or t.data_ptr() % align:
                raise ValueError(f'{name} must be a contiguous 4-D uint8 tensor of shape {tuple(like.shape)}, {align}-byte aligned')
        self.pages, self.kv_heads, self.page_size, width = keys.shape
        self.dim = 32 * key_scales.shape[3]
        if key_scales.shape[:3] != keys.shape[:3] or self.dim not in (64, 128) or width not in (self.dim // 2, self.dim):
            raise ValueError('scales must be [pages, kv_heads, page_size, dim / 32] beside codes of dim / 2 or dim bytes, dim 64 '
                             f'or 128; got {tuple(key_scales.shape)} and {tuple(keys.shape)}')
        if not 0 < self.pages < 2 ** 31 or not 0 < self.kv_heads <= 1024:
            raise ValueError(f'the cache needs pages and 1 to 1024 kv heads, got {self.pages} and {self.kv_heads}')
        if self.page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f'page_size must be 16, 32, 64, 128 or 256, got {self.page_size}')
        self.format = 'fp4' if width == self.dim // 2 else 'fp8'
        self.keys, self.key_scales, self.values, self.value_scales = keys, key_scales, values, value_scales
        self._desc = _lib.Cache(keys.data_ptr(), key_scales.data_ptr(), values.data_ptr(), value_scales.data_ptr(), self.pages,
                                self.page_size, self.kv_heads, self.dim, FORMATS[self.format])
        self._ptr = ctypes.addressof(self._desc)
        self._sizes = {}  # attend's workspace bytes by the shape of a call

    @classmethod
    def zeros(cls, pages, kv_heads=8, dim=64, page_size=64, format='fp4', device='cuda'):
        """An empty cache of `pages` pages."""
        if format not in FORMATS:
            raise ValueError(f'format must be one of {tuple(FORMATS)}, got {format!r}')
        width = dim // 2 if format == 'fp4' else dim
        t = [torch.zeros(pages, kv_heads, page_size, n, dtype=torch.uint8, device=device) for n in (width, dim // 32) * 2]
        return cls(*t)

    def _beside(self, *tensors):
        """Checks that all are on the cache's device."""
        for t in tensors:
            if t.device != self.device:
                one_device(self.keys, t)

    def _sequences(self, table, lengths, starts, rows):
        """noise_sequences_t of a call's tensors (kept alive by the caller until the call is enqueued)."""
        row_count(rows)
        self._beside(table, lengths)
        dims = table.shape
        if table.dtype != torch.int32 or len(dims) != 2 or (dims[1] > 1 and table.stride(1) != 1):
            raise ValueError('table must be an int32 tensor [sequences, pages of a sequence] with contiguous rows')
        n, pages = dims
        if lengths.dtype != torch.int32 or lengths.shape != (n,) or not lengths.is_contiguous():
            raise ValueError(f'lengths must be a contiguous int32 vector of {n} entries')
        if starts is None:
            if rows != n:
                raise ValueError(f'{rows} rows of {n} sequences need starts')
        elif sequence_starts(starts, self.device) != n:
            raise ValueError(f'starts must have {n + 1} entries')
        return _lib.Sequences(table.data_ptr(), table.stride(0) if n > 1 else 0, pages, lengths.data_ptr(), _ptr(starts), n, rows)

    def write(self, k, v, table, lengths, starts=None):
        """Quantises the rows k and v [n, kv_heads, dim] (bf16, fp16 or fp32, any strides) into their places. The places of one
        call must be distinct: two sequences may share pages that neither writes."""
        no_grad_rows(k, v)
        self._beside(k, v)
        if k.dtype not in ROW_TYPES or v.dtype != k.dtype:
            raise TypeError(f'k and v must be bfloat16, float16 or float32 alike, got {k.dtype} and {v.dtype}')
        if len(k.shape) != 3 or k.shape[1:] != (self.kv_heads, self.dim) or v.shape != k.shape:
            raise ValueError(f'k and v must be [n, {self.kv_heads}, {self.dim}], got {tuple(k.shape)} and {tuple(v.shape)}')
        seqs = self._sequences(table, lengths, starts, k.shape[0])
        if not seqs.rows or not seqs.sequences:
            return
        k, kp, kl, kh = heads_rows(k)
        v, vp, vl, vh = heads_rows(v)
        launch(self.device, 'noise_cache_write', self._ptr, ctypes.addressof(seqs), kp, kl, kh, vp, vl, vh, ROW_TYPES[k.dtype])

    def read(self, table, lengths, starts=None, rows=None, dtype=torch.bfloat16):
        """(k, v) [rows, kv_heads, dim]: the cached values at the rows' places, rounded to dtype (bf16, fp16 or fp32). With starts,
        `rows` is their number (starts' last entry, which only the GPU holds); the whole of each sequence is read with starts the
        running sum of lengths."""
        if dtype not in ROW_TYPES:
            raise TypeError(f'dtype must be bfloat16, float16 or float32, got {dtype}')
        if rows is None:
            if starts is not None:
                raise ValueError('rows must be given with starts')
            rows = table.shape[0]
        seqs = self._sequences(table, lengths, starts, rows)
        shape = (rows, self.kv_heads, self.dim)
        if not seqs.sequences:
            return torch.zeros(shape, device=self.device, dtype=dtype), torch.zeros(shape, device=self.device, dtype=dtype)
        k = torch.empty(shape, device=self.device, dtype=dtype)
        v = torch.empty_like(k)
        if rows:
            launch(self.device, 'noise_cache_read', self._ptr, ctypes.addressof(seqs), k.data_ptr(), v.data_ptr(),
                   ROW_TYPES[dtype])
        return k, v

    def attend(self, q, table, lengths, starts=None, window=None, sinks=0, scale=None, out=None):
        """Attention of the rows' queries q [n, heads, dim] (bf16 or fp16, heads a multiple of kv_heads) over the cached keys and
        values of their sequences: a query at position s sees the keys j <= s with s - j <= window (None: all) or j < sinks.
        Masks, scale, zero rows and `out` as in noise_amd.ops.sink_attention; a row that sees a bad place is NaN."""
        no_grad_rows(q)
        self._beside(q)
        if q.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f'q must be bfloat16 or float16, got {q.dtype}')
        dims = q.shape
        if len(dims) != 3 or dims[2] != self.dim or dims[1] == 0 or dims[1] % self.kv_heads or dims[1] > 1024:
            raise ValueError(f'q must be [n, heads, {self.dim}] with heads (at most 1024) a multiple of {self.kv_heads}, got '
                             f'{tuple(dims)}')
        window, sinks, scale = mask_args(window, sinks, scale, self.dim)
        rows, heads, _ = dims
        seqs = self._sequences(table, lengths, starts, rows)
        y, fill = output_rows(out, q, self.device)
        if not rows:
            return y
        if not seqs.sequences:
            return y.zero_() if fill else y
        q, qp, ql, qh = heads_rows(q)
        call = ctypes.addressof(seqs)
        shape = (seqs.sequences, rows, seqs.table_pages, starts is None, heads, q.dtype)
        size = self._sizes.get(shape)
        if size is None:
            if len(self._sizes) >= 256:
                self._sizes.clear()
            size = self._sizes[shape] = _lib.size_query('noise_cache_attend_workspace_size', self._ptr, call, heads,
                                                            ROW_TYPES[q.dtype])
        ws = torch.empty(size, device=self.device, dtype=torch.uint8) if size else None
        launch(self.device, 'noise_cache_attend', self._ptr, call, qp, ql, qh, ROW_TYPES[q.dtype], heads, window, sinks, scale,
               y.data_ptr(), fill, _ptr(ws), size)
        return y
