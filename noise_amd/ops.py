"""torch-facing wrappers of the C ABI (device memory and streams come from PyTorch-ROCm).

Each op validates shapes and dtypes on the host, allocates its outputs and workspace with torch, and
enqueues the HIP kernels on torch's current stream. Inputs must already be CUDA tensors: there is no
CPU path.
"""
import math

import torch

from . import _lib


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _need(t, dtype, shape=None, name='tensor'):
    if t.device.type != 'cuda':
        raise ValueError(f'{name} must be a CUDA tensor (no CPU path)')
    if t.dtype != dtype:
        raise TypeError(f'{name} must be {dtype}, got {t.dtype}')
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name} must have shape {tuple(shape)}, got {tuple(t.shape)}')
    if not t.is_contiguous():
        raise ValueError(f'{name} must be contiguous')


def _rows(x, members, T):
    """(ld, member stride) of a bf16 activation [members, T, in] or a shared [T, in]."""
    if x.dim() == 2:
        return x.stride(0), 0
    if x.shape[0] != members or x.shape[1] != T:
        raise ValueError(f'activation must be [members={members}, T={T}, in], got {tuple(x.shape)}')
    return x.stride(1), x.stride(0)


def _dirs(a, members, pair_shift):
    need = (members + (1 << pair_shift) - 1) >> pair_shift
    if a.shape[0] < need:
        raise ValueError(f'need {need} perturbation rows, got {a.shape[0]}')


def lowrank_linear(x, weight, a, b, sign, T=None, pair_shift=0, out=None, accumulate=False, out_dtype=torch.float32):
    """x [members, T, in] (or shared [T, in]) bf16 through weight [out, in] bf16 + sign_p a_p b_p^T.

    Returns fp32 (or bf16) [members, T, out]; with accumulate=True adds into `out` (fp32) in place."""
    members = sign.shape[0]
    T = T or x.shape[-2]
    d_out, d_in = weight.shape
    _need(x, torch.bfloat16, name='x')
    _need(weight, torch.bfloat16, name='weight')
    _need(a, torch.float32, name='a')
    _need(b, torch.float32, name='b')
    _need(sign, torch.float32, name='sign')
    if a.shape[1] != d_out or b.shape[1] != d_in or x.shape[-1] != d_in:
        raise ValueError('rank-1 vectors or activation do not match the weight')
    _dirs(a, members, pair_shift)
    _dirs(b, members, pair_shift)
    ld, mstride = _rows(x, members, T)
    if accumulate:
        if out is None or out.dtype != torch.float32:
            raise ValueError('accumulate needs an fp32 out tensor')
        y32, y16 = out, None
    else:
        y = out if out is not None else torch.empty(members, T, d_out, device=x.device, dtype=out_dtype)
        y32, y16 = (y, None) if y.dtype == torch.float32 else (None, y)
        out = y
    ws_bytes = _lib.size_query('noise_lowrank_linear_workspace_size', members, T)
    ws = torch.empty(ws_bytes, device=x.device, dtype=torch.uint8)
    _lib.call('noise_lowrank_linear', _ptr(x), ld, mstride, _ptr(weight), d_in, d_out, _ptr(a), _ptr(b), _ptr(sign),
              members, T, pair_shift, _ptr(y32), _ptr(y16), int(accumulate), _ptr(ws), ws_bytes, _stream())
    return out


def lowrank_mlp(x, w_fc, w_proj, a_fc, b_fc, a_proj, b_proj, sign, T=None, pair_shift=0, out=None,
                accumulate=False, out_dtype=torch.float32, workspace=None):
    """relu^2 MLP with rank-1 perturbations on both matrices (train/val/eggroll.py:93), per member.

    x: bf16 [members, T, d] or shared [T, d]; w_fc [f, d], w_proj [d, f] bf16 (nn.Linear orientation)."""
    members = sign.shape[0]
    T = T or x.shape[-2]
    f, d = w_fc.shape
    for t, n in ((x, 'x'), (w_fc, 'w_fc'), (w_proj, 'w_proj')):
        _need(t, torch.bfloat16, name=n)
    for t, n in ((a_fc, 'a_fc'), (b_fc, 'b_fc'), (a_proj, 'a_proj'), (b_proj, 'b_proj'), (sign, 'sign')):
        _need(t, torch.float32, name=n)
    if tuple(w_proj.shape) != (d, f) or a_fc.shape[1] != f or b_fc.shape[1] != d or a_proj.shape[1] != d \
            or b_proj.shape[1] != f:
        raise ValueError('MLP weights / rank-1 vectors have inconsistent shapes')
    for t in (a_fc, b_fc, a_proj, b_proj):
        _dirs(t, members, pair_shift)
    ld, mstride = _rows(x, members, T)
    if accumulate:
        if out is None or out.dtype != torch.float32:
            raise ValueError('accumulate needs an fp32 out tensor')
        y32, y16 = out, None
    else:
        y = out if out is not None else torch.empty(members, T, d, device=x.device, dtype=out_dtype)
        y32, y16 = (y, None) if y.dtype == torch.float32 else (None, y)
        out = y
    ws_bytes = _lib.size_query('noise_lowrank_mlp_workspace_size', members, T, d, f)
    if workspace is None or workspace.numel() < ws_bytes:
        workspace = torch.empty(ws_bytes, device=x.device, dtype=torch.uint8)
    _lib.call('noise_lowrank_mlp', _ptr(x), ld, mstride, _ptr(w_fc), _ptr(w_proj), d, f, _ptr(a_fc), _ptr(b_fc),
              _ptr(a_proj), _ptr(b_proj), _ptr(sign), members, T, pair_shift, _ptr(y32), _ptr(y16), int(accumulate),
              _ptr(workspace), ws_bytes, _stream())
    return out


def mlp_workspace_bytes(members, T, d=512, f=2048):
    return _lib.size_query('noise_lowrank_mlp_workspace_size', members, T, d, f)


ROW_TYPES = {torch.bfloat16: _lib.ROWS_BF16, torch.float16: _lib.ROWS_F16, torch.float32: _lib.ROWS_F32}
NO_WINDOW = 2 ** 31 - 1


def launch(dev, name, *args):
    """Calls an entry point on device dev, on its current stream (the last argument)."""
    index = dev.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(dev):
            return launch(dev, name, *args)
    status = getattr(_lib.load(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, name)


def no_grad_rows(*tensors):
    """The serving operators are forward-only: refuse a tensor whose gradient a caller would expect."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError('the serving operators have no backward pass: call them under torch.no_grad() or detach the inputs')


def one_device(*tensors):
    """The CUDA device that all of them are on."""
    dev = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise ValueError('the operands must be CUDA tensors (no CPU path)')
        if t.device != dev:
            raise ValueError(f'the operands are on different devices ({dev} and {t.device})')
    return dev


def row_count(rows):
    """Checks a call's number of packed rows, an int of the entry points."""
    if not 0 <= rows < 2 ** 31:
        raise ValueError(f'rows must lie in [0, 2^31), got {rows}')
    return rows


def heads_rows(t, below=2 ** 63):
    """(tensor to keep alive, pointer, row stride, head stride) of rows [n, heads, dim] as the kernels read them: in place
    where the channels are contiguous, rows and heads start at 16-byte addresses and the row stride is less than `below`, else
    from a contiguous copy."""
    n, heads, dim = t.shape
    p = t.data_ptr()
    if n > 1 and heads > 1 and t.is_contiguous() and not p % 16:
        return t, p, heads * dim, dim
    unit = 16 // t.itemsize
    ld, hs, one = t.stride()
    if n == 1:  # (the stride of a dimension of one entry means nothing)
        ld = 0
    if heads == 1:
        hs = 0
    if one != 1 or ld % unit or hs % unit or p % 16 or ld >= below:
        t = t.clone(memory_format=torch.contiguous_format)
        ld, hs, p = heads * dim, dim, t.data_ptr()
    return t, p, ld, hs


def mask_args(window, sinks, scale, dim):
    """(window, sinks, scale) as the entry points take them."""
    window = NO_WINDOW if window is None else int(window)
    sinks = int(sinks)
    if window < 0 or sinks < 0:
        raise ValueError('window (None for no window) and sinks must be >= 0')
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0 <= scale < math.inf:
        raise ValueError('scale must be finite and >= 0')
    return min(window, NO_WINDOW), min(sinks, NO_WINDOW), scale


def sequence_starts(starts, dev):
    """Checks the packed rows' starts and returns the number of sequences."""
    if starts.dtype != torch.int32 or starts.dim() != 1 or starts.numel() < 1 or not starts.is_contiguous():
        raise ValueError('starts must be a contiguous int32 vector of sequences + 1 entries')
    if starts.device != dev:
        raise ValueError(f'starts must be on {dev}, got {starts.device}')
    return starts.numel() - 1


def output_rows(out, like, dev):
    """The output [n, heads, dim] and whether rows of no sequence are to be zeroed (not in a tensor the caller gave)."""
    if out is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format), 1
    if out.shape != like.shape or out.dtype != like.dtype or out.device != dev or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f'out must be a contiguous {like.dtype} tensor of shape {tuple(like.shape)} beside q, 16-byte aligned')
    no_grad_rows(out)
    return out, 0


def sink_attention(q, k, v, starts=None, window=None, sinks=0, scale=None, out=None):
    """Causal attention of whole sequences with a left window and first tokens that stay visible: a query at position s sees
    the keys j <= s with s - j <= window (None: all of them) or j < sinks.

    q [n, heads, dim], k and v [n, kv_heads, dim] are packed rows of sequences of any lengths, sequence b owning rows
    starts[b] .. starts[b + 1] (int32 on the GPU, nondecreasing); or, without starts, [batch, T, heads, dim] and [batch, T,
    kv_heads, dim]. bf16 or fp16, dim 64 or 128, heads a multiple of kv_heads; any strides (read in place when the channels
    are contiguous and rows and heads are 16-byte aligned). scale defaults to dim ** -0.5. Returns q's shape and type. A
    row that sees no key is zero; what a row does not see takes no part in it, infinities and NaN included. Rows of no
    sequence come back zero, or, in a given `out` (which must not overlap the inputs), stay as they were. Forward only."""
    no_grad_rows(q, k, v)
    dev = one_device(q, k, v)
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f'q, k and v must all be bfloat16 or all float16, got {q.dtype}, {k.dtype}, {v.dtype}')
    qs, ks = q.shape, k.shape
    if len(qs) != (4 if starts is None else 3) or ks != v.shape or ks[:-2] != qs[:-2] or ks[-1] != qs[-1]:
        raise ValueError('q must be [n, heads, dim] and k, v [n, kv_heads, dim] with starts, [batch, T, ...] without; got '
                         f'{tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}')
    *_, heads, dim = qs
    kv = ks[-2]
    if dim not in (64, 128) or kv == 0 or heads == 0 or heads % kv or heads > 1024:
        raise ValueError(f'dim must be 64 or 128 and heads (at most 1024) a multiple of kv_heads: got {heads} x {dim} on {kv}')
    window, sinks, scale = mask_args(window, sinks, scale, dim)
    rows = row_count(qs[0] if starts is not None else qs[0] * qs[1])
    y, fill = output_rows(out, q, dev)
    T = 0
    if starts is None:
        n, T = qs[:2]
        q, k, v = q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1)
    else:
        n = sequence_starts(starts, dev)
    if rows == 0:
        return y
    if n == 0:  # no sequence at all: every row is behind the last one
        return y.zero_() if fill else y
    q, qp, ql, qh = heads_rows(q)
    k, kp, kl, kh = heads_rows(k, 2 ** 23)
    v, vp, vl, vh = heads_rows(v, 2 ** 23)
    launch(dev, 'noise_sink_attention', qp, ql, qh, kp, kl, kh, vp, vl, vh, _ptr(starts), n, rows, T, heads, kv, dim,
           ROW_TYPES[q.dtype], window, sinks, scale, y.data_ptr(), fill)
    return y
