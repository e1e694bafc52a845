"""ctypes binding of the dense operators' C ABI (include/tinydeform_dense.h) and their tensor-level host entries.

attn_forward / attn_backward and layer_norm_forward / layer_norm_backward take torch tensors on a HIP device, check them
(RuntimeError), allocate outputs and workspaces with torch.empty on the caching allocator, and launch on the current
stream of the tensors' device, as the entries in _native.py do. Nothing here computes on the CPU.
"""

import ctypes
import math
import struct

import torch

from . import _native
from ._native import DTYPE_CODES, INT32_MAX, _check, _ptr, _require, _stream, acc_dtype

MAX_HEAD_DIM = 256        # TD_ATTN_MAX_HEAD_DIM
MAX_NORM_CHANNELS = 16384  # TD_NORM_MAX_CHANNELS
MAX_ATTN_ROWS = INT32_MAX - 1023
MASK_NONE, MASK_BYTES, MASK_FLOAT = 0, 1, 2  # TD_MASK_*

_i64, _vp, _int = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int
# every symbol include/tinydeform_dense.h declares, with its ctypes signature
SIGNATURES = {
    'td_attn_forward_workspace': (_i64, [_vp]),
    'td_attn_forward': (_int, [_vp, _vp, _i64, _vp]),
    'td_attn_backward_workspace': (_i64, [_vp]),
    'td_attn_backward': (_int, [_vp] * 6 + [_i64, _vp]),
    'td_layer_norm_forward': (_int, [_int] + [_vp] * 6 + [_i64, _i64, ctypes.c_double, _vp]),
    'td_layer_norm_backward_workspace': (_i64, [_int, _i64, _i64]),
    'td_layer_norm_backward': (_int, [_int] + [_vp] * 8 + [_i64, _i64, _vp, _i64, _vp]),
}
# td_attn_args: dtype, mask_type, causal, reserved; B, Q, K, H, Hk, D; scale; query, key, value; their strides; mask and
# its strides; key_padding, out, stats, out_low
ATTN_ARGS = struct.Struct('4i6qd3Q9qQ3q4Q')


def _declare(lib):
    for name, (res, args) in SIGNATURES.items():
        try:
            fn = getattr(lib, name)
        except AttributeError:
            _native.load_error = f'{_native.LIB_PATH} has no {name}: it predates these sources (rebuild it)'
            return False
        fn.restype = res
        fn.argtypes = args
    return True


if _native.lib is not None and not _declare(_native.lib):
    _native.lib = None


def check_attn(query, key, value, attn_mask=None, key_padding_mask=None, scale=None, require_gpu=True):
    """Checks of ma_attn's arguments; returns the scale, the mask with its type and its strides by batch, head and query
    (0 where shared), and the padding mask."""
    if require_gpu and not query.is_cuda:
        raise RuntimeError('inputs must be GPU tensors')
    if query.dim() != 4:
        raise RuntimeError('query must be [B, Q, H, D]')
    if key.dim() != 4 or value.shape != key.shape:
        raise RuntimeError('key and value must be [B, K, Hk, D]')
    B, Q, H, D = query.shape
    Bk, K, Hk, Dk = key.shape
    if Bk != B:
        raise RuntimeError('batch size mismatch')
    if H <= 0 or Hk <= 0:
        raise RuntimeError('need at least one head')
    if H % Hk != 0:
        raise RuntimeError('the heads of key and value must divide the heads of query')
    if Dk != D:
        raise RuntimeError('key and value must have the head dim of query')
    if not 1 <= D <= MAX_HEAD_DIM:
        raise RuntimeError(f'head dim must be from 1 to {MAX_HEAD_DIM}')
    dtype, device = query.dtype, query.device
    if dtype not in DTYPE_CODES:
        raise RuntimeError(f'unsupported dtype {dtype}')
    if key.dtype != dtype or value.dtype != dtype:
        raise RuntimeError('all float tensors must have the same dtype')
    if key.device != device or value.device != device:
        raise RuntimeError('all tensors must be on the same device')
    if max(Q, K, B * Q * H, B * K * Hk) > MAX_ATTN_ROWS:
        raise RuntimeError('too many (batch, token, head) rows')
    if scale is None:
        scale = D ** -0.5
    elif not (scale > 0 and math.isfinite(scale)):
        raise RuntimeError('scale must be positive and finite')
    kind, strides = MASK_NONE, (0, 0, 0)
    if attn_mask is not None:
        shape = attn_mask.shape
        lead = (1,) * (4 - len(shape)) + tuple(shape)
        if len(shape) not in (2, 4) or lead[3] != K or lead[0] not in (1, B) or lead[1] not in (1, H) \
                or lead[2] not in (1, Q):
            raise RuntimeError('attn_mask must be [Q, K] or [B, H, Q, K] (1 for a shared batch, head or query)')
        if attn_mask.device != device:
            raise RuntimeError('all tensors must be on the same device')
        if attn_mask.dtype in (torch.bool, torch.uint8):
            kind = MASK_BYTES
        elif attn_mask.dtype == dtype:
            kind = MASK_FLOAT
        else:
            raise RuntimeError('attn_mask must be bool (True: may not attend) or have the dtype of query (added)')
        if attn_mask.requires_grad and torch.is_grad_enabled():
            raise RuntimeError('attn_mask has no gradient: pass attn_mask.detach()')
        if K > 1 and attn_mask.stride(-1) != 1:
            attn_mask = attn_mask.contiguous()
        st = (0,) * (4 - len(shape)) + attn_mask.stride()
        strides = tuple(0 if lead[i] == 1 else st[i] for i in range(3))
    if key_padding_mask is not None:
        if key_padding_mask.dtype not in (torch.bool, torch.uint8) or key_padding_mask.shape != (B, K):
            raise RuntimeError('key_padding_mask must be bool [B, K] (True: padded key)')
        if key_padding_mask.device != device:
            raise RuntimeError('all tensors must be on the same device')
        key_padding_mask = key_padding_mask.contiguous()
    return scale, attn_mask, kind, strides, key_padding_mask


def _rows(t):
    """t with its last dimension contiguous"""
    return t if t.stride(3) == 1 or t.size(3) == 1 else t.contiguous()


def _pack(query, key, value, mask, kind, mask_strides, padding, scale, causal, out, stats, low=None):
    B, Q, H, D = query.shape
    qs, ks, vs = query.stride(), key.stride(), value.stride()
    return ATTN_ARGS.pack(DTYPE_CODES[query.dtype], kind, 1 if causal else 0, 0, B, Q, key.size(1), H, key.size(2), D,
                          scale, query.data_ptr(), key.data_ptr(), value.data_ptr(), qs[0], qs[1], qs[2], ks[0], ks[1],
                          ks[2], vs[0], vs[1], vs[2], 0 if mask is None else mask.data_ptr(), *mask_strides,
                          0 if padding is None else padding.data_ptr(), out.data_ptr(),
                          0 if stats is None else stats.data_ptr(), 0 if low is None else low.data_ptr())


def _workspace(need, device):
    if need < 0:
        _check(need)
    return torch.empty((need,), dtype=torch.uint8, device=device) if need > 0 else None


def attn_forward(query, key, value, attn_mask=None, key_padding_mask=None, scale=None, causal=False, train=False):
    """Attention among tokens (td_attn_forward): out [B, Q, H * D], and with train what attn_backward takes: the tensors
    and the plain values of the call (else None, None)."""
    lib = _require()
    scale, mask, kind, strides, pad = check_attn(query, key, value, attn_mask, key_padding_mask, scale)
    q, k, v = _rows(query), _rows(key), _rows(value)
    B, Q, H, D = q.shape
    dev, dtype = q.device, q.dtype
    out = torch.empty((B, Q, H * D), dtype=dtype, device=dev)
    stats = low = None
    if train:
        stats = torch.empty((B, H, Q, 2), dtype=acc_dtype(dtype), device=dev)
        if dtype in (torch.float16, torch.bfloat16):  # what rounding took from out: grad_out . out needs it
            low = torch.empty_like(out)
    if B * Q > 0:
        args = _pack(q, k, v, mask, kind, strides, pad, scale, causal, out, stats, low)
        need = lib.td_attn_forward_workspace(args)
        ws = _workspace(need, dev)
        _check(lib.td_attn_forward(args, _ptr(ws), need, _stream(dev)))
    if not train:
        return out, None, None
    return out, (q, k, v, mask, pad, out, stats, low), (kind, strides, scale, causal)


def attn_backward(tensors, values, grad_out, need_query=True, need_key_value=True):
    """Gradients of attn_forward (td_attn_backward) from what it gave for training: grad_query like query, grad_key and
    grad_value like key; None for those not needed."""
    lib = _require()
    q, k, v, mask, pad, out, stats, low = tensors
    kind, strides, scale, causal = values
    if grad_out.shape != out.shape or grad_out.dtype != q.dtype or grad_out.device != q.device:
        raise RuntimeError('grad_out must be [B, Q, H * D] like the forward output')
    dev, go = q.device, grad_out.contiguous()
    dq = torch.empty_like(q, memory_format=torch.contiguous_format) if need_query else None
    dk = dv = None
    if need_key_value:
        dk = torch.empty_like(k, memory_format=torch.contiguous_format)
        dv = torch.empty_like(k, memory_format=torch.contiguous_format)
    if q.size(0) * (q.size(1) + k.size(1)) > 0:
        args = _pack(q, k, v, mask, kind, strides, pad, scale, causal, out, stats, low)
        need = lib.td_attn_backward_workspace(args)
        ws = _workspace(need, dev)
        _check(lib.td_attn_backward(args, go.data_ptr(), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), need, _stream(dev)))
    return dq, dk, dv


def check_norm(x, weight, bias, residual, require_gpu=True):
    """Checks of ma_layer_norm's arguments; returns rows and C."""
    if require_gpu and not x.is_cuda:
        raise RuntimeError('inputs must be GPU tensors')
    if x.dim() < 1:
        raise RuntimeError('x must be [..., C]')
    C = x.size(-1)
    if not 1 <= C <= MAX_NORM_CHANNELS:
        raise RuntimeError(f'channels must be from 1 to {MAX_NORM_CHANNELS}')
    if x.dtype not in DTYPE_CODES:
        raise RuntimeError(f'unsupported dtype {x.dtype}')
    for t, name in ((weight, 'weight'), (bias, 'bias')):
        if t is not None and t.shape != (C,):
            raise RuntimeError(f'{name} must be [C] with C = x.size(-1)')
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError('residual must have the shape of x')
    for t in (weight, bias, residual):
        if t is not None:
            if t.dtype != x.dtype:
                raise RuntimeError('all float tensors must have the same dtype')
            if t.device != x.device:
                raise RuntimeError('all tensors must be on the same device')
    rows = x.numel() // C
    if rows > INT32_MAX:
        raise RuntimeError('too many rows')
    return rows, C


def _contiguous(t):
    return None if t is None else t.contiguous()


def layer_norm_forward(x, weight, bias, residual=None, eps=1e-5, train=False):
    """Layer norm of x (+ residual) (td_layer_norm_forward): out like x, and with train the tensors that
    layer_norm_backward takes (else None)."""
    lib = _require()
    rows, C = check_norm(x, weight, bias, residual)
    if not (eps >= 0 and math.isfinite(eps)):
        raise RuntimeError('eps must be non-negative and finite')
    dev = x.device
    x, weight, bias, residual = x.contiguous(), _contiguous(weight), _contiguous(bias), _contiguous(residual)
    out = torch.empty_like(x)
    stats = torch.empty((rows, 2), dtype=acc_dtype(x.dtype), device=dev) if train else None
    if rows > 0:
        _check(lib.td_layer_norm_forward(DTYPE_CODES[x.dtype], x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(bias),
                                         out.data_ptr(), _ptr(stats), rows, C, eps, _stream(dev)))
    return out, (x, weight, residual, stats) if train else None


def layer_norm_backward(tensors, grad_out, need_weight=True, need_bias=True):
    """Gradients of layer_norm_forward (td_layer_norm_backward) from what it gave for training: grad_x like x (the
    residual's too), grad_weight and grad_bias [C], None where not needed."""
    lib = _require()
    x, weight, residual, stats = tensors
    if grad_out.shape != x.shape or grad_out.dtype != x.dtype or grad_out.device != x.device:
        raise RuntimeError('grad_out must be like the forward output')
    rows, C = stats.size(0), x.size(-1)
    dev, dtype, go = x.device, x.dtype, grad_out.contiguous()
    code = DTYPE_CODES[dtype]
    dx = torch.empty_like(x)
    dw = torch.empty((C,), dtype=dtype, device=dev) if need_weight else None
    db = torch.empty((C,), dtype=dtype, device=dev) if need_bias else None
    need = lib.td_layer_norm_backward_workspace(code, rows, C) if need_weight or need_bias else 0
    ws = _workspace(need, dev)
    _check(lib.td_layer_norm_backward(code, x.data_ptr(), _ptr(residual), _ptr(weight), stats.data_ptr(), go.data_ptr(),
                                      dx.data_ptr(), _ptr(dw), _ptr(db), rows, C, _ptr(ws), need, _stream(dev)))
    return dx, dw, db
