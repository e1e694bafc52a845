"""What a DETR-style layer runs beside deformable attention: attention among its tokens and the norm after a sublayer,
each for inference and for training. No counterpart in the reference, which is the deformable operator alone."""

import torch
from torch.autograd.function import once_differentiable

from . import _dense, _native
from .reference import ma_attn_reference, ma_layer_norm_reference


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _on_device(t, fn, *args):
    if t.device.index is None or t.device.index == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(t.device):
        return fn(*args)


def _once(backward):
    """A backward pass that can be run once: once_differentiable refuses a second derivative, but costs 5 us of host time
    that a step without one need not wait for."""
    once = once_differentiable(backward)

    def run(ctx, grad_out):
        return once(ctx, grad_out) if torch.is_grad_enabled() else backward(ctx, grad_out)
    return run


def ma_attn(query, key, value, attn_mask=None, key_padding_mask=None, scale=None, causal=False):
    """Attention among tokens: softmax(scale * query key^T + mask) value for each head; [B, Q, H * D].

    query             [B, Q, H, D]
    key, value        [B, K, Hk, D]; Hk divides H, and each key head serves H / Hk heads in a row
    attn_mask         [Q, K] or [B, H, Q, K] (1 for a shared batch, head or query): bool or uint8, True where a query may
                      not attend to a key, or of the inputs' dtype, added to the scaled scores (-inf: may not attend)
    key_padding_mask  bool [B, K], True for padded keys. They count for nothing, whatever they hold
    scale             D ** -0.5 by default; positive
    causal            query i sees the keys j <= i + K - Q only (the last query sees every key)

    A query that is left no key gives 0. Keys and values that only attn_mask or causal hide from some queries have to be
    finite. Any strides with a contiguous last dimension are read in place (slices of a joint projection, transposed
    heads). float32, float16, bfloat16, float64; scores, softmax and sums in float32 (float64 for float64).
    D <= 256. CPU tensors run ma_attn_reference. Inference only: for gradients call ma_attn_train.
    """
    if not query.is_cuda:
        _dense.check_attn(query, key, value, attn_mask, key_padding_mask, scale, require_gpu=False)
        return ma_attn_reference(query, key, value, attn_mask, key_padding_mask, scale, causal)
    _native._require()
    if _needs_grad(query, key, value):
        raise RuntimeError('ma_attn is inference only: run it under torch.no_grad() / torch.inference_mode(), or use '
                           'ma_attn_train for training')
    return _on_device(query, _dense.attn_forward, query, key, value, attn_mask, key_padding_mask, scale, causal)[0]


class _AttnFunction(torch.autograd.Function):
    """Attention among tokens on the library's kernels; the backward recomputes the probabilities from the softmax
    statistics (td_attn_backward)."""

    @staticmethod
    def forward(ctx, query, key, value, attn_mask, key_padding_mask, scale, causal):
        out, tensors, ctx.values = _dense.attn_forward(query, key, value, attn_mask, key_padding_mask, scale, causal,
                                                       train=True)
        ctx.save_for_backward(*tensors)
        return out

    @staticmethod
    @_once
    def backward(ctx, grad_out):
        need = ctx.needs_input_grad
        dq, dk, dv = _dense.attn_backward(ctx.saved_tensors, ctx.values, grad_out, need[0], need[1] or need[2])
        return dq, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def ma_attn_train(query, key, value, attn_mask=None, key_padding_mask=None, scale=None, causal=False):
    """ma_attn with autograd, for training: the same arguments and result, differentiable in query, key and value (not
    in attn_mask). The gradients of a shared key head are summed over its heads; the same on every run (no atomics).
    CPU tensors run ma_attn_reference under PyTorch's autograd."""
    if not query.is_cuda:
        _dense.check_attn(query, key, value, attn_mask, key_padding_mask, scale, require_gpu=False)
        return ma_attn_reference(query, key, value, attn_mask, key_padding_mask, scale, causal)
    _native._require()
    if attn_mask is not None and _needs_grad(attn_mask):  # autograd runs the function itself without gradients
        raise RuntimeError('attn_mask has no gradient: pass attn_mask.detach()')
    return _on_device(query, _AttnFunction.apply, query, key, value, attn_mask, key_padding_mask, scale, causal)


def ma_layer_norm(x, weight=None, bias=None, residual=None, eps=1e-5):
    """Layer norm over the last dimension of x, or of x + residual: the step after a sublayer of a DETR layer.

    x, residual [..., C] (the sum is not rounded before the norm), weight and bias [C] or None, all of one dtype
    (float32, float16, bfloat16, float64); mean and variance in float32 (float64 for float64). C <= 16384.
    CPU tensors run ma_layer_norm_reference. Inference only: for gradients call ma_layer_norm_train.
    """
    if not x.is_cuda:
        _dense.check_norm(x, weight, bias, residual, require_gpu=False)
        return ma_layer_norm_reference(x, weight, bias, residual, eps)
    _native._require()
    if _needs_grad(x, weight, bias, residual):
        raise RuntimeError('ma_layer_norm is inference only: run it under torch.no_grad() / torch.inference_mode(), or '
                           'use ma_layer_norm_train for training')
    return _on_device(x, _dense.layer_norm_forward, x, weight, bias, residual, eps)[0]


class _LayerNormFunction(torch.autograd.Function):
    """Layer norm with a residual on the library's kernels, with gradients for x, the residual, weight and bias."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        out, tensors = _dense.layer_norm_forward(x, weight, bias, residual, eps, train=True)
        ctx.save_for_backward(*tensors)
        return out

    @staticmethod
    @_once
    def backward(ctx, grad_out):
        need = ctx.needs_input_grad
        dx, dw, db = _dense.layer_norm_backward(ctx.saved_tensors, grad_out, need[1], need[2])
        return dx if need[0] else None, dw, db, dx if need[3] else None, None


def ma_layer_norm_train(x, weight=None, bias=None, residual=None, eps=1e-5):
    """ma_layer_norm with autograd, for training: the same arguments and result, differentiable in x, weight, bias and
    residual. The sums over the rows are taken in a fixed order: the same on every run. CPU tensors run
    ma_layer_norm_reference under PyTorch's autograd."""
    if not x.is_cuda:
        _dense.check_norm(x, weight, bias, residual, require_gpu=False)
        return ma_layer_norm_reference(x, weight, bias, residual, eps)
    _native._require()
    return _on_device(x, _LayerNormFunction.apply, x, weight, bias, residual, eps)
