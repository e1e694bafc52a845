"""Inputs of attention and layer norm tests, and the check of results against the float64 oracle (oracle/dense.py) within
bounds that its *_bounds functions derive from the number of roundings."""

import numpy as np
import torch

from oracle import dense

# B, Q, K, H, Hk, D: from one token to several tiles, tile edges, odd and extreme head widths, shared heads
ATTN_SIZES = [
    (1, 1, 1, 1, 1, 32), (2, 1, 77, 4, 4, 32), (1, 300, 300, 8, 8, 32), (2, 33, 64, 3, 3, 32), (1, 64, 63, 2, 2, 32),
    (2, 129, 65, 2, 2, 32), (1, 40, 257, 4, 4, 64), (1, 37, 300, 2, 2, 128), (1, 50, 130, 2, 2, 16),
    (2, 31, 45, 2, 2, 1), (1, 20, 70, 3, 3, 7), (2, 45, 100, 2, 2, 36), (1, 35, 90, 2, 2, 80), (1, 21, 75, 2, 2, 96),
    (1, 40, 70, 1, 1, 129), (1, 33, 150, 2, 2, 256), (2, 1, 1000, 16, 4, 64), (1, 70, 90, 8, 1, 32),
    (2, 43, 52, 6, 2, 40), (3, 2, 200, 12, 4, 32), (1, 7, 2500, 2, 1, 64), (1, 2500, 40, 4, 2, 32), (1, 1300, 70, 3, 1, 128), (1, 40, 1100, 1, 1, 50),
]
MASKS = ['none', 'bool', 'bool4', 'float', 'float4', 'lowest', 'padding', 'causal', 'all']


def randn(g, *shape):
    return torch.randn(*shape, generator=g)


def make_attn(size, dtype, mask='none', seed=0, grad_scale=1.0):
    """(q, k, v, grad_out, keyword arguments) on the CPU. Masks leave some rows empty; padded keys hold NaN and
    infinities."""
    B, Q, K, H, Hk, D = size
    g = torch.Generator().manual_seed(seed)
    q, k, v = randn(g, B, Q, H, D) * 1.5, randn(g, B, K, Hk, D), randn(g, B, K, Hk, D) + 0.2
    go = randn(g, B, Q, H * D) * grad_scale
    q, k, v, go = (t.to(dtype) for t in (q, k, v, go))
    kw = {}

    def some(*shape, p=0.4):
        return torch.rand(*shape, generator=g) < p
    if mask == 'bool':
        kw['attn_mask'] = some(Q, K)
        kw['attn_mask'][Q // 2] = True                       # a row left nothing
    elif mask == 'bool4':
        kw['attn_mask'] = some(B, 1, Q, K).to(torch.uint8) * 3   # any non-zero byte
    elif mask == 'float':
        kw['attn_mask'] = randn(g, Q, K).masked_fill(some(Q, K), float('-inf')).to(dtype)
        kw['attn_mask'][0] = float('-inf')
    elif mask == 'float4':
        kw['attn_mask'] = randn(g, 1, H, Q, K).to(dtype)
    elif mask == 'lowest':                                   # the type's lowest value: a row of it is a uniform row
        kw['attn_mask'] = torch.zeros(Q, K, dtype=dtype).masked_fill(some(Q, K), torch.finfo(dtype).min)
        kw['attn_mask'][Q - 1] = torch.finfo(dtype).min
    if mask in ('padding', 'all'):
        pad = some(B, K)
        pad[-1] = torch.arange(K) >= (K + 1) // 3
        if B > 1:
            pad[0] = True                                    # an image of nothing but padding
        kw['key_padding_mask'] = pad
        k[pad], v[pad] = float('nan'), float('inf')
    if mask in ('causal', 'all'):
        kw['causal'] = True
    if mask == 'all':
        kw['attn_mask'] = some(1, 1, Q, K, p=0.2)
        kw['scale'] = 0.37
    return q, k, v, go, kw


def half_steps(dtype):
    """Half steps of dtype, of its accumulation type, and of P and dS (rounded to dtype where it has 16 bits), and what a
    probability may be off by where it is too small: the smallest normal number (an exponential below it may come out as
    0), and in float16, whose P is held as 2^11 P or more with steps of 2^-24 where it is smallest, half such a step."""
    u = torch.finfo(dtype).eps / 2
    a = u if dtype == torch.float64 else 2.0 ** -24
    low = {torch.float64: 2.0 ** -1022, torch.float16: 2.0 ** -36}.get(dtype, 2.0 ** -126)
    return u, a, max(u, a), low


def agree(got, ref, bound, tiny, what):
    """got within bound of ref everywhere; tiny: the absolute step below the type's normal numbers"""
    got = got.detach().double().cpu().numpy()
    assert got.shape == ref.shape, f'{what}: shape {got.shape}, expected {ref.shape}'
    err = np.abs(got - ref)
    bad = ~(err <= bound + tiny)
    if bad.any():
        worst = np.unravel_index(np.nanargmax(np.where(bad, err / (bound + tiny), 0)), err.shape)
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.size} out of bounds, worst at {worst}: {got[worst]} for '
                             f'{ref[worst]}, bound {bound[worst]:.3g}')


def check_attn(dtype, q, k, v, go, kw, out, grads=None):
    r = dense.attn(q, k, v, grad_out=None if grads is None else go, **kw)
    b = dense.attn_bounds(r, *half_steps(dtype))
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps * 4
    agree(out, r['out'], b['out'], tiny, 'out')
    if grads is not None:
        for name, t in zip(('dq', 'dk', 'dv'), grads):
            agree(t, r[name], b[name], tiny, name)


NORM_SIZES = [(1, 256), (300, 256), (7, 1), (5, 3), (33, 64), (9, 100), (130, 257), (3, 1024), (2, 5000), (2, 16384),
              (600, 384), (1000, 8), (2049, 32)]


def make_norm(rows, C, dtype, weight=True, bias=True, residual=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (randn(g, rows, C) + randn(g, C)).to(dtype)
    w = (randn(g, C) * 0.2 + 1).to(dtype) if weight else None
    b = randn(g, C).to(dtype) if bias else None
    r = randn(g, rows, C).to(dtype) if residual else None
    return x, w, b, r, randn(g, rows, C).to(dtype)


def check_norm(dtype, x, w, b, r, go, out, grads=None, eps=1e-5):
    u, a = half_steps(dtype)[:2]
    ref = dense.layer_norm(x, w, b, r, eps, None if grads is None else go)
    bounds = dense.layer_norm_bounds(ref, u, a)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps * 4
    agree(out, ref['out'], bounds['out'], tiny, 'out')
    if grads is not None:
        for name, t in zip(('dx', 'dw', 'db'), grads):
            if t is not None:
                agree(t, ref[name], bounds[name], tiny, name)
