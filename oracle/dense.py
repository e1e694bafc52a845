"""Float64 oracle of attention among tokens and of layer norm, with their gradients (numpy). TEST INFRASTRUCTURE ONLY.

Written from the formulas: t = scale q k^T + mask, P = softmax over the keys that the masks leave (a row left none is 0),
out = P v; dV = P^T g, dP = g v^T, dS = P (dP - sum_j P dP), dq = scale dS k, dk = scale dS^T q, summed over the heads
that share a key head. A padded key's row counts for nothing, whatever it holds.
"""

import numpy as np

from .bruteforce import _f64


def left_out(Q, K, attn_mask=None, key_padding_mask=None, causal=False):
    """Pairs that no score reaches, broadcastable to [B, H, Q, K], and the additive mask (0 where there is none)."""
    out, add = np.zeros((1, 1, Q, K), bool), np.zeros((1, 1, 1, 1))
    if attn_mask is not None:
        m = _f64(attn_mask)
        m = m.reshape((1,) * (4 - m.ndim) + m.shape)
        if attn_mask.is_floating_point():
            gone = m == -np.inf
            out = out | gone
            add = np.where(gone, 0.0, m)
        else:
            out = out | (m != 0)
    if key_padding_mask is not None:
        out = out | (_f64(key_padding_mask) != 0)[:, None, None, :]
    if causal:
        out = out | (np.arange(K)[None, :] > np.arange(Q)[:, None] + (K - Q))
    return out, add


def attn(q, k, v, attn_mask=None, key_padding_mask=None, scale=None, causal=False, grad_out=None):
    """A dict of float64 arrays: out [B, Q, H * D] and the probabilities P and scores' inputs; with grad_out also dq, dk,
    dv and dS."""
    q, k, v = (_f64(t) for t in (q, k, v))
    B, Q, H, D = q.shape
    K, G = k.shape[1], H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    gone, add = left_out(Q, K, attn_mask, key_padding_mask, causal)
    if key_padding_mask is not None:
        pad = (_f64(key_padding_mask) != 0)[:, :, None, None]
        k, v = np.where(pad, 0.0, k), np.where(pad, 0.0, v)
    qh = q.transpose(0, 2, 1, 3)
    kh, vh = (np.repeat(t.transpose(0, 2, 1, 3), G, 1) for t in (k, v))
    t = np.where(gone, -np.inf, qh @ kh.transpose(0, 1, 3, 2) * scale + add)
    top = t.max(-1, keepdims=True, initial=-np.inf)
    e = np.exp(t - np.where(np.isfinite(top), top, 0.0))
    total = e.sum(-1, keepdims=True)
    P = e / np.where(total == 0, 1.0, total)
    o = P @ vh
    r = {'out': o.transpose(0, 2, 1, 3).reshape(B, Q, H * D), 'P': P, 'q': qh, 'k': kh, 'v': vh, 'o': o, 'scale': scale,
         'add': add}
    if grad_out is not None:
        g = _f64(grad_out).reshape(B, Q, H, D).transpose(0, 2, 1, 3)
        dP = g @ vh.transpose(0, 1, 3, 2)
        dS = P * (dP - (P * dP).sum(-1, keepdims=True))

        def shared(x):  # [B, H, K, D] summed over the heads of a key head, as [B, K, Hk, D]
            return x.reshape(B, H // G, G, K, D).sum(2).transpose(0, 2, 1, 3)
        r.update(g=g, dS=dS, shared=shared, dq=(dS @ kh * scale).transpose(0, 2, 1, 3),
                 dk=shared(dS.transpose(0, 1, 3, 2) @ qh * scale), dv=shared(P.transpose(0, 1, 3, 2) @ g))
    return r


def attn_bounds(r, dtype_half_step, acc_half_step, p_half_step, p_low=0.0):
    """How far a right kernel's results may be from attn()'s `r`, elementwise, by name. dtype_half_step: the largest
    relative error of one rounding to the outputs' type, acc_half_step: of one in the accumulation type, p_half_step: of
    the roundings of P and dS before their products (acc_half_step where they are not rounded). p_low: the absolute error
    of a probability too small for the type it is held in (one below the smallest normal number may count as 0); dS is
    held to p_low times twice the bound 2 D max|grad_out| max|value| of |dP - delta|.

    A sum of n products in the accumulation type is off by at most n + 1 half steps of the sum of their magnitudes. A
    score is off by e_t; a probability, exp of it over the sum of K such, by the relative e_p = 2 e_t + (K + 16) half
    steps (16: the exponential's own error and the softmax's few operations). An additive mask counts towards a score's
    magnitude, but one beyond 2^100 takes the whole score in, here as in the kernels. delta is grad_out . out with out
    rounded."""
    u, a, w = dtype_half_step, acc_half_step, p_half_step
    q, k, v, P, scale = (r[n] for n in ('q', 'k', 'v', 'P', 'scale'))
    D, Q, K = q.shape[-1], q.shape[-2], k.shape[-2]

    def t2(x):
        return x.transpose(0, 1, 3, 2)
    add = np.where(np.abs(r['add']) < 2.0 ** 100, np.abs(r['add']), 0.0)
    top = np.where(P > 0, np.abs(q) @ t2(np.abs(k)) * scale + add, 0.0).max((-1,), keepdims=True, initial=0.0)
    e_p = 2 * (D + 4) * a * (top + 1) + (K + 16) * a        # [B, H, Q, 1]
    out = u * np.abs(r['o']) + ((w + e_p + (K + 1) * a) * (P @ np.abs(v)) + p_low * np.abs(v).sum(-2, keepdims=True)) \
        * (1 + u)
    B, H = q.shape[:2]
    b = {'out': out.transpose(0, 2, 1, 3).reshape(B, Q, H * D)}
    if 'g' in r:
        g, dS = np.abs(r['g']), np.abs(r['dS'])
        e_d = u * (g * np.abs(r['o'])).sum(-1, keepdims=True) + (g * out).sum(-1, keepdims=True) \
            + (D + 2) * a * (g * np.abs(r['o'])).sum(-1, keepdims=True)
        off = (w + e_p + 4 * a) * dS + P * (1 + e_p) * ((D + 2) * a * (g @ t2(np.abs(v))) + e_d)
        off = off + p_low * 4 * D * g.max(initial=0.0) * np.abs(v).max(initial=0.0)
        b['dq'] = (u * np.abs(r['dq']).transpose(0, 2, 1, 3)
                   + scale * (off + (K + 3) * a * (dS + off)) @ np.abs(k) * (1 + u)).transpose(0, 2, 1, 3)
        rows = Q * (H // (r['dk'].shape[2]))
        b['dk'] = u * np.abs(r['dk']) + r['shared'](scale * t2(off + (rows + 3) * a * (dS + off)) @ np.abs(q) * (1 + u))
        b['dv'] = u * np.abs(r['dv']) + r['shared'](t2(P * (w + e_p + (rows + 3) * a) + p_low) @ g * (1 + u))
    return b


def layer_norm(x, weight=None, bias=None, residual=None, eps=1e-5, grad_out=None):
    """A dict: out, and with grad_out dx, dw, db; float64."""
    h = _f64(x) if residual is None else _f64(x) + _f64(residual)
    w = np.ones(h.shape[-1]) if weight is None else _f64(weight)
    d = h - h.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    xh = d * rstd
    r = {'h': h, 'xh': xh, 'rstd': rstd, 'w': w, 'out': xh * w + (0 if bias is None else _f64(bias))}
    if grad_out is not None:
        g = _f64(grad_out)
        wg = w * g
        lead = tuple(range(h.ndim - 1))
        r.update(g=g, dx=rstd * (wg - wg.mean(-1, keepdims=True) - xh * (wg * xh).mean(-1, keepdims=True)),
                 dw=(g * xh).sum(lead), db=g.sum(lead))
    return r


def layer_norm_bounds(r, dtype_half_step, acc_half_step):
    """How far a right kernel may be from layer_norm()'s `r`, elementwise. The sum of C values is off by at most C half
    steps of the sum of their magnitudes, and so the mean by e_m = (C + 2) half steps of the mean magnitude; the
    deviations by e_m and their own rounding, the variance by twice that times the mean deviation, and rstd by half the
    variance's relative error."""
    u, a = dtype_half_step, acc_half_step
    h, xh, rstd, w = r['h'], r['xh'], r['rstd'], np.abs(r['w'])
    C = h.shape[-1]
    e_m = (C + 2) * a * np.abs(h).mean(-1, keepdims=True)
    e_h = e_m + 2 * a * np.abs(h)                                              # of h - mean
    e_r = (np.abs(xh) * rstd * e_h).mean(-1, keepdims=True) + (C + 8) * a + (rstd * e_m) ** 2   # relative, of rstd
    e_x = rstd * e_h + np.abs(xh) * (e_r + 2 * a)                              # of xhat
    b = {'out': u * np.abs(r['out']) + (w * e_x + 3 * a * (w * np.abs(xh) + np.abs(r['out']))) * (1 + u)}
    if 'g' in r:
        g = np.abs(r['g'])
        wg = w * g
        m1, m2 = wg.mean(-1, keepdims=True), (wg * np.abs(xh)).mean(-1, keepdims=True)
        e1 = (C + 4) * a * m1
        e2 = (C + 6) * a * m2 + (wg * e_x).mean(-1, keepdims=True)
        inner = wg + m1 + np.abs(xh) * m2
        b['dx'] = u * np.abs(r['dx']) + rstd * (e1 + np.abs(xh) * e2 + e_x * m2 + (e_r + 8 * a) * inner) * (1 + u)
        rows = h.size // C
        lead = tuple(range(h.ndim - 1))
        b['dw'] = u * np.abs(r['dw']) + ((g * e_x).sum(lead) + (rows + 2) * a * (g * np.abs(xh)).sum(lead)) * (1 + u)
        b['db'] = u * np.abs(r['db']) + (rows + 2) * a * g.sum(lead) * (1 + u)
    return b
