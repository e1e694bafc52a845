"""Performance cases of the dense operators beside deformable attention: attention among tokens and layer norm.

A case is a dict of plain values:

  kind     'attn'        ma_attn: attention of [B, Q, H, D] queries over [B, K, Hk, D] keys and values
           'attn_train'  ma_attn_train, forward and backward: the output and the gradients of all three inputs
           'norm'        ma_layer_norm over C channels of [B, Q, C] rows
           'norm_train'  ma_layer_norm_train, forward and backward: the output and every input's gradient
  dtype    'float32', 'float16' or 'bfloat16'
  attention:  B, Q, K, H, Hk, D   batch, queries, keys, heads, key heads (each shared by H / Hk heads), head width
              mask  'none'; 'padding': images padded to one length; 'denoising': a bool mask that keeps the groups of
                    denoising queries and the matching queries apart; 'denoising_float': the same as 0 / -inf in the
                    inputs' type; 'causal': each token sees itself and the ones before
  norm:       B, Q, C, residual   rows as [B, Q, C], and whether a residual is added before the norm
"""

import torch

own = False  # True: run() calls the package's entry points; False: it computes the same in plain torch


def _attn(name, kind, dtype, B, Q, K, H, Hk, D, mask):
    return {'name': name, 'kind': kind, 'dtype': dtype, 'B': B, 'Q': Q, 'K': K, 'H': H, 'Hk': Hk, 'D': D, 'mask': mask}


def _norm(name, kind, dtype, B, Q, C, residual):
    return {'name': name, 'kind': kind, 'dtype': dtype, 'B': B, 'Q': Q, 'C': C, 'residual': residual}


def listed():
    return [
        # a decoder layer's self-attention among its object queries, one frame: what single-stream serving calls
        _attn('decoder-fp16-b1-q300', 'attn', 'float16', 1, 300, 300, 8, 8, 32, 'none'),
        # every token of three 640-pixel maps attends to all the others: a dense encoder layer
        _attn('tokens-fp16-b2-n8400', 'attn', 'float16', 2, 8400, 8400, 8, 8, 32, 'none'),
        # one new token over long kept keys and values with shared heads, sequences of different lengths
        _attn('token-bf16-b4-k21760', 'attn', 'bfloat16', 4, 1, 21760, 16, 4, 64, 'padding'),
        # cross-attention in PyTorch's default type, odd sizes, padded images
        _attn('ragged-fp32-b3-q391-k1050', 'attn', 'float32', 3, 391, 1050, 6, 6, 36, 'padding'),
        # a training step's decoder self-attention: 300 matching queries and 200 denoising ones, float32
        _attn('train-fp32-b4-q500', 'attn_train', 'float32', 4, 500, 500, 8, 8, 32, 'denoising'),
        # the same with 900 and 200 in mixed precision, the mask as a model adds it to the scores
        _attn('train-bf16-b8-q1100', 'attn_train', 'bfloat16', 8, 1100, 1100, 8, 8, 32, 'denoising_float'),
        # the dense encoder layer's training step
        _attn('train-tokens-fp16-b2-n8400', 'attn_train', 'float16', 2, 8400, 8400, 8, 8, 32, 'none'),
        # a causal sequence with wide and shared heads, an odd length
        _attn('train-causal-bf16-b2-n4099', 'attn_train', 'bfloat16', 2, 4099, 4099, 16, 4, 128, 'causal'),
        # the norm after a decoder sublayer, one frame: the smallest call
        _norm('norm-fp16-b1-q300', 'norm', 'float16', 1, 300, 256, True),
        # the norm after an encoder sublayer on a batch
        _norm('norm-bf16-b8-n8400', 'norm', 'bfloat16', 8, 8400, 256, True),
        # a training step's norm over the tokens of four 800 x 1333 maps, float32
        _norm('train-norm-fp32-b2-n22223', 'norm_train', 'float32', 2, 22223, 256, True),
        # the widest model's: 1024 channels
        _norm('train-norm-bf16-c1024-b2-n21760', 'norm_train', 'bfloat16', 2, 21760, 1024, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    while True:
        kind = rng.choice(['attn', 'attn', 'attn_train', 'attn_train', 'attn_train', 'norm', 'norm_train', 'norm_train'])
        dtype = rng.choice(['float32', 'float16', 'bfloat16'])
        B = _log_int(rng, 1, 8)
        if kind.startswith('norm'):
            C = rng.choice([256, 256, 384, 1024, _log_int(rng, 64, 2048)])
            case = _norm('', kind, dtype, B, _log_int(rng, 100, 22000), C, rng.random() < 0.5)
        else:
            H, Hk = rng.choice([(8, 8), (8, 8), (8, 8), (6, 6), (12, 12), (16, 16), (16, 4), (8, 2), (12, 4), (8, 1)])
            D = rng.choice([32, 32, 32, 64, 64, 128, 16, 24, 36, 80])
            mask = rng.choice(['none', 'none', 'padding', 'causal', 'denoising', 'denoising_float'])
            Q = _log_int(rng, 50, 8400)
            K = Q
            if mask in ('none', 'padding') and rng.random() < 0.5:
                K = _log_int(rng, 50, 22000)
                if kind == 'attn' and rng.random() < 0.5:
                    Q = rng.choice([1, 1, 2, 7])
            case = _attn('', kind, dtype, B, Q, K, H, Hk, D, mask)
        del case['name']
        if kind.startswith('norm'):
            fits = _cost(case) <= _LARGEST['norm']
        else:  # nor more pairs of a query and a key: the plain form holds them all
            fits = _cost(case) <= _LARGEST['attn'] and B * H * Q * K <= 16 * 8400 * 8400
        if fits:
            return case


def _size(case):
    return 4 if case['dtype'] == 'float32' else 2


def work(case):
    s, B, Q = _size(case), case['B'], case['Q']
    if case['kind'].startswith('norm'):
        n, C = B * Q * case['C'], case['C']
        read, written = n * (2 if case['residual'] else 1) + 2 * C, n
        if case['kind'] == 'norm':
            return {'bytes': (read + written) * s, 'flops': 8 * n}
        return {'bytes': (read + written + n + n + 2 * C) * s, 'flops': 20 * n}  # and the incoming and outgoing gradient
    K, H, Hk, D = case['K'], case['H'], case['Hk'], case['D']
    pairs = B * H * (Q * (Q + 1) // 2 if case['mask'] == 'causal' else Q * K)
    rows, keys = B * Q * H * D, B * K * Hk * D
    masks = {'padding': B * K, 'denoising': Q * K, 'denoising_float': Q * K * s}.get(case['mask'], 0)
    if case['kind'] == 'attn':
        return {'bytes': (2 * rows + 2 * keys) * s + masks, 'flops': 4 * pairs * D}
    return {'bytes': (4 * rows + 4 * keys) * s + masks, 'flops': 14 * pairs * D}


def _cost(case):
    w = work(case)
    return w['bytes'] if case['kind'].startswith('norm') else w['flops'] * (_size(case) / 2) ** 2 + 1000 * w['bytes']


_LARGEST = {kind: max(_cost(c) for c in listed() if c['kind'].startswith(kind)) for kind in ('attn', 'norm')}


def _denoising(Q, device):
    """True where a query may not attend to a key: the first 2 Q / 11 or so queries are denoising queries in groups of
    10; groups do not see each other, and matching queries see no denoising query (a denoising query sees the matching
    ones)."""
    dn = max(1, Q * 2 // 11)
    group = torch.arange(Q, device=device) // 10
    group[dn:] = -1
    q, k = group[:, None], group[None, :]
    return (k >= 0) & (q != k)


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dtype = getattr(torch, case['dtype'])
    B, Q, train = case['B'], case['Q'], case['kind'].endswith('train')

    def randn(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device='cuda') * scale + shift).to(dtype)

    state = {'case': case}
    if case['kind'].startswith('norm'):
        C = case['C']
        # hidden states whose channels have means of their own, as they do after a few layers
        means = torch.randn(C, generator=g, device='cuda') * 0.5
        state['x'] = (torch.randn(B, Q, C, generator=g, device='cuda') + means).to(dtype)
        state['residual'] = randn(B, Q, C) if case['residual'] else None
        state['weight'], state['bias'] = randn(C, scale=0.1, shift=1.0), randn(C, scale=0.1)
        leaves = ['x', 'residual', 'weight', 'bias']
        if train:
            state['grad'] = randn(B, Q, C)
    else:
        K, H, Hk, D = case['K'], case['H'], case['Hk'], case['D']
        if Q == K and not train:  # self-attention: queries and keys of one projection, values of another
            qk = randn(B, Q, H + Hk, D, scale=1.2)
            state['q'], state['k'] = qk[:, :, :H], qk[:, :, H:]
        else:
            state['q'], state['k'] = randn(B, Q, H, D, scale=1.2), randn(B, K, Hk, D, scale=1.2)
        state['v'] = randn(B, K, Hk, D, shift=0.1)
        state['mask'] = state['padding'] = None
        if case['mask'] == 'padding':
            valid = torch.randint(K // 2, K + 1, (B, 1), generator=g, device='cuda')
            state['padding'] = torch.arange(K, device='cuda')[None, :] >= valid
        elif case['mask'].startswith('denoising'):
            state['mask'] = _denoising(Q, 'cuda')
            if case['mask'] == 'denoising_float':
                state['mask'] = torch.zeros(Q, K, dtype=dtype, device='cuda').masked_fill_(state['mask'], float('-inf'))
        leaves = ['q', 'k', 'v']
        if train:
            state['grad'] = randn(B, Q, H * D)
    if train:
        state['leaves'] = [state[n].requires_grad_() for n in leaves if state[n] is not None]
    return state


def run(state):
    kind = state['case']['kind']
    if own:
        return _own(state, kind)
    with torch.no_grad():
        return (_plain_norm if kind.startswith('norm') else _plain_attn)(state, kind.endswith('train'))


def _own(state, kind):
    import marearts_tinydeform_amd as td
    if kind.startswith('norm'):
        args = (state['x'], state['weight'], state['bias'])
        if kind == 'norm':
            return td.ma_layer_norm(*args, residual=state['residual'])
        out = td.ma_layer_norm_train(*args, residual=state['residual'])
    else:
        masks = {'attn_mask': state['mask'], 'key_padding_mask': state['padding'],
                 'causal': state['case']['mask'] == 'causal'}
        if kind == 'attn':
            return td.ma_attn(state['q'], state['k'], state['v'], **masks)
        out = td.ma_attn_train(state['q'], state['k'], state['v'], **masks)
    return (out.detach(),) + torch.autograd.grad(out, state['leaves'], state['grad'])


def _plain_attn(state, train):
    case, dtype = state['case'], state['q'].dtype
    B, Q, K, H, Hk, D = (case[n] for n in ('B', 'Q', 'K', 'H', 'Hk', 'D'))
    G = H // Hk
    scale = D ** -0.5
    q = state['q'].float().transpose(1, 2)                                              # [B, H, Q, D]
    k = state['k'].float().transpose(1, 2).repeat_interleave(G, 1)                      # [B, H, K, D]
    v = state['v'].float().transpose(1, 2).repeat_interleave(G, 1)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale                         # [B, H, Q, K]
    if case['mask'] == 'padding':
        s.masked_fill_(state['padding'][:, None, None, :], float('-inf'))
    elif case['mask'] == 'denoising':
        s.masked_fill_(state['mask'], float('-inf'))
    elif case['mask'] == 'denoising_float':
        s += state['mask'].float()
    elif case['mask'] == 'causal':
        i = torch.arange(K, device=s.device)
        s.masked_fill_(i[None, :] > i[:, None], float('-inf'))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p, v)
    out = o.transpose(1, 2).reshape(B, Q, H * D).to(dtype)
    if not train:
        return out
    do = state['grad'].float().view(B, Q, H, D).transpose(1, 2)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    dp -= (do * o).sum(-1, keepdim=True)
    ds = dp.mul_(p)
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dk, dv = (t.view(B, Hk, G, K, D).sum(2).transpose(1, 2).to(dtype) for t in (dk, dv))
    return out, dq.transpose(1, 2).to(dtype), dk, dv


def _plain_norm(state, train, eps=1e-5):
    dtype = state['x'].dtype
    x, w = state['x'].float(), state['weight'].float()
    if state['residual'] is not None:
        x = x + state['residual'].float()
    x = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    x *= rstd
    out = (x * w + state['bias'].float()).to(dtype)
    if not train:
        return out
    g = state['grad'].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - x * (gw * x).mean(-1, keepdim=True))
    dx = dx.to(dtype)
    grads = (dx, dx) if state['residual'] is not None else (dx,)
    return (out,) + grads + ((g * x).sum((0, 1)).to(dtype), g.sum((0, 1)).to(dtype))


def exact(case, seed):
    """The outputs in 64 bits: heads one after another, gradients by differentiating the definition."""
    state = prepare(case, seed)
    train = case['kind'].endswith('train')
    if case['kind'].startswith('norm'):
        names = [n for n in ('x', 'residual', 'weight', 'bias') if state[n] is not None]
        t = {n: state[n].detach().double().requires_grad_(train) for n in names}
        h = t['x'] + t['residual'] if 'residual' in t else t['x']
        var, mean = torch.var_mean(h, -1, unbiased=False, keepdim=True)
        out = (h - mean) / (var + 1e-5).sqrt() * t['weight'] + t['bias']
        if not train:
            return out
        return (out.detach(),) + torch.autograd.grad(out, [t[n] for n in names], state['grad'].double())
    B, Q, K, H, Hk, D = (case[n] for n in ('B', 'Q', 'K', 'H', 'Hk', 'D'))
    q, k, v = (state[n].detach().double() for n in ('q', 'k', 'v'))
    out = torch.empty(B, Q, H, D, dtype=torch.float64, device='cuda')
    grads = [torch.zeros_like(t, memory_format=torch.contiguous_format) for t in (q, k, v)] if train else []
    for b in range(B):
        bias = torch.zeros(Q, K, dtype=torch.float64, device='cuda')
        if state['padding'] is not None:
            bias[:, state['padding'][b]] = float('-inf')
        if state['mask'] is not None:
            bias[(state['mask'] if state['mask'].dtype == torch.bool else state['mask'] == float('-inf'))] = float('-inf')
        if case['mask'] == 'causal':
            bias = bias.masked_fill(torch.ones(Q, K, dtype=torch.bool, device='cuda').triu(1), float('-inf'))
        for h in range(H):
            j = h // (H // Hk)
            one = [t.contiguous().requires_grad_(train) for t in (q[b, :, h], k[b, :, j], v[b, :, j])]
            o = torch.softmax(one[0] @ one[1].T / D ** 0.5 + bias, -1) @ one[2]
            out[b, :, h] = o.detach()
            if train:
                got = torch.autograd.grad(o, one, state['grad'][b].double().view(Q, H, D)[:, h])
                for to, at, grad in zip(grads, (h, j, j), got):
                    to[b, :, at] += grad
    out = out.view(B, Q, H * D)
    return (out, *grads) if train else out
