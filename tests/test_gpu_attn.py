"""Attention among tokens on the GPU against the float64 oracle (oracle/dense.py), within the bounds that its
attn_bounds derives: forward, backward, every mask, strides, streams, graphs and the C ABI's buffers."""

import numpy as np
import pytest
import torch

import marearts_tinydeform_amd as td
from marearts_tinydeform_amd import _dense, _native
from oracle import dense
from dense_cases import ATTN_SIZES, MASKS, agree, check_attn, half_steps, make_attn

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def say(msg):
    print(msg, flush=True)


def on_gpu(kw):
    return {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in kw.items()}


def run(q, k, v, go, kw, train=True):
    """(out, grads) of the GPU entries for CPU inputs"""
    kw = on_gpu(kw)
    a, b, c = (t.cuda().requires_grad_(train) for t in (q, k, v))
    if not train:
        with torch.inference_mode():
            out = td.ma_attn(a, b, c, **kw)
        torch.cuda.synchronize()
        return out, None
    out = td.ma_attn_train(a, b, c, **kw)
    grads = torch.autograd.grad(out, (a, b, c), go.cuda())
    torch.cuda.synchronize()
    return out, grads


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', ATTN_SIZES, ids=str)
def test_sizes(size, dtype):
    say(f'  attention {size} {dtype}')
    q, k, v, go, kw = make_attn(size, dtype)
    out, grads = run(q, k, v, go, kw)
    check_attn(dtype, q, k, v, go, kw, out, grads)
    again, _ = run(q, k, v, go, kw, train=False)
    assert torch.equal(again, out), 'inference and training forward differ'


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('mask', MASKS[1:])
def test_masks(mask, dtype):
    for i, size in enumerate([(2, 45, 100, 2, 2, 32), (1, 130, 70, 4, 2, 64), (3, 5, 300, 4, 1, 36),
                              (2, 150, 150, 2, 2, 32), (2, 1, 513, 4, 4, 128)]):
        say(f'  attention {mask} {size} {dtype}')
        q, k, v, go, kw = make_attn(size, dtype, mask, seed=i)
        out, grads = run(q, k, v, go, kw)
        check_attn(dtype, q, k, v, go, kw, out, grads)
        again, _ = run(q, k, v, go, kw, train=False)
        assert torch.equal(again, out), 'inference and training forward differ'


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('form', ['bool', 'float', 'float with a value'])
def test_block_masks(form, dtype):
    """Masks of whole blocks (denoising groups): 32 x 32 tiles with nothing, something and everything masked, for
    shared and single heads, a mask by head and by batch, more keys than queries and fewer."""
    g = torch.Generator().manual_seed(3)
    for size, lead in (((2, 200, 200, 4, 4, 32), (200,)), ((2, 130, 330, 6, 2, 64), (2, 6, 130)),
                       ((1, 300, 100, 8, 8, 32), (1, 8, 1)), ((2, 100, 100, 12, 4, 32), (2, 1, 100)),
                       ((2, 70, 600, 4, 1, 128), (1, 4, 70))):
        say(f'  block mask {form} {size} {lead} {dtype}')
        q, k, v, go, _ = make_attn(size, dtype)
        Q, K = size[1], size[2]
        rows, cols = torch.arange(lead[-1])[:, None] // 48, torch.arange(K)[None, :] // 80
        mask = ((rows * 7 + cols * 3) % 5 < 2) & (rows != 1)
        shape = tuple(lead[:-1]) + (lead[-1], K)
        mask = mask.expand(shape).clone()
        if len(shape) == 4:
            mask ^= torch.rand(shape[:2], generator=g)[:, :, None, None] < 0.3
            mask &= torch.rand(shape[:2], generator=g)[:, :, None, None] < 0.9
        kw = dict(attn_mask=mask)
        if form != 'bool':
            kw['attn_mask'] = torch.zeros(shape, dtype=dtype).masked_fill(mask, float('-inf'))
            if form != 'float':
                kw['attn_mask'][..., ::70, 5::64] += 1.25
        out, grads = run(q, k, v, go, kw)
        check_attn(dtype, q, k, v, go, kw, out, grads)


@pytest.mark.parametrize('mask', ['none', 'bool', 'float', 'lowest', 'all'])
def test_float64(mask):
    for size in [(2, 33, 70, 4, 2, 36), (1, 1, 65, 2, 2, 128)]:
        q, k, v, go, kw = make_attn(size, torch.float64, mask)
        out, grads = run(q, k, v, go, kw)
        check_attn(torch.float64, q, k, v, go, kw, out, grads)


@pytest.mark.parametrize('dtype', TYPES)
def test_tiles_left_over_after_an_even_share(dtype):
    # 130 heads of four tiles: on 256 CUs 512 tiles and 8 more, which several workgroups share. Heads at both ends
    # against the oracle; the others are the first head's, bit for bit
    one, two = (make_attn((1, 500, 500, 1, 1, 32), dtype, seed=i) for i in (0, 1))
    for mask in (None, torch.rand(500, 500, generator=torch.Generator().manual_seed(2)) < 0.3):
        kw = {} if mask is None else dict(attn_mask=mask)
        q, k, v, go = (torch.cat([a.unflatten(-1, (-1, 32)) if a.dim() == 3 else a] * 129
                                 + [b.unflatten(-1, (-1, 32)) if b.dim() == 3 else b], 2)
                       for a, b in zip(one[:4], two[:4]))
        out, grads = run(q, k, v, go.flatten(2), kw)
        parts = [out.unflatten(-1, (130, 32))] + list(grads)
        for h, (a, b, c, g, _) in ((0, one), (128, one), (129, two)):
            at = [t[:, :, h:h + 1] for t in parts]
            check_attn(dtype, a, b, c, g, kw, at[0].flatten(2), at[1:])
        for t in parts:
            assert torch.equal(t[:, :, :1].expand(-1, -1, 128, -1), t[:, :, :128])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('mask', ['none', 'bool', 'float', 'padding', 'causal'])
@pytest.mark.parametrize('size', [(1, 530, 8300, 2, 2, 32), (1, 8300, 530, 1, 1, 64), (2, 700, 1500, 2, 1, 128),
                                  (1, 1100, 1100, 2, 2, 100)], ids=str)
def test_long_loops_in_parts(size, mask, dtype):
    # few tiles and long loops: keys (and for dK and dV rows) are split over workgroups and the parts joined
    say(f'  attention {mask} {size} {dtype}')
    q, k, v, go, kw = make_attn(size, dtype, mask, seed=3)
    out, grads = run(q, k, v, go, kw)
    check_attn(dtype, q, k, v, go, kw, out, grads)


@pytest.mark.parametrize('dtype', TYPES)
def test_two_calls_at_once(dtype):
    # a training step on each of two streams, their kernels and workspaces side by side
    cases = [make_attn((1, 700, 1500, 2, 1, 128), dtype, 'bool', seed=1), make_attn((2, 300, 900, 4, 4, 32), dtype, 'float')]
    want = [run(*c[:4], c[4]) for c in cases]
    inputs = [([t.cuda().requires_grad_() for t in c[:3]], c[3].cuda(), on_gpu(c[4])) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, (ts, g, kw) in zip(streams, inputs):
            with torch.cuda.stream(s):
                out = td.ma_attn_train(*ts, **kw)
                got.append((out.detach(),) + torch.autograd.grad(out, ts, g))
    torch.cuda.synchronize()
    for i, ts in enumerate(got):
        for a, b in zip(ts, (want[i % 2][0],) + want[i % 2][1]):
            assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', TYPES)
def test_a_row_left_nothing_gives_zeros(dtype):
    q, k, v, go, _ = make_attn((2, 40, 50, 2, 2, 32), dtype)
    mask = torch.zeros(2, 1, 40, 50, dtype=torch.bool)
    mask[0, 0, 3] = True
    mask[1] = True
    out, (dq, dk, dv) = run(q, k, v, go, dict(attn_mask=mask))
    out = out.detach()
    assert float(out[0, 3].abs().sum()) == 0 and float(out[1].abs().sum()) == 0
    assert float(dq[0, 3].abs().sum()) == 0 and float(dq[1].abs().sum()) == 0
    assert float(dk[1].abs().sum()) == 0 and float(dv[1].abs().sum()) == 0
    assert float(out[0].abs().sum()) > 0 and torch.isfinite(dk).all()


@pytest.mark.parametrize('dtype', TYPES + [torch.float64])
def test_padded_keys_count_for_nothing_whatever_they_hold(dtype):
    q, k, v, go, _ = make_attn((2, 40, 90, 2, 2, 32), dtype)
    pad = torch.zeros(2, 90, dtype=torch.bool)
    pad[0, 70:] = True
    pad[1, ::3] = True
    clean = run(q, k, v, go, dict(key_padding_mask=pad))
    for value in (float('nan'), float('inf'), -float('inf')):
        k2, v2 = k.clone(), v.clone()
        k2[pad], v2[pad] = value, value
        out, grads = run(q, k2, v2, go, dict(key_padding_mask=pad))
        assert torch.equal(out, clean[0])
        for a, b in zip(grads, clean[1]):
            assert torch.equal(a, b)
        assert float(grads[1][pad.cuda()].abs().sum()) == 0 and float(grads[2][pad.cuda()].abs().sum()) == 0


@pytest.mark.parametrize('dtype', TYPES)
def test_large_scores(dtype):
    # scores of hundreds: one key takes nearly all of each row, the others underflow
    q, k, v, go, _ = make_attn((1, 60, 130, 2, 2, 32), dtype)
    q, k = q * 8, k * 8
    out, grads = run(q, k, v, go, {})
    check_attn(dtype, q, k, v, go, {}, out, grads)
    # the first keys' scores far below the last ones': the running maximum moves on every tile
    k = (k.float() * torch.linspace(0.01, 2, 130)[None, :, None, None]).to(dtype)
    out, grads = run(q, k, v, go, {})
    check_attn(dtype, q, k, v, go, {}, out, grads)


@pytest.mark.parametrize('size', [(1, 60, 130), (2, 8400, 130), (1, 3, 4100)])
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('dtype', TYPES)
def test_scores_past_the_bits_of_their_logarithm(dtype, masked, size):
    """Scores of 2^25 and more, whose float32 steps are larger than log2 of the row's sum: ten patterns of signs as queries
    and keys, so that each query attends evenly to the keys of its own pattern and every score is exact.

    The bounds: an even probability is exact before it is divided; rounded to the type (half a step u) in the backward
    pass, as dS is, and every result is rounded once. grad_out . out holds u^2 of its terms (out with its remainder), sums
    in float32 64 half steps of theirs."""
    B, Q, K = size
    g = torch.Generator().manual_seed(5)
    signs = torch.randint(0, 2, (10, 32), generator=g).double() * 4096 - 2048
    q = signs[torch.arange(Q) % 10][None, :, None].expand(B, -1, -1, -1).to(dtype)
    k = signs[torch.arange(K) % 10][None, :, None].expand(B, -1, -1, -1).to(dtype)
    v = torch.randn(B, K, 1, 32, generator=g).to(dtype)
    go = torch.randn(B, Q, 32, generator=g).to(dtype)
    go[:, 100:] = 0  # so that sums over thousands of queries stay within float16
    kw = {}
    if masked:
        kw['key_padding_mask'] = torch.zeros(B, K, dtype=torch.bool)
        kw['key_padding_mask'][:, -3:] = True
    out, grads = run(q, k, v, go, kw)
    out, (dq, dk, dv) = out.detach().double().cpu()[:, :100], [t.double().cpu()[:, :, 0] for t in grads]
    q, k, v, go = q.double()[:, :100, 0], k.double()[:, :, 0], v.double()[:, :, 0], go.double()[:, :100]
    live = torch.ones(B, K) if not masked else (~kw['key_padding_mask']).double()
    P = (torch.arange(q.size(1))[:, None] % 10 == torch.arange(K)[None] % 10).double() * live[:, None]
    P = P / P.sum(-1, keepdim=True)
    o = P @ v
    scale, u, f = 32 ** -0.5, torch.finfo(dtype).eps / 2, 2.0 ** -24
    dp, delta = go @ v.transpose(1, 2), (go * o).sum(-1, keepdim=True)
    ds = P * (dp - delta)
    e_ds = 2 * u * ds.abs() + P * (u * u + 64 * f) * (go.abs() @ v.abs().transpose(1, 2) +
                                                      (go * o).abs().sum(-1, keepdim=True))
    for name, got, want, bound in (
            ('out', out, o, 64 * f * (P @ v.abs())),
            ('dv', dv, P.transpose(1, 2) @ go, (u + 64 * f) * (P.transpose(1, 2) @ go.abs())),
            ('dq', dq[:, :100], ds @ k * scale, e_ds @ k.abs() * scale),
            ('dk', dk, ds.transpose(1, 2) @ q * scale, e_ds.transpose(1, 2) @ q.abs() * scale)):
        excess = (got - want).abs() - bound - u * want.abs() - 2.0 ** -24
        assert float(excess.max()) <= 0, f'{name}: {float(excess.max()):.3g} past its bound'
        assert torch.isfinite(got).all(), name


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
def test_small_and_large_gradients(dtype):
    # gradients of a loss over many tokens (1e-4) and of a scaled loss (1e3): dS is rounded to 16 bits
    for scale in (1e-4, 1e3):
        q, k, v, go, kw = make_attn((1, 100, 700, 2, 2, 32), dtype, grad_scale=scale)
        out, grads = run(q, k, v, go, kw)
        check_attn(dtype, q, k, v, go, kw, out, grads)


@pytest.mark.parametrize('dtype', TYPES)
def test_strides(dtype):
    B, N, H, D = 2, 70, 3, 32
    q, k, v, go, _ = make_attn((B, N, N, H, H, D), dtype)
    want, wgrads = run(q, k, v, go, {})
    joint = torch.stack([q, k, v], 2).cuda()                            # slices of a joint projection
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2).cuda() for t in (q, k, v)]   # head-major
    odd = torch.zeros(B * N * H * D + 1, dtype=dtype, device='cuda')     # off 16-byte boundaries
    odd = [torch.cat([odd[:1], t.cuda().flatten()])[1:].view(B, N, H, D) for t in (q, k, v)]
    wide = [torch.cat([t, t[..., :5]], -1).cuda()[..., :D] for t in (q, k, v)]           # head rows of 37 elements
    last = [t.transpose(1, 3).contiguous().transpose(1, 3).cuda() for t in (q, k, v)]    # last dimension strided
    for name, ts in (('joint', joint.unbind(2)), ('heads', heads), ('odd', odd), ('wide', wide), ('last', last)):
        say(f'  strides {name} {dtype}')
        ts = [t.detach().requires_grad_() for t in ts]
        out = td.ma_attn_train(*ts)
        grads = torch.autograd.grad(out, ts, go.cuda())
        check_attn(dtype, q, k, v, go, {}, out, grads)
    one = k[:1].cuda().requires_grad_()                                 # one image's keys for the whole batch
    val = v[:1].cuda().requires_grad_()
    qg = q.cuda().requires_grad_()
    out = td.ma_attn_train(qg, one.expand(B, N, H, D), val.expand(B, N, H, D))
    grads = torch.autograd.grad(out, (qg, one, val), go.cuda())
    k2, v2 = k[:1].expand(B, N, H, D), v[:1].expand(B, N, H, D)
    r = dense.attn(q, k2, v2, grad_out=go)
    u = half_steps(dtype)[0]
    b = dense.attn_bounds(r, *half_steps(dtype))
    agree(out, r['out'], b['out'], 1e-6, 'broadcast out')
    for name, t in (('dk', grads[1]), ('dv', grads[2])):                # autograd adds the images' in dtype: 2 u more
        ref = r[name].sum(0, keepdims=True)
        agree(t, ref, b[name].sum(0, keepdims=True) + 2 * u * np.abs(r[name]).sum(0, keepdims=True), 1e-6, name)
    # a mask with strides of its own, and a non-contiguous incoming gradient
    big = torch.rand(N, 2 * N, generator=torch.Generator().manual_seed(1)) < 0.5
    m, gt = big[:, ::2], go.transpose(0, 1).contiguous().transpose(0, 1)
    for mm in (m, big[:, :N], m.t().contiguous().t()):
        ts = [t.cuda().requires_grad_() for t in (q, k, v)]
        out = td.ma_attn_train(*ts, attn_mask=mm.cuda())
        grads = torch.autograd.grad(out, ts, gt.cuda())
        check_attn(dtype, q, k, v, go, dict(attn_mask=mm.contiguous()), out, grads)


def test_some_gradients_only():
    q, k, v, go, _ = make_attn((1, 30, 40, 2, 2, 32), torch.float32)
    _, want = run(q, k, v, go, {})
    for pick in ((0,), (1,), (2,), (0, 2)):
        ts = [t.cuda().requires_grad_(i in pick) for i, t in enumerate((q, k, v))]
        grads = torch.autograd.grad(td.ma_attn_train(*ts), [ts[i] for i in pick], go.cuda())
        for i, g in zip(pick, grads):
            assert torch.equal(g, want[i])


def test_nothing_to_attend_to():
    for B, Q, K in ((0, 3, 4), (2, 0, 4), (2, 3, 0), (2, 0, 0)):
        ts = [torch.randn(B, n, 2, 8, device='cuda').requires_grad_() for n in (Q, K, K)]
        out = td.ma_attn_train(*ts)
        assert out.shape == (B, Q, 16) and float(out.detach().abs().sum()) == 0
        for t, g in zip(ts, torch.autograd.grad(out, ts, torch.ones_like(out))):
            assert g.shape == t.shape and float(g.abs().sum()) == 0


def test_refuses_gradients_in_the_inference_entry():
    t = torch.randn(1, 4, 2, 8, device='cuda', requires_grad=True)
    with pytest.raises(RuntimeError, match='inference only'):
        td.ma_attn(t, t, t)
    with pytest.raises(RuntimeError, match='attn_mask has no gradient'):
        td.ma_attn_train(t, t, t, attn_mask=torch.zeros(4, 4, device='cuda', requires_grad=True))
    out = td.ma_attn_train(t, t, t)
    g, = torch.autograd.grad(out, t, torch.ones_like(out).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), t)


@pytest.mark.parametrize('dtype', TYPES)
def test_the_same_on_every_run_and_on_another_stream(dtype):
    q, k, v, go, kw = make_attn((2, 200, 333, 4, 2, 64), dtype, 'padding')
    want = run(q, k, v, go, kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(q, k, v, go, kw)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip((want[0],) + want[1], (got[0],) + got[1]):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
def test_graphs_replay_forward_and_backward(dtype):
    """Two captured graphs (a training step each, other sizes) and eager work in between: every replay is the eager
    result. The leaves of a captured step have no eager graph alive, as torch asks of captured backward passes."""
    graphs = []
    for size, mask in (((2, 100, 100, 4, 4, 32), 'bool'), ((1, 2, 3000, 8, 2, 64), 'padding')):
        q, k, v, go, kw = make_attn(size, dtype, mask)
        want, wgrads = run(q, k, v, go, kw)
        ts = [t.cuda().requires_grad_() for t in (q, k, v)]
        kw, g = on_gpu(kw), go.cuda()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            torch.autograd.grad(td.ma_attn_train(*ts, **kw), ts, g)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = td.ma_attn_train(*ts, **kw)
            grads = torch.autograd.grad(out, ts, g)
        graphs.append((graph, (out.detach(),) + grads, (want,) + wgrads, (ts, kw, g)))
    for i in range(3):
        for graph, got, want, _ in graphs:
            for t in got:
                t.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for _, got, want, (ts, kw, g) in graphs:
            for a, b in zip(got, want):
                assert torch.equal(a, b), f'replay {i}'
            with torch.inference_mode():
                assert torch.equal(td.ma_attn(*[t.detach() for t in ts], **kw), want[0])


@pytest.mark.parametrize('dtype', TYPES)
def test_c_abi_writes_its_buffers_and_nothing_else(dtype):
    for size in [(1, 33, 70, 4, 2, 36), (2, 1, 2000, 4, 1, 64), (1, 130, 60, 2, 2, 32)]:
        B, Q, K, H, Hk, D = size
        q, k, v, go, _ = make_attn(size, dtype)
        q, k, v, go = (t.cuda() for t in (q, k, v, go))
        lib, acc = _native.lib, torch.float32
        fence = 64

        def fenced(n, dt):
            t = torch.full((n + 2 * fence,), 7.0, dtype=dt, device='cuda')
            return t, t[fence:fence + n]
        bufs = [fenced(B * Q * H * D, dtype), fenced(B * H * Q * 2, acc), fenced(B * Q * H * D, dtype),
                fenced(B * K * Hk * D, dtype), fenced(B * K * Hk * D, dtype)]
        out, stats, dq, dk, dv = (b[1] for b in bufs)
        low = fenced(B * Q * H * D, dtype)
        bufs.append(low)
        args = _dense._pack(q, k, v, None, 0, (0, 0, 0), None, D ** -0.5, False, out, stats,
                            None if dtype == torch.float32 else low[1])
        need = lib.td_attn_forward_workspace(args)
        w1 = fenced(max(need, 4) // 4, torch.float32)
        assert lib.td_attn_forward(args, w1[1].data_ptr(), need, None) == 0
        need = lib.td_attn_backward_workspace(args)
        w2 = fenced(max(need, 4) // 4, torch.float32)
        assert lib.td_attn_backward(args, go.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), w2[1].data_ptr(),
                                    need, None) == 0
        torch.cuda.synchronize()
        for whole, part in bufs + [w1, w2]:
            n = part.numel()
            assert (whole[:fence] == 7).all() and (whole[fence + n:] == 7).all()
        check_attn(dtype, q.cpu(), k.cpu(), v.cpu(), go.cpu(), {}, out.view(B, Q, H * D),
                   (dq.view(q.shape), dk.view(k.shape), dv.view(v.shape)))


def test_a_long_cache_past_32_bit_offsets():
    # 4.5e9 elements of keys: rows behind the 2^32nd element are read through 64-bit offsets
    K, Hk, D = 70_000_000, 1, 64
    key = torch.zeros(1, K, Hk, D, dtype=torch.float16, device='cuda')
    value = torch.zeros(1, K, Hk, D, dtype=torch.float16, device='cuda')
    key[0, K - 3], value[0, K - 3] = 10, torch.arange(D, device='cuda').half()[None]
    key[0, 1], value[0, 1] = 10, 1
    q = torch.full((1, 1, 1, D), 10.0, dtype=torch.float16, device='cuda')  # scores 800 there, 0 elsewhere
    out = td.ma_attn(q, key, value)
    want = (torch.arange(D).double() + 1) / 2
    agree(out.view(D), want.numpy(), want.numpy() * 2.0 ** -10, 1e-3, 'out')
