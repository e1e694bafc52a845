"""Layer norm on the GPU against the float64 oracle (oracle/dense.py), within the bounds that its layer_norm_bounds
derives: forward, backward, streams, graphs, alignments and the C ABI's buffers."""

import pytest
import torch

import marearts_tinydeform_amd as td
from marearts_tinydeform_amd import _native
from dense_cases import NORM_SIZES, check_norm, make_norm

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float64]


def say(msg):
    print(msg, flush=True)


def run(x, w, b, r, go, train=True, eps=1e-5):
    ts = [None if t is None else t.cuda().requires_grad_(train) for t in (x, w, b, r)]
    if not train:
        with torch.inference_mode():
            out = td.ma_layer_norm(ts[0], ts[1], ts[2], residual=ts[3], eps=eps)
        torch.cuda.synchronize()
        return out, None
    out = td.ma_layer_norm_train(ts[0], ts[1], ts[2], residual=ts[3], eps=eps)
    leaves = [t for t in ts if t is not None]
    got = dict(zip([id(t) for t in leaves], torch.autograd.grad(out, leaves, go.cuda())))
    grads = [got.get(id(t)) for t in ts]
    torch.cuda.synchronize()
    return out, grads


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', NORM_SIZES, ids=str)
def test_sizes(size, dtype):
    say(f'  norm {size} {dtype}')
    for w, b, r in ((True, True, True), (True, True, False), (False, False, True)):
        args = make_norm(*size, dtype, w, b, r)
        out, grads = run(*args)
        check_norm(dtype, *args, out, grads[:3])
        if grads[3] is not None:
            assert torch.equal(grads[3], grads[0])
        again, _ = run(*args, train=False)
        assert torch.equal(again, out)


@pytest.mark.parametrize('dtype', TYPES)
def test_constant_rows_and_large_means(dtype):
    x, w, b, r, go = make_norm(40, 256, dtype, residual=False)
    x[3] = 2.0                                     # no variance: rstd = 1 / sqrt(eps)
    x[5] = x[5] * 0.01 + 30                        # a mean far above the deviations
    out, grads = run(x, w, b, r, go)
    check_norm(dtype, x, w, b, r, go, out, grads[:3])
    assert torch.equal(out[3].cpu(), b)
    out, grads = run(x, w, b, r, go, eps=0.1)
    check_norm(dtype, x, w, b, r, go, out, grads[:3], eps=0.1)


@pytest.mark.parametrize('dtype', TYPES)
def test_shapes_strides_and_alignment(dtype):
    x, w, b, r, go = make_norm(60, 256, dtype)
    out, grads = run(x, w, b, r, go)

    def off(t):  # the same values one element off a 16-byte boundary
        return torch.cat([t.new_zeros(1).cuda(), t.cuda().flatten()])[1:].view(t.shape)
    for name, f in (('4-D', lambda t: t.cuda().view(3, 4, 5, 256) if t.dim() == 2 else t.cuda()),
                    ('transposed', lambda t: t.cuda().t().contiguous().t() if t.dim() == 2 else t.cuda()),
                    ('unaligned', off)):
        say(f'  norm {name} {dtype}')
        ts = [f(t).detach().requires_grad_() for t in (x, w, b, r)]
        o = td.ma_layer_norm_train(ts[0], ts[1], ts[2], residual=ts[3])
        got = torch.autograd.grad(o, ts, f(go))
        check_norm(dtype, x, w, b, r, go, o.reshape(60, 256), [t.reshape(s.shape) for t, s in zip(got, (x, w, b))])
    # a residual that is x itself: both gradients add up
    t = x.cuda().requires_grad_()
    o = td.ma_layer_norm_train(t, w.cuda(), b.cuda(), residual=t)
    g, = torch.autograd.grad(o, t, go.cuda())
    args = (x, w, b, x, go)
    check_norm(dtype, *args, o)
    _, one = run(*args)
    assert torch.equal(g, one[0] + one[3])


def test_some_gradients_only():
    x, w, b, r, go = make_norm(50, 128, torch.float32)
    _, want = run(x, w, b, r, go)
    for pick in ((0,), (1,), (2,), (3,), (0, 2)):
        ts = [t.cuda().requires_grad_(i in pick) for i, t in enumerate((x, w, b, r))]
        out = td.ma_layer_norm_train(ts[0], ts[1], ts[2], residual=ts[3])
        for i, g in zip(pick, torch.autograd.grad(out, [ts[i] for i in pick], go.cuda())):
            assert torch.equal(g, want[i])


def test_no_rows():
    x = torch.empty(0, 64, device='cuda', requires_grad=True)
    w = torch.ones(64, device='cuda', requires_grad=True)
    out = td.ma_layer_norm_train(x, w)
    dx, dw = torch.autograd.grad(out, (x, w), torch.empty(0, 64, device='cuda'))
    assert out.shape == dx.shape == (0, 64) and float(dw.abs().sum()) == 0
    with pytest.raises(RuntimeError, match='inference only'):
        td.ma_layer_norm(x, w)


@pytest.mark.parametrize('dtype', TYPES[:3])
def test_graphs_and_streams(dtype):
    graphs = []
    for rows, C in ((900, 256), (70, 1000)):
        x, w, b, r, go = make_norm(rows, C, dtype)
        want = run(x, w, b, r, go)
        ts = [t.cuda().requires_grad_() for t in (x, w, b, r)]
        g, s = go.cuda(), torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            side = run(x, w, b, r, go)
            torch.autograd.grad(td.ma_layer_norm_train(ts[0], ts[1], ts[2], residual=ts[3]), ts, g)
        torch.cuda.current_stream().wait_stream(s)
        for p, q in zip([side[0]] + side[1], [want[0]] + want[1]):
            assert torch.equal(p, q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = td.ma_layer_norm_train(ts[0], ts[1], ts[2], residual=ts[3])
            grads = torch.autograd.grad(out, ts, g)
        graphs.append((graph, (out.detach(),) + grads, [want[0]] + want[1], (ts, g)))
    for i in range(3):
        for graph, got, want, _ in graphs:
            for t in got:
                t.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for _, got, want, (ts, g) in graphs:
            for p, q in zip(got, want):
                assert torch.equal(p, q), f'replay {i}'
            with torch.no_grad():
                assert torch.equal(td.ma_layer_norm(*[t.detach() for t in ts[:3]], residual=ts[3].detach()), want[0])


@pytest.mark.parametrize('dtype', TYPES)
def test_c_abi_writes_its_buffers_and_nothing_else(dtype):
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    lib, code, fence = _native.lib, _native.DTYPE_CODES[dtype], 64

    def fenced(n, dt):
        t = torch.full((n + 2 * fence,), 7.0, dtype=dt, device='cuda')
        return t, t[fence:fence + n]
    for rows, C in ((33, 256), (1, 1000), (300, 36), (5, 4097)):
        x, w, b, r, go = make_norm(rows, C, dtype)
        dev = [t.cuda() for t in (x, w, b, r, go)]
        px, pw, pb, pr, pg = (t.data_ptr() for t in dev)
        need = lib.td_layer_norm_backward_workspace(code, rows, C)
        bufs = [fenced(rows * C, dtype), fenced(2 * rows, acc), fenced(rows * C, dtype), fenced(C, dtype),
                fenced(C, dtype), fenced(max(need, 8) // acc.itemsize, acc)]
        out, stats, dx, dw, db, ws = (t[1] for t in bufs)
        assert lib.td_layer_norm_forward(code, px, pr, pw, pb, out.data_ptr(), stats.data_ptr(), rows, C, 1e-5,
                                         None) == 0
        assert lib.td_layer_norm_backward(code, px, pr, pw, stats.data_ptr(), pg, dx.data_ptr(), dw.data_ptr(),
                                          db.data_ptr(), rows, C, ws.data_ptr(), need, None) == 0
        torch.cuda.synchronize()
        for whole, part in bufs:
            assert (whole[:fence] == 7).all() and (whole[fence + part.numel():] == 7).all()
        check_norm(dtype, x, w, b, r, go, out.view(rows, C), (dx.view(rows, C), dw, db))
