"""Attention among tokens and layer norm on the CPU: the float64 oracle against PyTorch's autograd and against planted
mistakes, the package's PyTorch path against the oracle, the host checks, and the C ABI's (include/tinydeform_dense.h)."""

import ctypes
import os
import re

import numpy as np
import pytest
import torch

import marearts_tinydeform_amd as td
from marearts_tinydeform_amd import _dense, _native
from oracle import dense
from dense_cases import ATTN_SIZES, MASKS, check_attn, check_norm, make_attn, make_norm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, 'include', 'tinydeform_dense.h')
SMALL = [s for s in ATTN_SIZES if s[0] * s[1] * s[2] * s[3] <= 60000]
TYPES = [torch.float64, torch.float32, torch.float16, torch.bfloat16]


def exact(*ts):
    return [t.detach().double().requires_grad_() for t in ts]


@pytest.mark.parametrize('mask', MASKS)
def test_attention_oracle_matches_autograd(mask):
    q, k, v, go, kw = make_attn((2, 9, 13, 6, 2, 5), torch.float64, mask)
    a, b, c = exact(q, k, v)
    out = td.ma_attn_reference(a, b, c, **kw)
    grads = torch.autograd.grad(out, (a, b, c), go)
    r = dense.attn(q, k, v, grad_out=go, **kw)
    for name, t in zip(('out', 'dq', 'dk', 'dv'), (out,) + grads):
        np.testing.assert_allclose(t.detach().numpy(), r[name], rtol=0, atol=1e-12, err_msg=name)


def test_attention_matches_torch_softmax_and_differences():
    q, k, v, go, _ = make_attn((1, 4, 6, 2, 2, 3), torch.float64)
    want = torch.softmax(torch.einsum('bqhd,bkhd->bhqk', q, k) * 3 ** -0.5, -1)
    want = torch.einsum('bhqk,bkhd->bqhd', want, v).reshape(1, 4, 6)
    r = dense.attn(q, k, v, grad_out=go)
    np.testing.assert_allclose(r['out'], want.numpy(), rtol=0, atol=1e-13)
    for name, t in (('dq', q), ('dk', k), ('dv', v)):  # central differences of sum(out * go)
        flat = t.view(-1)
        for i in range(0, flat.numel(), 5):
            old, step, f = float(flat[i]), 1e-5, []
            for s in (step, -step):
                flat[i] = old + s
                f.append(float((dense.attn(q, k, v)['out'] * go.numpy()).sum()))
            flat[i] = old
            assert abs((f[0] - f[1]) / (2 * step) - r[name].reshape(-1)[i]) < 1e-8, (name, i)


def test_planted_mistakes_leave_the_bounds():
    # the bounds a kernel is held to notice a dropped key, a wrong scale and an unshared head's gradient
    q, k, v, go, _ = make_attn((1, 20, 70, 4, 2, 32), torch.bfloat16)
    r = dense.attn(q, k, v, grad_out=go)
    good = [torch.from_numpy(r[n]).bfloat16() for n in ('out', 'dq', 'dk', 'dv')]
    check_attn(torch.bfloat16, q, k, v, go, {}, good[0], good[1:])
    pad = torch.zeros(1, 70, dtype=torch.bool)
    pad[0, 69] = True
    for wrong in (dense.attn(q, k, v, key_padding_mask=pad, grad_out=go), dense.attn(q, k, v, scale=0.18, grad_out=go),
                  dense.attn(q, k, v, causal=True, grad_out=go)):
        for i, n in enumerate(('out', 'dq', 'dk', 'dv')):
            t = list(good)
            t[i] = torch.from_numpy(wrong[n]).bfloat16()
            with pytest.raises(AssertionError, match='out of bounds'):
                check_attn(torch.bfloat16, q, k, v, go, {}, t[0], t[1:])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('mask', MASKS)
def test_attention_on_the_cpu(mask, dtype):
    for size in SMALL[:8]:
        q, k, v, go, kw = make_attn(size, dtype, mask)
        with torch.inference_mode():
            check_attn(dtype, q, k, v, go, kw, td.ma_attn(q, k, v, **kw))
        if dtype in (torch.float64, torch.float32):
            a, b, c = (t.requires_grad_() for t in (q, k, v))
            out = td.ma_attn_train(a, b, c, **kw)
            check_attn(dtype, q, k, v, go, kw, out, torch.autograd.grad(out, (a, b, c), go))


def test_attention_of_nothing():
    for B, Q, K in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        out = td.ma_attn(torch.randn(B, Q, 2, 8), torch.randn(B, K, 2, 8), torch.randn(B, K, 2, 8))
        assert out.shape == (B, Q, 16) and float(out.abs().sum()) == 0


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(7, 1), (5, 3), (9, 100), (3, 1024)])
def test_layer_norm_on_the_cpu(size, dtype):
    for w, b, r in ((True, True, True), (False, False, False), (True, False, True)):
        x, w, b, r, go = make_norm(*size, dtype, w, b, r)
        check_norm(dtype, x, w, b, r, go, td.ma_layer_norm(x, w, b, residual=r))
        if dtype in (torch.float64, torch.float32):
            leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
            out = td.ma_layer_norm_train(x, w, b, residual=r)
            got = dict(zip([id(t) for t in leaves], torch.autograd.grad(out, leaves, go)))
            check_norm(dtype, x, w, b, r, go, out, [got.get(id(t)) for t in (x, w, b)])


def test_layer_norm_oracle_matches_torch():
    x, w, b, r, go = make_norm(6, 10, torch.float64)
    a, c, d = exact(x, w, b)
    out = torch.nn.functional.layer_norm(a + r, (10,), c, d)
    grads = torch.autograd.grad(out, (a, c, d), go)
    ref = dense.layer_norm(x, w, b, r, grad_out=go)
    for name, t in zip(('out', 'dx', 'dw', 'db'), (out,) + grads):
        np.testing.assert_allclose(t.detach().numpy(), ref[name], rtol=0, atol=1e-12, err_msg=name)


# ---- refusals -----------------------------------------------------------------------------------------------------

def attn_args(B=2, Q=5, K=7, H=4, Hk=2, D=8, dtype=torch.float32):
    return [torch.randn(B, Q, H, D, dtype=dtype), torch.randn(B, K, Hk, D, dtype=dtype),
            torch.randn(B, K, Hk, D, dtype=dtype)]


@pytest.mark.parametrize('change,message', [
    (lambda a: a.__setitem__(0, a[0][0]), 'query must be [B, Q, H, D]'),
    (lambda a: a.__setitem__(1, a[1][0]), 'key and value must be [B, K, Hk, D]'),
    (lambda a: a.__setitem__(2, a[2][:, :6]), 'key and value must be [B, K, Hk, D]'),
    (lambda a: a.__setitem__(0, a[0][:1]), 'batch size mismatch'),
    (lambda a: a.__setitem__(0, a[0][:, :, :3]), 'the heads of key and value must divide'),
    (lambda a: a.__setitem__(0, a[0][:, :, :0]), 'need at least one head'),
    (lambda a: a.__setitem__(0, a[0][..., :4]), 'key and value must have the head dim of query'),
    (lambda a: a.__setitem__(1, a[1].double()), 'all float tensors must have the same dtype'),
    (lambda a: a.__setitem__(slice(0, 3), [t.int() for t in a]), 'unsupported dtype'),
    (lambda a: a.__setitem__(slice(0, 3), attn_args(D=257)), 'head dim must be from 1 to 256'),
    (lambda a: a.__setitem__(slice(0, 3), [t[..., :0] for t in a]), 'head dim must be from 1 to 256'),
])
def test_attention_refuses(change, message):
    a = attn_args()
    change(a)
    for fn in (td.ma_attn, td.ma_attn_train):
        with pytest.raises(RuntimeError, match=re.escape(message)):
            fn(*a)


@pytest.mark.parametrize('kw,message', [
    (dict(attn_mask=torch.zeros(5, 1, dtype=torch.bool)), 'attn_mask must be [Q, K] or [B, H, Q, K]'),
    (dict(attn_mask=torch.zeros(2, 5, 7, dtype=torch.bool)), 'attn_mask must be [Q, K] or [B, H, Q, K]'),
    (dict(attn_mask=torch.zeros(2, 2, 5, 7, dtype=torch.bool)), 'attn_mask must be [Q, K] or [B, H, Q, K]'),
    (dict(attn_mask=torch.zeros(5, 7, dtype=torch.float64)), 'attn_mask must be bool'),
    (dict(attn_mask=torch.zeros(5, 7, dtype=torch.int64)), 'attn_mask must be bool'),
    (dict(attn_mask=torch.zeros(5, 7, requires_grad=True)), 'attn_mask has no gradient'),
    (dict(key_padding_mask=torch.zeros(2, 6, dtype=torch.bool)), 'key_padding_mask must be bool [B, K]'),
    (dict(key_padding_mask=torch.zeros(2, 7)), 'key_padding_mask must be bool [B, K]'),
    (dict(scale=0.0), 'scale must be positive and finite'),
    (dict(scale=-1.0), 'scale must be positive and finite'),
    (dict(scale=float('nan')), 'scale must be positive and finite'),
    (dict(scale=float('inf')), 'scale must be positive and finite'),
])
def test_attention_refuses_masks_and_scales(kw, message):
    for fn in (td.ma_attn, td.ma_attn_train):
        with pytest.raises(RuntimeError, match=re.escape(message)):
            fn(*attn_args(), **kw)


@pytest.mark.parametrize('kw,message', [
    (dict(weight=torch.ones(5)), 'weight must be [C]'),
    (dict(bias=torch.ones(6, 1)), 'bias must be [C]'),
    (dict(residual=torch.ones(3, 6)), 'residual must have the shape of x'),
    (dict(weight=torch.ones(6).double()), 'all float tensors must have the same dtype'),
    (dict(x=torch.ones(4, 0)), 'channels must be from 1 to 16384'),
    (dict(x=torch.ones(2, 16385)), 'channels must be from 1 to 16384'),
    (dict(x=torch.ones(4, 6, dtype=torch.int32)), 'unsupported dtype'),
    (dict(x=torch.tensor(1.0)), 'x must be [..., C]'),
])
def test_layer_norm_refuses(kw, message):
    args = dict(dict(x=torch.randn(4, 6)), **kw)
    for fn in (td.ma_layer_norm, td.ma_layer_norm_train):
        with pytest.raises(RuntimeError, match=re.escape(message)):
            fn(**args)


def test_device_entries_refuse_cpu_tensors_and_a_missing_library(monkeypatch):
    a = attn_args()
    if _native.lib is not None:
        with pytest.raises(RuntimeError, match='inputs must be GPU tensors'):
            _dense.attn_forward(*a)
        with pytest.raises(RuntimeError, match='inputs must be GPU tensors'):
            _dense.layer_norm_forward(a[0], None, None)
    monkeypatch.setattr(_native, 'lib', None)
    with pytest.raises(RuntimeError, match='without its HIP extension'):
        _dense.attn_forward(*a)
    assert td.ma_attn(*a).shape == (2, 5, 32)  # CPU tensors still run the PyTorch path


# ---- the C ABI ----------------------------------------------------------------------------------------------------

def defines():
    text = open(HEADER).read() + open(os.path.join(ROOT, 'include', 'tinydeform.h')).read()
    return {k: int(v) for k, v in re.findall(r'#define\s+(TD_\w+)\s+(-?\d+)', text)}


@pytest.fixture(scope='module')
def lib():
    assert _native.lib is not None, _native.load_error
    return _native.lib


def test_header_library_and_binding_agree(lib):
    names = sorted(set(re.findall(r'^\s*int(?:64_t)?\s+(td_\w+)\s*\(', open(HEADER).read(), flags=re.M)))
    assert names == sorted(_dense.SIGNATURES)
    raw = ctypes.CDLL(_native.LIB_PATH)
    assert all(hasattr(raw, n) for n in names)
    d = defines()
    assert d['TD_ATTN_MAX_HEAD_DIM'] == _dense.MAX_HEAD_DIM and d['TD_NORM_MAX_CHANNELS'] == _dense.MAX_NORM_CHANNELS
    assert (d['TD_MASK_NONE'], d['TD_MASK_BYTES'], d['TD_MASK_FLOAT']) == \
        (_dense.MASK_NONE, _dense.MASK_BYTES, _dense.MASK_FLOAT)


P = 4096  # a stand-in address: these calls end before anything is read


def packed(dtype=1, kind=0, causal=0, B=2, Q=5, K=7, H=4, Hk=2, D=8, scale=1.0, q=P, k=P, v=P, mask=0, pad=0, out=P,
           stats=P, stride=8):
    return _dense.ATTN_ARGS.pack(dtype, kind, causal, 0, B, Q, K, H, Hk, D, scale, q, k, v, *([8] * 8), stride, mask, 0,
                                 0, 0, pad, out, stats, 0)


@pytest.mark.parametrize('kw,code,message', [
    (dict(dtype=4), 'TD_E_DTYPE', 'unknown dtype'), (dict(dtype=-1), 'TD_E_DTYPE', 'unknown dtype'),
    (dict(B=-1), 'TD_E_ARG', 'non-negative'), (dict(Hk=0), 'TD_E_ARG', 'at least one head'),
    (dict(H=3), 'TD_E_ARG', 'must divide'), (dict(D=0), 'TD_E_ARG', 'head dim'), (dict(D=257), 'TD_E_ARG', 'head dim'),
    (dict(Q=2 ** 31), 'TD_E_ARG', 'too many'), (dict(K=2 ** 31), 'TD_E_ARG', 'too many'),
    (dict(B=2 ** 20, Q=2 ** 20), 'TD_E_ARG', 'too many'), (dict(B=2 ** 31 - 1, Q=2 ** 31 - 1), 'TD_E_ARG', 'too many'),
    (dict(scale=0.0), 'TD_E_ARG', 'scale'), (dict(scale=float('nan')), 'TD_E_ARG', 'scale'),
    (dict(kind=3), 'TD_E_ARG', 'mask type'), (dict(kind=1), 'TD_E_ARG', 'null pointer'),
    (dict(q=0), 'TD_E_ARG', 'null pointer'), (dict(v=0), 'TD_E_ARG', 'null pointer'),
    (dict(out=0), 'TD_E_ARG', 'null pointer'), (dict(stride=-8), 'TD_E_ARG', 'strides'),
])
def test_attention_entries_reject_on_host(lib, kw, code, message):
    a = packed(**kw)
    assert lib.td_attn_forward(a, P, 1 << 40, None) == defines()[code]
    assert re.search(message, lib.td_last_error().decode())
    assert lib.td_attn_backward(a, P, P, P, P, P, 1 << 40, None) == defines()[code]


def test_attention_entries_check_pointers_and_workspaces(lib):
    E = defines()
    assert lib.td_attn_forward(None, None, 0, None) == E['TD_E_ARG']
    need = lib.td_attn_backward_workspace(packed())
    assert need > 0 and lib.td_attn_forward_workspace(packed()) >= 0
    assert lib.td_attn_backward(packed(), P, P, P, P, P, need - 1, None) == E['TD_E_WORKSPACE']
    assert lib.td_attn_backward(packed(), P, P, P, P, None, need, None) == E['TD_E_WORKSPACE']
    assert lib.td_attn_backward(packed(), None, P, P, P, P, need, None) == E['TD_E_ARG']
    assert lib.td_attn_backward(packed(stats=0), P, P, P, P, P, need, None) == E['TD_E_ARG']
    assert lib.td_attn_backward(packed(), P, P, P, None, P, need, None) == E['TD_E_ARG']
    assert lib.td_attn_forward(packed(Q=0), None, 0, None) == 0  # nothing to compute
    assert lib.td_attn_forward(packed(B=0), None, 0, None) == 0
    assert lib.td_attn_backward(packed(B=0), None, None, None, None, None, 0, None) == 0


def test_layer_norm_entries_reject_on_host(lib):
    E = defines()
    fwd, bwd = lib.td_layer_norm_forward, lib.td_layer_norm_backward
    assert fwd(4, P, None, P, P, P, P, 3, 8, 1e-5, None) == E['TD_E_DTYPE']
    assert fwd(1, P, None, P, P, P, P, -1, 8, 1e-5, None) == E['TD_E_ARG']
    assert fwd(1, P, None, P, P, P, P, 3, 0, 1e-5, None) == E['TD_E_ARG']
    assert fwd(1, P, None, P, P, P, P, 3, 16385, 1e-5, None) == E['TD_E_ARG']
    assert fwd(1, P, None, P, P, P, P, 3, 8, -1.0, None) == E['TD_E_ARG']
    assert fwd(1, None, None, P, P, P, P, 3, 8, 1e-5, None) == E['TD_E_ARG']
    assert fwd(1, None, None, None, None, None, None, 0, 8, 1e-5, None) == 0
    need = lib.td_layer_norm_backward_workspace(1, 1000, 256)
    assert need > 0
    assert bwd(1, P, None, P, P, P, P, P, P, 1000, 256, P, need - 1, None) == E['TD_E_WORKSPACE']
    assert bwd(1, P, None, P, None, P, P, P, P, 1000, 256, P, need, None) == E['TD_E_ARG']
