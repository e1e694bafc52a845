"""The decoder layer on the GPU: self-attention, deformable attention, the norms and their gradients as one training
step and as inference, against the same layer in float64 on the CPU.

Tolerances, in units of the largest relative error u of one rounding and of the root mean square of the tensor compared:
between its input and its output the layer rounds at most 32 times to its type (the embeddings' sum, per sublayer the
projections' results, the cores, the output projections, the norms; softmax weights and their logits), each keeping the
scale of what it rounds, for the norms hold it at one: 32 u. A gradient passes the same roundings once more on its way
back: 64 u. In float32 the sums over up to 320 terms round as often as they have terms, their errors growing like the
square root of that: times 18.
"""

import pytest
import torch

from decoder_cases import cast, make, step

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 18 * 2 ** -24, torch.float16: 2 ** -11, torch.bfloat16: 2 ** -8}


def close(name, got, want, tol):
    got = got.detach().double().cpu()
    err = (got - want).square().mean().sqrt() / want.square().mean().sqrt()
    print(f'  {name}: {err:.3g} of {tol:.3g}', flush=True)
    assert err <= tol, f'{name}: relative error {err:.3g}, allowed {tol:.3g}'


@pytest.mark.parametrize('dtype', list(HALF_STEP))
def test_training_step_and_inference(dtype):
    layer, args, grad = make(dtype)
    want, wgrads = step(layer, args, grad)
    layer, args = layer.to('cuda', dtype), cast(args, dtype, 'cuda')
    out, grads = step(layer, args, grad.to('cuda', dtype))
    close('out', out, want.detach(), 32 * HALF_STEP[dtype])
    assert grads.keys() == wgrads.keys()
    for n in grads:
        if n == 'self_attn.k_proj.bias':  # adding a constant to every key moves no softmax: exactly zero
            continue
        close(n, grads[n], wgrads[n], 64 * HALF_STEP[dtype])
    with torch.inference_mode():
        close('inference', layer(**args), want.detach(), 32 * HALF_STEP[dtype])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_graphs_replay_the_layer(dtype):
    """Inference and a training step, each captured, replayed in turn with eager work in between."""
    layer, args, grad = make(dtype)
    layer, args, grad = layer.to('cuda', dtype), cast(args, dtype, 'cuda'), grad.to('cuda', dtype)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step(layer, args, grad)
            with torch.inference_mode():
                layer(**args)
    torch.cuda.current_stream().wait_stream(s)
    want, wgrads = step(layer, args, grad)
    want = want.detach()
    train, serve = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(train):
        out, grads = step(layer, args, grad)
        out = out.detach()
    with torch.inference_mode():
        still = layer(**args)
        with torch.cuda.graph(serve):
            served = layer(**args)
    for i in range(3):
        with torch.inference_mode():
            for t in (out, *grads.values(), served):
                t.zero_()
        train.replay()
        serve.replay()
        with torch.inference_mode():
            assert torch.equal(layer(**args), still)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(served, still), f'replay {i}'
        for n in grads:
            # deformable attention adds its gradients with atomics, in any order
            tol = 64 * HALF_STEP[dtype]
            if n != 'self_attn.k_proj.bias':
                close(f'replay {i} {n}', grads[n], wgrads[n].double().cpu(), tol)
