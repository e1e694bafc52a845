"""A decoder layer and its inputs for tests/test_decoder.py (CPU) and tests/test_gpu_decoder.py."""

import torch

import marearts_tinydeform_amd as td

C, H, P, FFN = 64, 4, 4, 128
LEVELS = [(16, 16), (8, 8)]


def make(dtype=torch.float64, B=2, Q=21, seed=0):
    """(layer, args of its forward): parameters and inputs of `dtype`'s values held in float64.

    The offsets are the module's own grid (their weights are zero, so rounding does not move a sample) and the reference
    points lie a quarter of a pixel past a token's centre on the first level, three eighths off on the second: no sample
    sits where bilinear sampling has a kink, and gradients of 16-bit inputs can be compared with exact ones.
    """
    g = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64).to(dtype).double()

    layer = td.DeformDecoderLayer(C, len(LEVELS), H, P, FFN).double()
    with torch.no_grad():
        for name, p in layer.named_parameters():
            if 'sampling_offsets' in name:
                continue
            if p.dim() == 2:
                p.copy_((randn(*p.shape) * p.shape[1] ** -0.5).to(dtype))
            elif 'layer_norm.weight' in name:
                p.copy_((1 + 0.1 * randn(*p.shape)).to(dtype))
            else:
                p.copy_((0.1 * randn(*p.shape)).to(dtype))
    shapes = torch.tensor(LEVELS)
    starts = torch.tensor([0, 256])
    N = 320
    cell = torch.randint(0, 16, (B, Q, 1, 2), generator=g)
    ref = (4 * cell + 3).double() / 64
    padded_q = torch.zeros(B, Q, dtype=torch.bool)
    padded_q[1, Q - 3:] = True
    padded_m = torch.zeros(B, N, dtype=torch.bool)
    padded_m[0, 300:] = True
    groups = torch.arange(Q) // 8  # denoising groups, which do not see each other
    args = dict(hidden_states=randn(B, Q, C), object_queries_position_embeddings=randn(B, Q, C), reference_points=ref,
                spatial_shapes=shapes, spatial_shapes_list=LEVELS, level_start_index=starts,
                encoder_hidden_states=randn(B, N, C), encoder_attention_mask=groups[:, None] != groups[None],
                query_padding_mask=padded_q, memory_padding_mask=padded_m)
    return layer, args, randn(B, Q, C)


def step(layer, args, grad):
    """(out, gradients by name) of a training step: of the inputs and every parameter"""
    leaves = {n: args[n] for n in ('hidden_states', 'object_queries_position_embeddings', 'encoder_hidden_states')}
    leaves = {n: t.detach().clone().requires_grad_() for n, t in leaves.items()}
    out = layer(**{**args, **leaves})
    leaves.update(layer.named_parameters())
    return out, dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), grad)))


def cast(args, dtype, device):
    return {n: t.to(device, dtype if t.is_floating_point() else t.dtype) if isinstance(t, torch.Tensor) else t
            for n, t in args.items()}
