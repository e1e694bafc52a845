"""The decoder layer on the CPU: against HF transformers' RTDetrDecoderLayer run here in float64, its masks, and its
inference against its training path."""

import pytest
import torch

import marearts_tinydeform_amd as td
from decoder_cases import C, FFN, H, LEVELS, P, make, step

HF_ARGS = ('hidden_states', 'object_queries_position_embeddings', 'reference_points', 'spatial_shapes',
           'spatial_shapes_list', 'level_start_index', 'encoder_hidden_states')


def hf_layer():
    pytest.importorskip('transformers')
    from transformers import RTDetrConfig
    from transformers.models.rt_detr.modeling_rt_detr import RTDetrDecoderLayer
    cfg = RTDetrConfig(d_model=C, num_feature_levels=len(LEVELS), decoder_attention_heads=H, decoder_n_points=P,
                       decoder_ffn_dim=FFN, dropout=0.0, attention_dropout=0.0, activation_dropout=0.0)
    cfg.disable_custom_kernels = True
    cfg._attn_implementation = 'eager'
    return RTDetrDecoderLayer(cfg).double()


@pytest.mark.parametrize('masked', [False, True])
def test_matches_transformers_with_gradients(masked):
    layer, args, grad = make()
    hf = hf_layer()
    hf.load_state_dict(layer.state_dict())
    args = {n: args[n] for n in HF_ARGS + ('encoder_attention_mask',)}
    args['encoder_attention_mask'] = torch.zeros(21, 21, dtype=torch.float64).masked_fill(
        args['encoder_attention_mask'], -1e30)[None, None] if masked else None
    out, grads = step(layer, args, grad)
    want, wgrads = step(hf, args, grad)
    torch.testing.assert_close(out, want, rtol=1e-10, atol=1e-11)
    assert grads.keys() == wgrads.keys()
    for n in grads:
        torch.testing.assert_close(grads[n], wgrads[n], rtol=1e-9, atol=1e-10, msg=lambda m: f'{n}: {m}')


def test_inference_is_training_and_a_bool_mask_is_a_float_one():
    layer, args, grad = make()
    out, _ = step(layer, args, grad)
    with torch.inference_mode():
        torch.testing.assert_close(layer(**args), out, rtol=1e-12, atol=1e-13)
        mask = torch.zeros(21, 21, dtype=torch.float64).masked_fill(args['encoder_attention_mask'], -torch.inf)
        torch.testing.assert_close(layer(**{**args, 'encoder_attention_mask': mask}), out, rtol=1e-12, atol=1e-13)


def test_padded_queries_and_tokens_are_not_seen():
    layer, args, _ = make()
    other = dict(args)
    other['hidden_states'] = args['hidden_states'].clone()
    other['hidden_states'][1, 18:] += 3.0
    other['encoder_hidden_states'] = args['encoder_hidden_states'].clone()
    other['encoder_hidden_states'][0, 300:] = 7.0
    with torch.inference_mode():
        a, b = layer(**args), layer(**other)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1, :18], b[1, :18])
        seen = layer(**{**other, 'query_padding_mask': None, 'memory_padding_mask': None})
    assert not torch.allclose(a[0], seen[0]) and not torch.allclose(a[1, :18], seen[1, :18])


def test_self_attention_refuses_heads_that_do_not_divide():
    with pytest.raises(ValueError, match='divisible'):
        td.SelfAttnLayer(66, 4)
