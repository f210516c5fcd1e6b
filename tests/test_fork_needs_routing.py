"""A memory-bound cache behind a model that was not routed to ``veloxquant_attention`` fails instead of attending over nothing."""

from __future__ import annotations

import pytest
import torch

from veloxquant_mlx_b200 import integration as I


class _Bound:
    """What a memory-bound cache looks like to the layer."""

    _memory_bound = True
    offset = 3

    def update_and_fetch(self, k, v):
        z = k.new_zeros((*k.shape[:2], 0, k.shape[3]))
        return z, z

    def fused_sdpa(self, q, scale, causal=True, sliding_window=0):
        return torch.ones_like(q)


@pytest.mark.parametrize("gqa", [False, True])
def test_dense_attention_over_the_sentinels_raises(gqa):
    pytest.importorskip("transformers")
    layer = I.make_cache_layer_class()(_Bound())
    q, k = torch.randn(2, 4, 1, 64), torch.randn(2, 2, 1, 64)
    keys, values = layer.update(k, k.clone())
    assert keys.shape[-2] == 0 and keys.velox_cache is layer.cache
    wide = [x if gqa else x[:, :, None].expand(2, 2, 2, *x.shape[2:]).reshape(2, 4, *x.shape[2:]) for x in (keys, values)]
    with pytest.raises(RuntimeError):
        torch.nn.functional.scaled_dot_product_attention(q, *wide, enable_gqa=gqa)
    if not gqa:
        with pytest.raises(RuntimeError):
            torch.softmax(q @ wide[0].transpose(2, 3), -1) @ wide[1]
    out, _ = I.veloxquant_attention(torch.nn.Module(), q, keys, values, None)
    assert torch.equal(out, torch.ones(2, 1, 4, 64))
    with pytest.raises(RuntimeError, match="without a cache reference"):
        I.veloxquant_attention(torch.nn.Module(), q, keys.clone(), values, None)


def test_only_layers_of_this_package_are_forked():
    pytest.importorskip("transformers")
    from transformers.cache_utils import Cache, DynamicLayer

    with pytest.raises(ValueError, match="DynamicLayer"):
        I.fork_hf_cache(Cache(layers=[DynamicLayer()]), 2)


@pytest.mark.gpu
@pytest.mark.parametrize("implementation", ["sdpa", "eager"])
@pytest.mark.parametrize("layers", [1, 2])
def test_a_fork_of_a_standard_cache(layers, implementation):
    pytest.importorskip("transformers")
    from transformers import LlamaConfig, LlamaForCausalLM

    from veloxquant_mlx_b200.cache import KVCacheConfig

    torch.manual_seed(0)
    model = LlamaForCausalLM(LlamaConfig(hidden_size=128, intermediate_size=128, num_hidden_layers=layers, num_attention_heads=2, num_key_value_heads=1,
                                         head_dim=64, vocab_size=64, attn_implementation=implementation)).to("cuda", torch.float16).eval()
    cfg = KVCacheConfig(method="kivi", head_dim=64, bit_width_inlier=8, residual_length=32)  # (standard mode)
    prompt, ask = torch.randint(0, 64, (1, 50), device="cuda"), torch.randint(0, 64, (3, 1), device="cuda")
    with torch.no_grad():
        cache = I.make_hf_cache(model, cfg)
        model(prompt, past_key_values=cache, use_cache=True)
        fork = I.fork_hf_cache(cache, 3)
        with pytest.raises(RuntimeError):
            model(ask, past_key_values=fork, use_cache=True)
        # routed, the same fork attends over the prompt
        I.patch_hf_for_fused_sdpa(model)
        fork = I.fork_hf_cache(cache, 3)
        got = model(ask, past_key_values=fork, use_cache=True).logits[:, -1]
        for b in range(3):
            alone = I.make_hf_cache(model, cfg)
            model(prompt, past_key_values=alone, use_cache=True)
            want = model(ask[b : b + 1], past_key_values=alone, use_cache=True).logits[0, -1]
            # the same 8-bit codes (a step is 2^-8 of a group's range) and float16 activations: 2^-6 of the largest logit
            assert float((got[b].float() - want.float()).abs().max()) < 2.0**-6 * float(want.float().abs().max())
