"""The scaling dictionaries of model configurations: every key that changes frequencies or their factor counts or is refused."""

from __future__ import annotations

import math

import pytest
import torch

from veloxquant_mlx_b200.rotary import RotaryEmbedding, rotary_frequencies

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


@pytest.mark.parametrize("scaling", [
    {**YARN, "rope_theta": 10000.0, "mscale": 1.0, "mscale_all_dim": 1.0},
    {**YARN, "rope_theta": 10000.0, "mscale": 0.707, "mscale_all_dim": 1.0, "beta_fast": 32, "beta_slow": 1},
    {**YARN, "rope_theta": 10000.0, "mscale": 1.0},
    {**YARN, "rope_theta": 10000.0, "mscale_all_dim": 1.0},
    {**YARN, "rope_theta": 10000.0, "mscale": 1.0, "mscale_all_dim": 0.0},
    {**YARN, "rope_theta": 10000.0, "mscale": 1.0, "mscale_all_dim": 0.5, "attention_factor": 1.5},
    {**YARN, "rope_theta": 500000.0, "truncate": False},
    {**YARN, "rope_theta": 500000.0, "truncate": False, "mscale": 0.5, "mscale_all_dim": 2.0},
    {**YARN, "rope_theta": 150000.0, "beta_fast": None, "beta_slow": None},
    {"rope_type": "llama3", "rope_theta": 500000.0, "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
    {"rope_type": "linear", "rope_theta": 1000000.0, "factor": 4.0},
    {"rope_type": "default", "rope_theta": 500000.0},
])
def test_frequencies_and_factor_are_those_a_transformers_model_uses(scaling):
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding

    theirs = LlamaRotaryEmbedding(LlamaConfig(hidden_size=512, num_attention_heads=4, max_position_embeddings=163840, rope_parameters=dict(scaling)))
    for f, m in (rotary_frequencies(128, scaling=scaling), rotary_frequencies(128, scaling["rope_theta"], scaling)):
        # float32 frequencies: a few roundings of base ** x and of the ramp, each at most 2^-24
        assert torch.allclose(f.float(), theirs.inv_freq, rtol=2e-6, atol=0) and m == pytest.approx(theirs.attention_scaling, rel=1e-12)
    rope = RotaryEmbedding(128, scaling=scaling)
    assert torch.equal(rope.inv_freq, f) and rope.attention_factor == m


def test_the_factor_of_yarn_by_formula():
    ln = math.log(40.0)
    for extra, want in (({}, 0.1 * ln + 1), ({"mscale": 1, "mscale_all_dim": 1}, 1.0), ({"mscale": 2, "mscale_all_dim": 0.5}, (0.2 * ln + 1) / (0.05 * ln + 1)),
                        ({"mscale": 2}, 0.1 * ln + 1), ({"mscale": 2, "mscale_all_dim": None}, 0.1 * ln + 1), ({"attention_factor": 0.25}, 0.25),
                        ({"attention_factor": None, "mscale": 1, "mscale_all_dim": 1}, 1.0)):
        assert rotary_frequencies(64, scaling={**YARN, **extra})[1] == pytest.approx(want, rel=1e-15)
    assert rotary_frequencies(64, scaling={**YARN, "factor": 0.5, "mscale": 3, "mscale_all_dim": 1})[1] == 1.0


def test_the_base_is_the_dictionary_s():
    theta = {"rope_type": "default", "rope_theta": 500000.0}
    assert torch.equal(rotary_frequencies(128, scaling=theta)[0], rotary_frequencies(128, 500000.0)[0])
    assert torch.equal(rotary_frequencies(128)[0], rotary_frequencies(128, 10000.0)[0])
    assert torch.equal(RotaryEmbedding(128, scaling=theta).inv_freq, RotaryEmbedding(128, base=500000.0).inv_freq)
    for call in (lambda: rotary_frequencies(128, 10000.0, theta), lambda: RotaryEmbedding(128, base=10000.0, scaling=theta)):
        with pytest.raises(ValueError, match="contradicts rope_theta"):
            call()


@pytest.mark.parametrize("scaling,what", [
    ({"rope_type": "linear", "factor": 2.0, "partial_rotary_factor": 0.5}, "partial_rotary_factor"),
    ({"rope_type": "default", "factor": 2.0}, "does not take 'factor'"),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 64, "mscale": 1.0}, "mscale"),
    ({**YARN, "mscale_all": 1.0}, "mscale_all"), ({"mrope_section": [16, 24, 24]}, "mrope_section"), ({"full_attention": {"rope_type": "default"}}, "full_attention"),
    ({**YARN, "factor": None}, "needs 'factor'"), ({**YARN, "beta_slow": 0.0}, "beta_slow"), ({**YARN, "rope_theta": 1.0}, "other than 1"),
    ({**YARN, "original_max_position_embeddings": 0}, "must be positive"),
])
def test_keys_that_are_not_known_are_refused(scaling, what):
    with pytest.raises(ValueError, match=what):
        rotary_frequencies(64, scaling=scaling)


def test_keys_without_an_effect_are_taken():
    f, _ = rotary_frequencies(64, scaling={"type": "linear", "rope_type": "linear", "factor": 2.0, "original_max_position_embeddings": 64,
                                           "max_position_embeddings": 128, "finetuned": True, "mscale": None})
    assert torch.equal(f, rotary_frequencies(64)[0] / 2)


def test_part_of_the_head_by_its_factor():
    part = {"rope_type": "default", "partial_rotary_factor": 0.25}
    assert RotaryEmbedding(128, scaling=part).rotary_dim == RotaryEmbedding(128, scaling=part, rotary_dim=32).rotary_dim == 32
    assert torch.equal(RotaryEmbedding(128, scaling=part).inv_freq, rotary_frequencies(32)[0])
    with pytest.raises(ValueError, match="contradicts partial_rotary_factor"):
        RotaryEmbedding(128, scaling=part, rotary_dim=64)
    with pytest.raises(ValueError, match="rotary_dim"):
        RotaryEmbedding(128, scaling={"partial_rotary_factor": 1.5})


@pytest.mark.parametrize("kind", ["float64 tensor", "float64 array"])
def test_given_frequencies_are_the_embedding_s_own(kind):
    import numpy as np

    given = torch.linspace(1, 0.1, 8, dtype=torch.float64) if kind == "float64 tensor" else np.linspace(1, 0.1, 8)
    rope, want = RotaryEmbedding(16, inv_freq=given), torch.as_tensor(given).clone()
    given *= 0  # the caller's buffer is used again
    assert torch.equal(rope.inv_freq, want)
    rope.inv_freq.zero_()  # and what the property gives is a copy
    assert torch.equal(rope.inv_freq, want)
