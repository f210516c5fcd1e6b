"""Rotary positions without a GPU: the frequencies of every scaling against formulas restated here in
64 bits, and the calls that are refused before the device is looked at."""

from __future__ import annotations

import math

import pytest
import torch

from veloxquant_mlx_b200 import VQLibraryError
from veloxquant_mlx_b200.rotary import RotaryEmbedding, rotary_frequencies


@pytest.mark.parametrize("r", [2, 6, 64, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_default_and_linear_and_ntk(r, base):
    plain = [base ** (-2 * i / r) for i in range(r // 2)]
    f, m = rotary_frequencies(r, base)
    assert m == 1.0 and f.dtype == torch.float64 and f.tolist() == pytest.approx(plain, rel=1e-14)
    f, m = rotary_frequencies(r, base, {"rope_type": "linear", "factor": 4.0})
    assert m == 1.0 and f.tolist() == pytest.approx([x / 4 for x in plain], rel=1e-14)
    f, _ = rotary_frequencies(r, base, {"rope_type": "ntk", "factor": 4.0})
    if r > 2:  # the slowest pair is stretched by the factor, the fastest kept
        assert f[0] == 1.0 and f[-1].item() == pytest.approx(plain[-1] / 4, rel=1e-12)


def test_llama3_ramp():
    r, base, sc = 128, 500000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                  "original_max_position_embeddings": 8192}
    f, m = rotary_frequencies(r, base, sc)
    assert m == 1.0
    for i in range(r // 2):
        w = base ** (-2 * i / r)
        wavelength = 2 * math.pi / w
        if wavelength < 8192 / 4:
            want = w
        elif wavelength > 8192:
            want = w / 8
        else:
            smooth = (8192 / wavelength - 1) / 3
            want = (1 - smooth) * w / 8 + smooth * w
        assert f[i].item() == pytest.approx(want, rel=1e-12)


@pytest.mark.parametrize("given", [None, 1.25])
def test_yarn_ramp_and_factor(given):
    r, base, old, factor = 64, 10000.0, 4096, 16.0
    sc = {"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": old}
    if given is not None:
        sc["attention_factor"] = given
    f, m = rotary_frequencies(r, base, sc)
    assert m == pytest.approx(given if given is not None else 0.1 * math.log(16) + 1)
    # pair i makes old * w / 2 pi turns; pairs that make more than 32 are kept, fewer than 1 stretched
    index = lambda turns: r * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = math.floor(index(32)), math.ceil(index(1))
    for i in range(r // 2):
        w = base ** (-2 * i / r)
        t = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        assert f[i].item() == pytest.approx(w * (1 - t) + w / factor * t, rel=1e-12)


@pytest.mark.parametrize("scaling", [
    {"rope_type": "llama3", "rope_theta": 10000.0, "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "rope_theta": 10000.0, "factor": 4.0, "original_max_position_embeddings": 2048},
    {"rope_type": "linear", "rope_theta": 10000.0, "factor": 4.0},
    {"rope_type": "default", "rope_theta": 10000.0},
])
def test_frequencies_are_those_a_transformers_model_uses(scaling):
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding

    cfg = LlamaConfig(hidden_size=256, num_attention_heads=4, max_position_embeddings=8192, rope_parameters=dict(scaling))
    theirs = LlamaRotaryEmbedding(cfg)
    f, m = rotary_frequencies(64, 10000.0, scaling)
    # float32 frequencies: a few roundings of base ** x and of the ramp, each at most 2^-24
    assert torch.allclose(f.float(), theirs.inv_freq, rtol=2e-6, atol=0) and m == pytest.approx(theirs.attention_scaling)


def test_bad_descriptions_are_refused():
    with pytest.raises(ValueError, match="even"):
        rotary_frequencies(7)
    with pytest.raises(ValueError, match="unknown rope_type"):
        rotary_frequencies(8, scaling={"rope_type": "spiral", "factor": 2.0})
    with pytest.raises(ValueError, match="needs 'factor'"):
        rotary_frequencies(8, scaling={"rope_type": "linear"})
    with pytest.raises(ValueError, match="original_max_position_embeddings"):
        rotary_frequencies(8, scaling={"rope_type": "yarn", "factor": 2.0})
    with pytest.raises(ValueError, match="exceed low_freq_factor"):
        rotary_frequencies(8, scaling={"rope_type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0,
                                       "original_max_position_embeddings": 64})
    with pytest.raises(ValueError, match="positive"):
        rotary_frequencies(8, base=0.0)
    for kw in (dict(rotary_dim=0), dict(rotary_dim=130), dict(rotary_dim=31)):
        with pytest.raises(ValueError, match="rotary_dim"):
            RotaryEmbedding(128, **kw)
    with pytest.raises(ValueError, match="layout"):
        RotaryEmbedding(128, layout="spiral")
    with pytest.raises(ValueError, match="shape"):
        RotaryEmbedding(128, inv_freq=torch.ones(63))
    with pytest.raises(ValueError, match="not both"):
        RotaryEmbedding(128, inv_freq=torch.ones(64), scaling={"rope_type": "default"})


def test_bad_calls_are_refused_before_the_device_is_looked_at():
    rope = RotaryEmbedding(16)
    q, k = torch.zeros(2, 4, 3, 16), torch.zeros(2, 2, 3, 16)
    bad = [
        ((torch.zeros(4, 3, 16),), "must be"), ((torch.zeros(2, 4, 3, 8),), "must be"), ((q.double(),), "unsupported dtype"),
        ((q, k[:1]), "must agree"), ((q, k[:, :, :2]), "must agree"), ((q, k.half()), "must agree"),
    ]
    for args, what in bad:
        with pytest.raises(ValueError, match=what):
            rope(*args)
    for pos in (torch.zeros(3), 1.5, torch.zeros(3, dtype=torch.int16)):
        with pytest.raises(ValueError, match="int32 / int64"):
            RotaryEmbedding._positions("x", pos, 2, 3, q.device)
    for shape in ((2,), (3, 2), (2, 1), (1,), (2, 1, 3)):
        with pytest.raises(ValueError, match="positions must be"):
            RotaryEmbedding._positions("x", torch.zeros(shape, dtype=torch.int64), 2, 3, q.device)
    with pytest.raises(VQLibraryError):
        rope(q, k)
    with pytest.raises(VQLibraryError):
        rope(q.requires_grad_(True), k)


def test_bad_appends_are_refused():
    rope = RotaryEmbedding(16)
    q, k, v, kr, vr = torch.zeros(2, 4, 3, 16), torch.zeros(2, 2, 3, 16), torch.zeros(2, 2, 3, 16), torch.zeros(2, 2, 8, 16), torch.zeros(2, 2, 8, 16)
    with pytest.raises(ValueError, match="must be like k"):
        rope.append(q, k, v[:, :1], kr, vr, 0)
    with pytest.raises(ValueError, match="not differentiable"):
        rope.append(q, k.clone().requires_grad_(True), v, kr, vr, 0)
    with pytest.raises(ValueError, match="exceed k_res"):
        rope.append(q, k, v, kr, vr, 6)
    with pytest.raises(ValueError, match="exceed k_res"):
        rope.append(q, k, v, kr, vr, -1)
    with pytest.raises(ValueError, match="v_res must be"):
        rope.append(q, k, v, kr, vr.half(), 0)
    with pytest.raises(ValueError, match="rows apart"):
        rope.append(q, k, v, torch.zeros(2, 1, 8, 16).expand(2, 2, 8, 16), vr, 0)
    with pytest.raises(VQLibraryError):
        rope.append(q, k, v, kr, vr, 0)
