"""Copied and reloaded embeddings: a frequency table is used on the device it lies on, or made anew."""

from __future__ import annotations

import copy
import io

import pytest
import torch

from veloxquant_mlx_b200.rotary import RotaryEmbedding


def _reload(rope, where):
    buffer = io.BytesIO()
    torch.save(rope, buffer)
    buffer.seek(0)
    return torch.load(buffer, map_location=where, weights_only=False)


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda r: _reload(r, "cpu"), lambda r: _reload(r, None)])
def test_a_table_in_host_memory_is_dropped(again):
    rope = RotaryEmbedding(64, rotary_dim=32, layout="interleaved", attention_factor=1.5)
    rope._turns[0] = torch.zeros(16, dtype=torch.float64)  # what a load to the host leaves of device 0's table
    other = again(rope)
    assert other._turns == {} and torch.equal(other.inv_freq, rope.inv_freq)
    assert (other.head_dim, other.rotary_dim, other.layout, other.attention_factor) == (64, 32, "interleaved", 1.5)
    with pytest.raises(Exception, match="CUDA"):
        other(torch.zeros(1, 1, 1, 64))


@pytest.mark.gpu
def test_copies_and_reloads_turn_alike():
    rope = RotaryEmbedding(64, inv_freq=torch.linspace(1, 0.01, 32, device="cuda", dtype=torch.float64))
    q = torch.randn(2, 3, 5, 64, device="cuda")
    want = rope(q, positions=9)
    for other in (copy.copy(rope), copy.deepcopy(rope), _reload(rope, "cpu"), _reload(rope, None)):
        assert all(t.is_cuda for t in other._turns.values())
        assert torch.equal(other(q, positions=9), want)
