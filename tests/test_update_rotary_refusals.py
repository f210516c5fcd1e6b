"""``KIVIKVCache.update_rotary``: a refused call counts nothing, and blocks with derivatives are taken whatever their length."""

from __future__ import annotations

import pytest
import torch

from veloxquant_mlx_b200 import VQLibraryError, kernels
from veloxquant_mlx_b200.cache import KIVIKVCache, KVCacheConfig
from veloxquant_mlx_b200.rotary import RotaryEmbedding


def _cache(**kw):
    return KIVIKVCache(KVCacheConfig(method="kivi", head_dim=64, bit_width_inlier=4, residual_length=64, fused_sdpa_memory_bound=True, **kw))


def _block(S, device="cpu", B=1, seed=0):
    g = torch.Generator(device).manual_seed(seed)
    return [torch.randn(B, h, S, 64, device=device, generator=g).half() for h in (4, 2, 2)]


def _held(c):
    return c.offset, c._n_quantized, c._n_res, c.nbytes


def test_counters_stay_when_the_append_is_refused(monkeypatch):
    monkeypatch.setattr(kernels, "kivi_available", lambda: True)  # (the host logic over CPU tensors: the append itself asks for a device)
    c, rope = _cache(), RotaryEmbedding(64)
    for _ in range(2):
        with pytest.raises(VQLibraryError):
            c.update_rotary(*_block(5), rope)
        assert _held(c) == (0, 0, 0, 0)
    _, k, v = _block(9)
    c.update_and_fetch(k, v)
    held, rows = _held(c), [t.clone() for t in c._live_res()]
    for S in (1, 30, 90):  # into the window, and past it
        with pytest.raises(VQLibraryError):
            c.update_rotary(*_block(S), rope)
        assert _held(c) == held
    inside = c._k_res[:, :, :1]
    with pytest.raises((ValueError, VQLibraryError)):
        c.update_rotary(_block(1)[0], inside, _block(1)[2], rope)
    assert _held(c) == held and all(torch.equal(a, b) for a, b in zip(rows, c._live_res()))
    c.update_and_fetch(k, v)
    assert c.offset == c._n_res == 18


@pytest.mark.gpu
def test_counters_stay_on_the_device():
    c, rope = _cache(), RotaryEmbedding(64, device="cuda")
    c.update_rotary(*_block(100, "cuda"), rope)
    held, state = _held(c), [t.clone() for t in c.state]
    q, k, v = _block(1, "cuda")
    with pytest.raises(ValueError, match="share memory"):
        c.update_rotary(q, c._k_res[:, :, :1], v, rope)
    with pytest.raises(ValueError, match="positions must be"):
        c.update_rotary(q, k, v, rope, torch.zeros(2, dtype=torch.int64, device="cuda"))
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="inside a graph capture"), torch.cuda.graph(graph):
        c.update_rotary(q, k, v, RotaryEmbedding(64))
    assert _held(c) == held and all(torch.equal(a, b) for a, b in zip(state, c.state))
    # the tokens that follow stand where they would have stood
    other = _cache()
    other.update_rotary(*_block(100, "cuda"), rope)
    for step in range(40):
        block = _block(1, "cuda", seed=step)
        a, b = c.update_rotary(*block, rope)[0], other.update_rotary(*block, rope)[0]
        assert torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(c.state, other.state))


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [(100, 1, 5), (1, 3, 200)])
def test_blocks_with_derivatives(lengths):
    rope, c, plain = RotaryEmbedding(64), _cache(), _cache()
    for i, S in enumerate(lengths):
        q, k, v = _block(S, "cuda", seed=i)
        with torch.no_grad():
            want = plain.update_rotary(q, k, v, rope)[0]
            turned_back = rope(torch.ones_like(want), positions=plain.offset - S, inverse=True)
        q.requires_grad_(True)
        k.requires_grad_(True)
        got = c.update_rotary(q, k, v, rope)[0]
        got.sum().backward()
        assert torch.equal(got, want) and torch.equal(q.grad, turned_back) and k.grad is None
        assert not c._k_res.requires_grad
    assert all(torch.equal(a, b) for a, b in zip(c.state, plain.state))
