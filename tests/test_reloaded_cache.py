"""A KIVI cache that was loaded to another device refuses keys of the one it came from; nothing off its device reaches a kernel."""

from __future__ import annotations

import io

import pytest
import torch

from veloxquant_mlx_b200 import kernels
from veloxquant_mlx_b200.cache import KIVIKVCache, KVCacheConfig


class _OnDevice:
    """Keys as the flush sees them: rows on a CUDA device (their address is never used)."""

    is_cuda, dtype, device = True, torch.float16, torch.device("cuda", 0)

    def __init__(self, *shape):
        self.shape = torch.Size(shape)

    def stride(self):
        return torch.empty(self.shape, device="meta").stride()

    def data_ptr(self):
        raise AssertionError("a block's address was taken for a launch over buffers on the host")

    def __getitem__(self, at):
        return self


def test_the_flush_looks_at_the_buffers_device(monkeypatch):
    monkeypatch.setattr(kernels, "kivi_available", lambda: True)
    monkeypatch.setattr(kernels, "kivi_quantize_into", lambda x, *a, codes, **kw: (_ for _ in ()).throw(ValueError(f"{codes.device} {x.device}")))
    c = KIVIKVCache(KVCacheConfig(method="kivi", head_dim=64, bit_width_inlier=4, residual_length=0, fused_sdpa_memory_bound=True))
    c._ensure_capacity(1, 2, 64, 64, "cpu", torch.float16)
    with pytest.raises(ValueError, match="cpu cuda:0"):
        c._quantize_rows(_OnDevice(1, 2, 32, 64), _OnDevice(1, 2, 32, 64), 32)


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [0, 32])
def test_a_cache_loaded_to_the_host(residual):
    block = lambda S: [torch.randn(1, 2, S, 64, device="cuda").half() for _ in range(2)]  # noqa: E731
    c = KIVIKVCache(KVCacheConfig(method="kivi", head_dim=64, bit_width_inlier=4, residual_length=residual, fused_sdpa_memory_bound=True))
    c.update_and_fetch(*block(96))
    buffer = io.BytesIO()
    torch.save(c, buffer)
    buffer.seek(0)
    host = torch.load(buffer, map_location="cpu", weights_only=False)
    assert host._k_codes.device.type == "cpu" and host.offset == 96
    q = torch.randn(1, 4, 1, 64, device="cuda").half()
    with pytest.raises(ValueError):
        host.fused_sdpa(q, 0.1)
    if residual == 0:
        with pytest.raises(ValueError):
            host.update_and_fetch(*block(64))
        assert host.offset == 96
    buffer.seek(0)
    back = torch.load(buffer, weights_only=False)
    assert torch.equal(back.fused_sdpa(q, 0.1), c.fused_sdpa(q, 0.1))
