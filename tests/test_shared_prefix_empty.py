"""Stores without heads are refused, and calls without query rows return before the device is asked for work."""

from __future__ import annotations

import pytest
import torch

from veloxquant_mlx_b200.kernels import KiviRows


def test_a_store_without_heads():
    z = torch.zeros(1, 0, 5, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="at least one kv head"):
        KiviRows(k_res=z, v_res=z.clone())
    assert len(KiviRows(k_res=torch.zeros(0, 2, 5, 128, dtype=torch.float16), v_res=torch.zeros(0, 2, 5, 128, dtype=torch.float16))) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,S", [(0, 4, 1), (3, 0, 1), (3, 4, 0)])
def test_calls_without_query_rows(B, H, S):
    from veloxquant_mlx_b200.kernels import kivi_shared_prefix_attend

    pre, own = ([torch.zeros(b, 2, 5, 128, dtype=torch.float16, device="cuda") for _ in range(2)] for b in (1, B))
    q = torch.zeros(B, H, S, 128, dtype=torch.float16, device="cuda")
    out, lse = kivi_shared_prefix_attend(q, KiviRows(k_res=pre[0], v_res=pre[1]), KiviRows(k_res=own[0], v_res=own[1]), 0.1, return_lse=True)
    assert out.shape == q.shape and lse.shape == (B, H, S)
