"""Calls without derivatives refuse tensors that carry one, in reverse and in forward mode, before the device is looked at."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from veloxquant_mlx_b200 import VQLibraryError
from veloxquant_mlx_b200.kernels import KiviRows, kivi_shared_prefix_attend
from veloxquant_mlx_b200.rotary import RotaryEmbedding


def _store(B, leaf=None):
    t = dict(k_codes=torch.zeros(B, 2, 64, 64, dtype=torch.uint8), k_scale=torch.zeros(B, 2, 2, 128), k_zero=torch.zeros(B, 2, 2, 128),
             v_codes=torch.zeros(B, 2, 64, 64, dtype=torch.uint8), v_scale=torch.zeros(B, 2, 64, 4), v_zero=torch.zeros(B, 2, 64, 4),
             k_res=torch.zeros(B, 2, 5, 128, dtype=torch.float16), v_res=torch.zeros(B, 2, 5, 128, dtype=torch.float16))
    if leaf:
        t[leaf].requires_grad_(True)
    return t


@pytest.mark.parametrize("leaf", ["k_res", "v_res", "k_scale", "k_zero", "v_scale", "v_zero", "q"])
def test_attention_behind_a_shared_prefix(leaf):
    q = torch.zeros(3, 8, 1, 128, dtype=torch.float16)
    for at in (0, 1):
        stores = [_store(b, leaf if leaf != "q" and i == at else None) for i, b in enumerate((1, 3))]
        x = q.clone().requires_grad_(True) if leaf == "q" else q
        call = lambda a=x, s=stores: kivi_shared_prefix_attend(a, KiviRows(**s[0]), KiviRows(**s[1]), 0.1)  # noqa: E731
        with pytest.raises(ValueError, match="not differentiable"):
            call()
        with torch.no_grad(), pytest.raises(VQLibraryError):  # (accepted: what is missing is the device)
            call()
        with fw.dual_level():
            stores = [_store(1), _store(3)]
            with pytest.raises(VQLibraryError):
                call(q, stores)
            if leaf == "q":
                x = fw.make_dual(q, torch.ones_like(q))
            else:
                stores[at][leaf] = fw.make_dual(stores[at][leaf], torch.ones_like(stores[at][leaf]))
            with pytest.raises(ValueError, match="not differentiable"):
                call(q if leaf != "q" else x, stores)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_rotary_append(which):
    rope = RotaryEmbedding(16)
    xs = [torch.zeros(2, h, 3, 16) for h in (4, 2, 2)]
    res = torch.zeros(2, 2, 8, 16), torch.zeros(2, 2, 8, 16)
    with fw.dual_level():
        with pytest.raises(VQLibraryError):
            rope.append(*xs, *res, 0)
        xs[which] = fw.make_dual(xs[which], torch.ones_like(xs[which]))
        with pytest.raises(ValueError, match="not differentiable"):
            rope.append(*xs, *res, 0)
