"""Padding that shares a packed group of 32 with live tokens: what it may hold and whom it reaches.

Padding values, exact rows and key groups of padding alone may hold anything. A key group that straddles ``own_start`` has
one scale and zero a channel for its padding and its live tokens: padding keys of ordinary size cost nothing beyond
the codes' own step, and what is not finite there stays within its request."""

from __future__ import annotations

import pytest
import torch

from shared_prefix_bounds import compare, expected
from veloxquant_mlx_b200 import kernels

pytestmark = pytest.mark.gpu
START = [0, 5, 31, 33, 70, 40]


def _own(dtype, junk_keys, junk_values):
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(6, 2, 96 + 20, 128, device="cuda", generator=g) for _ in range(2))
    for b, s in enumerate(START):
        k[b, :, :s] *= junk_keys
        v[b, :, :s] = junk_values
    k, v = k.to(dtype), v.to(dtype)
    t = {}
    t["k_codes"], t["k_scale"], t["k_zero"] = kernels.kivi_quantize(k[:, :, :96], -2, 32, 4)
    t["v_codes"], t["v_scale"], t["v_zero"] = kernels.kivi_quantize(v[:, :, :96], -1, 32, 4)
    return kernels.KiviRows(**t, k_res=k[:, :, 96:].contiguous(), v_res=v[:, :, 96:].contiguous())


@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_groups_that_straddle_the_start(dtype, variant, S):
    g = torch.Generator("cuda").manual_seed(4)
    q = torch.randn(6, 4, S, 128, device="cuda", generator=g).to(dtype)
    z = torch.randn(1, 2, 9, 128, device="cuda", generator=g).to(dtype)
    pre = kernels.KiviRows(k_res=z, v_res=z.clone())
    start = torch.tensor(START, dtype=torch.int32, device="cuda")
    call = lambda own: kernels.kivi_shared_prefix_attend(q, pre, own, 0.09, own_start=start, return_lse=True, variant=variant)  # noqa: E731
    for keys in (1.0, 20.0):
        own = _own(dtype, keys, float("nan"))
        got = call(own)
        for t in (4, 5):  # (the helper wants numbers where nothing is seen)
            for b, s in enumerate(START):
                own._tensors[t][b, :, :s] = 1.0
        compare(got, expected(q, pre, own, 0.09, start=start))
    clean = call(_own(dtype, 1.0, 1.0))
    bad = call(_own(dtype, float("inf"), 1.0))
    straddles = [s % 32 != 0 and s < 96 for s in START]
    for b, s in enumerate(straddles):
        if s:
            assert bool(bad[0][b].isnan().any())  # as the contract says
        else:
            assert torch.equal(bad[0][b], clean[0][b]) and torch.equal(bad[1][b], clean[1][b])
