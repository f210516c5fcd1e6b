"""Many tokens behind one that outweighs each of them by far: their weights must not vanish in float16's smallest step."""

from __future__ import annotations

import math

import pytest
import torch

from shared_prefix_bounds import compare, expected
from veloxquant_mlx_b200 import kernels

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
STEP = 2.0**-32  # half of float16's smallest step, 2^-25, on weights that are held times 2^7 or more


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("log2", [18, 24, 26, 29])
@pytest.mark.parametrize("at", [0, 70, 4000])
def test_the_tail_behind_one_token(at, log2, dtype, variant):
    """One token of weight 1 and value 0 (an attention sink), 4095 of 2^-log2 and value about 1, in one split."""
    g = torch.Generator("cuda").manual_seed(7)
    k, v = torch.zeros(1, 1, 4096, 128, device="cuda"), 1 + 0.1 * torch.randn(1, 1, 4096, 128, device="cuda", generator=g)
    k[:, :, at, 0], v[:, :, at] = log2 * math.log(2), 0.0
    rows = kernels.KiviRows(k_res=k.to(dtype), v_res=v.to(dtype))
    q = torch.zeros(40, 1, 1, 128, device="cuda", dtype=dtype)
    q[..., 0] = 1
    got = kernels.kivi_shared_prefix_attend(q, rows, None, 1.0, return_lse=True, variant=variant, n_splits=1)
    compare(got, expected(q, rows, None, 1.0, weight_step=STEP))
    assert float(got[0].float().min()) > 0.5 * 4095 * 2.0**-log2 or log2 == 29 and dtype == HF


@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("variant", [0, 1, 2])
def test_the_tail_of_own_tokens_and_packed_ones(variant, S):
    g = torch.Generator("cuda").manual_seed(8)
    k, v = 0.01 * torch.randn(5, 1, 640, 128, device="cuda", generator=g), 1 + 0.1 * torch.randn(5, 1, 640, 128, device="cuda", generator=g)
    k[:, :, 32, 0], v[:, :, 32] = 26 * math.log(2), 0.0
    t = {}
    t["k_codes"], t["k_scale"], t["k_zero"] = kernels.kivi_quantize(k[:, :, :576].half(), -2, 32, 8)
    t["v_codes"], t["v_scale"], t["v_zero"] = kernels.kivi_quantize(v[:, :, :576].half(), -1, 32, 8)
    own = kernels.KiviRows(**t, k_res=k[:, :, 576:].half().contiguous(), v_res=v[:, :, 576:].half().contiguous(), store_bits=8)
    z = torch.zeros(1, 1, 1, 128, device="cuda", dtype=HF)
    pre = kernels.KiviRows(k_res=z, v_res=z.clone(), store_bits=8)
    q = torch.zeros(5, 1, S, 128, device="cuda", dtype=HF)
    q[..., 0] = 1
    got = kernels.kivi_shared_prefix_attend(q, pre, own, 1.0, return_lse=True, variant=variant)
    compare(got, expected(q, pre, own, 1.0, weight_step=STEP))


@pytest.mark.parametrize("variant", [1, 2])
def test_the_largest_weights_and_values_together(variant):
    """Scores that rise by just under 2^8 (the maximum stays) with values at the end of the range: nothing overflows."""
    n = 512
    k, v = torch.zeros(1, 1, n, 128, device="cuda"), torch.full((1, 1, n, 128), 60000.0, device="cuda")
    k[:, :, 64:, 0] = 7.9 * math.log(2)
    v[:, :, ::2] = -60000.0
    v[:, :, 64:] = 65504.0
    rows = kernels.KiviRows(k_res=k.half(), v_res=v.half())
    q = torch.zeros(40, 1, 1, 128, device="cuda", dtype=HF)
    q[..., 0] = 1
    got = kernels.kivi_shared_prefix_attend(q, rows, None, 1.0, return_lse=True, variant=variant, n_splits=1)
    want = expected(q, rows, None, 1.0, weight_step=STEP)
    assert bool(got[0].isfinite().all())
    compare(got, want)
