"""Scores of any size that keys and queries within float16's range can make (here up to 2^33 in base 2): the weights stay
finite, equal scores give the average, and a score that leads by more than float32's spacing gives its own value."""

from __future__ import annotations

import math

import pytest
import torch

from veloxquant_mlx_b200 import kernels

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
SIZES = [0.0, 20.0, 1000.0, 3000.0, 11111.0, 30000.0, 60000.0]


def _run(key, lead, dtype, variant, splits, part):
    """Keys: channel 0 = `key`, channel 1 = `lead` by token; all queries (57344, 57344, 0, ...); values are whole sixteenths."""
    n = 700
    g = torch.Generator("cuda").manual_seed(2)
    k, v = torch.zeros(1, 1, n, 128, device="cuda"), torch.randint(-100, 101, (1, 1, n, 128), device="cuda", generator=g) / 16
    k[..., 0], k[..., 1] = key, lead
    q = torch.zeros(40, 1, 1, 128, device="cuda", dtype=dtype)
    q[..., 0] = q[..., 1] = 57344.0
    k, v = k.to(dtype), v.to(dtype)
    if part == "prefix":
        rows, own = kernels.KiviRows(k_res=k, v_res=v), None
    else:  # a prefix token that is far behind, and every request's own copy
        far = torch.zeros(1, 1, 1, 128, device="cuda", dtype=dtype)
        far[..., 0], far[..., 1] = k[0, 0, 0, 0], -64.0
        rows = kernels.KiviRows(k_res=far, v_res=torch.full_like(far, 1000.0))
        q = q[:2].expand(2, 1, 40, 128).contiguous()  # (40 rows: own tokens on the tensor-memory kernel too)
        own = kernels.KiviRows(k_res=k.expand(2, -1, -1, -1).contiguous(), v_res=v.expand(2, -1, -1, -1).contiguous())
    out, lse = kernels.kivi_shared_prefix_attend(q, rows, own, 0.7, causal=False, return_lse=True, variant=variant, n_splits=splits)
    kernels.attend_status()
    return out, lse, v


def _is_value(out, v):
    """out is v: one token's float16 weight (off by 2^-11 of itself) over the same weight as it was before that rounding (it is a
    power of two only where its exponent is whole), 2^-21 for the exponential and the quotient, and the output's rounding."""
    near = (2.0**-11 + 2.0**-21) * v.double().abs()
    near = near + torch.finfo(out.dtype).eps / 2 * (v.double().abs() + near)
    return bool(((out.double() - v.double()).abs() <= near).all())


@pytest.mark.parametrize("part", ["prefix", "own"])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_equal_scores_give_the_average(dtype, variant, splits, part):
    for key in SIZES:
        for sign in (1.0, -1.0):
            key16 = float(torch.tensor(key, dtype=dtype))
            out, lse, v = _run(sign * key16, 0.0, dtype, variant, splits, part)
            want = v.double().mean(2)
            # equal weights; values are exact: sums of 700, one rounding of the weight, one of the output
            tol = (700 * 2.0**-24 + 2.0**-11) * v.double().abs().mean(2) + torch.finfo(dtype).eps / 2 * want.abs() + 2.0**-24
            assert bool(((out.double() - want[:, :, None]).abs() <= tol[:, :, None]).all()), (key, sign)
            score = sign * key16 * 57344.0 * 0.7
            assert bool(((lse.double() - (score + math.log(700))).abs() <= 8 * 2.0**-24 * abs(score) + 1e-5).all())


@pytest.mark.parametrize("part", ["prefix", "own"])
@pytest.mark.parametrize("at", [0, 63, 300, 699])
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_the_leading_score_gives_its_value(dtype, variant, at, part):
    for key in SIZES:
        for sign in (1.0, -1.0):
            lead = torch.zeros(700, device="cuda")
            lead[at] = 8.0  # 8 * 57344 * 0.7 = 321126 ahead, the spacing at 57344 * 60000 * 0.7 is 256
            out, _, v = _run(sign * float(torch.tensor(key, dtype=dtype)), lead, dtype, variant, 1, part)
            assert _is_value(out, v[:, :, at : at + 1]), (key, sign)


@pytest.mark.parametrize("variant", [1, 2])
def test_scores_that_rise_far_from_zero(variant):
    """Every token outweighs the ones before it: the last one's value."""
    lead = 8.0 * (1 + torch.arange(700, device="cuda")) // 1
    for key in (-30000.0, 0.0, 30000.0):
        out, _, v = _run(float(torch.tensor(key, dtype=HF)), lead, HF, variant, 1, "prefix")
        assert _is_value(out, v[:, :, 699:]), key
