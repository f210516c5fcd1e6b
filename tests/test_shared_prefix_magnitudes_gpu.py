"""Keys and values from 10 down to 1e-6 in the shared-prefix attention, against 64 bits within the bound of what the kernels
round (tests/shared_prefix_bounds.py), and that bound against the one the contract states."""

from __future__ import annotations

import pytest
import torch

from shared_prefix_bounds import A, H, compare, expected, numbers
from veloxquant_mlx_b200 import kernels

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _store(B, nq, nr, D, bits, dtype, seed, k_size, v_size, shift):
    g = torch.Generator("cuda").manual_seed(seed)
    k, v = ((size * (shift + torch.randn(B, 2, nq + nr, D, device="cuda", generator=g))).to(dtype) for size in (k_size, v_size))
    t = {}
    t["k_codes"], t["k_scale"], t["k_zero"] = kernels.kivi_quantize(k[:, :, :nq], -2, 32, bits)
    t["v_codes"], t["v_scale"], t["v_zero"] = kernels.kivi_quantize(v[:, :, :nq], -1, 32, bits)
    return kernels.KiviRows(**t, k_res=k[:, :, nq:].contiguous(), v_res=v[:, :, nq:].contiguous(), store_bits=kernels.storage_bits(bits))


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("size", [10.0, 1e-2, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bits,D,S", [(2, 128, 1), (4, 128, 1), (4, 64, 5), (3, 128, 40), (8, 64, 1)])
def test_every_magnitude(bits, D, S, dtype, size, variant):
    q = torch.randn(9, 8, S, D, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dtype)
    for k_size, v_size, shift in ((1.0, size, 0.0), (size, 1.0, 0.0), (size, size, 3.0)):
        pre, own = _store(1, 224, 9, D, bits, dtype, 2, k_size, v_size, shift), _store(9, 96, 40, D, bits, dtype, 3, k_size, v_size, shift)
        q2 = q if k_size <= 1 else q / k_size
        got = kernels.kivi_shared_prefix_attend(q2, pre, own, D**-0.5, return_lse=True, variant=variant)
        compare(got, expected(q2, pre, own, D**-0.5))


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-5])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bits", [2, 4, 8])
def test_the_stated_bound_covers_the_derived_one(bits, dtype, size):
    rows = _store(2, 128, 20, 128, bits, dtype, 5, size, size, 1.0)
    k, ek, v, ev = numbers(rows, dtype)
    _, ks, kz, _, vs, vz, _, _ = rows._tensors
    for val, err, s, z, axis in ((k, ek, ks, kz, 2), (v, ev, vs, vz, 3)):
        val, err = val[:, :, :128], err[:, :, :128]
        s, z = (t.double().repeat_interleave(32, axis) for t in (s, z))
        if dtype == BF and bits != 8:
            stated = H * ((val - z).abs() + z.abs() + val.abs()) * (1 + 2 * H) + 2.0**-20
        else:  # (2^-9 of a quantization step at 8 bits, 2^-17 at 2 and 4: the offset of the float32 form, beside the code)
            stated = H * val.abs() + A + 2.0**-23 * z.abs() + (2.0**-8 if bits == 8 else 2.0**-16) * s
        assert bool((err <= stated).all())
