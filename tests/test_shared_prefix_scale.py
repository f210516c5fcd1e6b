"""Scales that are zero, negative or tiny in the shared-prefix attention: which kernel they take (host) and what comes out
(GPU), at sizes that the tcgen05 kernel takes for a positive scale, with token tiles that are partly filled."""

from __future__ import annotations

import pytest
import torch

from veloxquant_mlx_b200 import _lib, kernels

# B, H_q, H_kv, S_q, pre_q, pre_r, own_q, own_r: prefix on tcgen05; prefix and own tokens on it
SIZES = [(64, 8, 2, 1, 2080, 9, 32, 7), (9, 8, 1, 40, 640, 3, 608, 77)]


def _workspace(size, scale, variant):
    B, Hq, Hk, S, *n = size
    rows = [_lib.KIVI_ROWS_PACK.pack(*[64] * 8, 1 << 20, 1 << 20, 1 << 18, 1 << 18, 1 << 20, n[i], n[i + 1]) for i in (0, 2)]
    head = _lib.SHARED_ATTEND_HEAD.pack(64, 64, 0, 0, 0, B, Hq, Hk, S, 128, 4, 32, scale, _lib.VQ_ATTEND_CAUSAL)
    return _lib.lib().vq_kivi_shared_attend_workspace_bytes(head + b"".join(rows) + _lib.SHARED_ATTEND_TAIL.pack(0, 0, variant, 0))


def test_a_scale_that_is_not_positive_takes_the_warp_tiles():
    size = SIZES[0]  # (here the two kernels split the prefix differently, which shows in the workspace)
    assert _workspace(size, 0.1, 0) == _workspace(size, 0.1, 2) != _workspace(size, 0.1, 1) > 0
    for scale in (0.0, -0.0, -0.1, float("nan")):
        assert _workspace(size, scale, 0) == _workspace(size, scale, 1) == _workspace(size, 0.1, 1)
        for other in SIZES:
            assert _workspace(other, scale, 2) == 0  # refused


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-45, 1e-30])
@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("size", SIZES)
def test_scales_against_64_bits(size, variant, scale):
    from shared_prefix_bounds import compare, expected
    from test_shared_prefix_gpu import BF, DEV, HF, _gen, make_store

    B, Hq, Hk, S, pq, pr, oq, orr = size
    for dtype in (HF, BF):
        q = torch.randn(B, Hq, S, 128, device=DEV, generator=_gen(1)).to(dtype)
        pre, own = make_store(1, Hk, 128, 4, pq, pr, dtype, 2)[0], make_store(B, Hk, 128, 4, oq, orr, dtype, 3)[0]
        start = torch.tensor([(37 * b) % (oq + orr) for b in range(B)], dtype=torch.int32, device=DEV)
        if variant == 2 and not scale > 0:
            with pytest.raises(ValueError, match="positive scale"):
                kernels.kivi_shared_prefix_attend(q, pre, own, scale, own_start=start, variant=variant)
            continue
        got = kernels.kivi_shared_prefix_attend(q, pre, own, scale, own_start=start, return_lse=True, variant=variant)
        compare(got, expected(q, pre, own, scale, start=start))
