"""C entries: sizes whose product passes 64 bits are refused, not taken for the small number they wrap to."""

from __future__ import annotations

import pytest

from veloxquant_mlx_b200 import _lib


def _rotary(B, S, heads):
    # (addresses are never reached: the sizes are refused, or nothing is to be done, before a launch)
    block = _lib.ROTARY_PACK.pack(64, 0, 0, 64, 0, 0, *[128] * 9, *[128] * 9, heads, 0, 0, 0, B, S, 128, 128, 0, 0, 0, 8, 1.0, 0, 0, 0, 64)
    return _lib.lib().vq_rotary(block, None)


@pytest.mark.parametrize("B,S", [(1 << 62, 4), (1 << 33, 1 << 31), (1 << 60, 16), (1 << 40, 0), (1 << 30, 1 << 30)])
def test_rotary(B, S):
    assert _rotary(0, S & 7, 4) == 0 and _rotary(2, 3, 0) == 0
    assert _rotary(B, S, 4) != 0


@pytest.mark.parametrize("B,H,S", [(1 << 30, 1 << 30, 16), (1 << 24, 1 << 24, 1 << 16), (1 << 16, 1 << 16, 1)])
def test_shared_prefix(B, H, S):
    rows = _lib.KIVI_ROWS_PACK.pack(*[64] * 8, 0, 0, 0, 0, 0, 0, 5)
    need = lambda b, h, s: _lib.lib().vq_kivi_shared_attend_workspace_bytes(  # noqa: E731
        _lib.SHARED_ATTEND_HEAD.pack(64, 64, 0, 0, 0, b, h, h, s, 128, 4, 32, 0.1, 0) + rows + rows + _lib.SHARED_ATTEND_TAIL.pack(0, 0, 1, 0))
    assert need(2, 2, 2) > 0
    assert need(B, H, S) == 0
