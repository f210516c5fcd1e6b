"""``RotaryEmbedding.append`` over one buffer: parts that lie apart are taken, parts that meet are refused."""

from __future__ import annotations

import pytest
import torch

from veloxquant_mlx_b200 import VQLibraryError
from veloxquant_mlx_b200.rotary import RotaryEmbedding, _overlap


def _arena(device):
    B, S, D = 2, 3, 64
    sizes = {"q": (B, 4, S, D), "k": (B, 2, S, D), "v": (B, 2, S, D), "k_res": (B, 2, 8, D), "v_res": (B, 2, 8, D)}
    at, offsets = 0, {}
    for name, shape in sizes.items():
        offsets[name] = at
        at += torch.Size(shape).numel()
    buf = torch.randn(at, device=device, generator=torch.Generator(device).manual_seed(1))
    return {n: buf[offsets[n] : offsets[n] + torch.Size(s).numel()].view(s) for n, s in sizes.items()}


def test_what_meets():
    t = torch.zeros(4, 6, 8)
    assert not _overlap(t[0], t[1]) and _overlap(t[0], t[0, 5:]) and _overlap(t[:, :1], t[1]) and not _overlap(t[0, :0], t[0])
    assert _overlap(t[0, 0, :1], t[0, 0]) and not _overlap(t[0, 0, :4], t[0, 0, 4:])


def test_one_buffer_without_a_device():
    rope = RotaryEmbedding(64)
    a = _arena("cpu")
    # (the checks of memory come behind the one for a device: called in its place)
    with pytest.raises(VQLibraryError):
        rope.append(a["q"], a["k"], a["v"], a["k_res"], a["v_res"], 2)


@pytest.mark.gpu
def test_one_buffer():
    rope = RotaryEmbedding(64)
    a = _arena("cuda")
    b = {n: t.clone() for n, t in a.items()}
    got = rope.append(a["q"], a["k"], a["v"], a["k_res"], a["v_res"], 2, 5)
    want = rope.append(b["q"], b["k"], b["v"], b["k_res"], b["v_res"], 2, 5)
    assert torch.equal(got, want) and all(torch.equal(a[n], b[n]) for n in a)
    for name in ("q", "k", "v"):
        inside = a["k_res"][:, :, :3] if name != "q" else a["v_res"].view(2, 2, 8, 64)[:, :, 5:]
        with pytest.raises(ValueError, match="share memory"):
            rope.append(**{**{n: a[n] for n in ("q", "k", "v")}, name: inside}, k_res=a["k_res"], v_res=a["v_res"], tok_offset=0)
