"""Forward-mode derivatives of the turn: the direction's own turn. The host logic over a plain form of the launch, and the kernel."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from veloxquant_mlx_b200.rotary import RotaryEmbedding


def _plain(rope):
    """The launch's formula in torch, so that the host logic runs without a device."""
    def rotate(fn, q, k, positions, inverse):
        def turn(x):
            if x is None:
                return None
            assert not x._is_zerotensor()
            S, r = x.shape[2], rope.rotary_dim
            pos = torch.arange(S) + positions if not isinstance(positions, torch.Tensor) else positions
            t = pos.to(rope.inv_freq)[:, None] * rope.inv_freq * (-1 if inverse else 1)
            c, s = rope.attention_factor * t.cos().to(x), rope.attention_factor * t.sin().to(x)
            a, b = x[..., : r // 2], x[..., r // 2 : r]
            return torch.cat((a * c - b * s, b * c + a * s, x[..., r:]), -1)
        return turn(q), turn(k)
    return rotate


def _cases(rope, device, dtype, positions):
    g = torch.Generator(device).manual_seed(3)
    rand = lambda h: torch.randn(2, h, 5, rope.head_dim, generator=g, device=device).to(dtype)  # noqa: E731
    q, k, tq, tk = rand(3), rand(2), rand(3), rand(2)
    with torch.no_grad():
        want = rope(tq, tk, positions), rope(q, k, positions)
    for grad in (False, True):
        q.requires_grad_(grad)
        for has_q, has_k in ((1, 1), (1, 0), (0, 1)):
            with fw.dual_level():
                y, z = rope(fw.make_dual(q, tq) if has_q else q, fw.make_dual(k, tk) if has_k else k, positions)
                assert torch.equal(y, want[1][0]) and torch.equal(z, want[1][1])
                for out, has, w in ((y, has_q, want[0][0]), (z, has_k, want[0][1])):
                    t = fw.unpack_dual(out).tangent
                    assert torch.equal(t, w) if has else t is None or not bool(t.any())
        with fw.dual_level():  # one tensor, the other way
            y = rope(fw.make_dual(q, tq), positions=positions, inverse=True)
            assert torch.equal(fw.unpack_dual(y).tangent, rope(tq, positions=positions, inverse=True))
            assert fw.unpack_dual(rope(q, positions=positions)).tangent is None  # nothing to derive
            zero = fw.make_dual(q, torch._efficientzerotensor(q.shape, dtype=q.dtype, device=q.device))
            t = fw.unpack_dual(rope(zero, positions=positions)).tangent
            assert t is None or not bool(t.any())
    # forward over reverse: the product of the Hessian of sum(y ** 3) / 6 with a direction, J^T (y * J t)
    with fw.dual_level():
        x = fw.make_dual(q, tq)
        y = rope(x, positions=positions)
        (got,) = torch.autograd.grad((y * y * y).sum() / 6, x)
        got = fw.unpack_dual(got).tangent
    with torch.no_grad():
        y, ty = rope(q, positions=positions), rope(tq, positions=positions)
        hess = rope(y * ty, positions=positions, inverse=True)
    # the products in between are rounded in another order: four roundings of values of at most max |y ty| times the factor
    assert float((got - hess).abs().max()) <= 8 * torch.finfo(dtype).eps * float((y * ty).abs().max()) * rope.attention_factor


@pytest.mark.parametrize("positions", [7, torch.tensor([4, 0, 9, 1, 1000])])
def test_the_host_logic(positions):
    rope = RotaryEmbedding(16, rotary_dim=12, attention_factor=1.25)
    rope._rotate = _plain(rope)
    _cases(rope, "cpu", torch.float32, positions)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("positions", [7, torch.tensor([4, 0, 9, 1, 1000])])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_the_tangent_is_the_direction_turned(layout, positions, dtype):
    rope = RotaryEmbedding(128, rotary_dim=64, layout=layout, attention_factor=1.25)
    _cases(rope, "cuda", dtype, positions if isinstance(positions, int) else positions.cuda())


@pytest.mark.gpu
def test_the_tangent_against_differences():
    # the turn is linear: (f(q + t) - f(q)) is f(t) up to the roundings of three float32 results below 2^4 each
    rope = RotaryEmbedding(64)
    q, t = (torch.randn(1, 2, 6, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(i)) for i in (1, 2))
    with fw.dual_level():
        got = fw.unpack_dual(rope(fw.make_dual(q, t), positions=3)).tangent
    assert float((got - (rope(q + t, positions=3) - rope(q, positions=3))).abs().max()) < 4 * 2.0**-24 * 2**4
