"""Rotary positions on the GPU against complex multiplication in 64 bits.

Tolerance of an output: the angle is 2 pi times a turn count in [-1/2, 1/2] that was rounded to float32 (off by at
most 2^-26 turns: 2 pi 2^-26 < 2^-23 radian) after a 64-bit product (position * 2^-52: nothing); sine and cosine
are within 2^-22 of theirs (1.5 ulp of 1, documented for sincospi at 2 ulp), times the factor; two products and a
sum round by 2^-24 each. Together below 2^-20 * factor * (|a| + |b|); then one rounding to the type, eps / 2."""

from __future__ import annotations

import pytest
import torch

from veloxquant_mlx_b200.rotary import RotaryEmbedding

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def _rand(shape, dtype, seed, strided=False):
    g = torch.Generator(DEV).manual_seed(seed)
    B, H, S, D = shape
    if strided:
        return torch.randn(B, S, H, D, device=DEV, generator=g).to(dtype).transpose(1, 2)
    return torch.randn(shape, device=DEV, generator=g).to(dtype)


def _turn64(x, freq, pos, layout, r, factor=1.0, sign=1.0):
    """(result, |a| + |b| of each element's pair) in 64 bits; pos [B or 1, S]."""
    x = x.detach().double()
    t = sign * pos.double()[:, None, :, None] * freq.to(x.device)
    z = torch.complex(factor * torch.cos(t), factor * torch.sin(t))
    y, mag = x.clone(), torch.zeros_like(x)
    if layout == "interleaved":
        w = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous())
        y[..., :r] = torch.view_as_real(w * z).reshape(*x.shape[:-1], r)
        mag[..., :r] = (w.real.abs() + w.imag.abs()).repeat_interleave(2, -1)
    else:
        w = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2 : r].contiguous())
        p = w * z
        y[..., :r] = torch.cat((p.real, p.imag), -1)
        mag[..., :r] = (w.real.abs() + w.imag.abs()).repeat(1, 1, 1, 2)
    return y, mag


def _close(got, want, mag, factor=1.0):
    tol = 2.0**-20 * abs(factor) * mag + torch.finfo(got.dtype).eps / 2 * (want.abs() + 2.0**-20 * abs(factor) * mag)
    if got.dtype == HF:
        tol = tol + 2.0**-25  # half of float16's smallest step
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), f"off by {off.max().item():.3e} more than allowed"


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,r", [(128, 128), (128, 64), (80, 32), (80, 40), (96, 96), (64, 6), (256, 256), (2, 2), (130, 10), (36, 36)])
def test_turns_every_width_and_part(D, r, layout, dtype):
    B, S, Hq, Hk = 2, 5, 6, 3
    rope = RotaryEmbedding(D, rotary_dim=r, layout=layout)
    q, k = _rand((B, Hq, S, D), dtype, 1), _rand((B, Hk, S, D), dtype, 2, strided=True)
    pos = torch.tensor([[0, 1, 2, 3, 4], [7, 100000, 3, 1048575, 12]], device=DEV)
    yq, yk = rope(q, k, pos)
    assert yq.is_contiguous() and yk.is_contiguous() and yq.dtype == dtype
    for x, y in ((q, yq), (k, yk)):
        _close(y, *_turn64(x, rope.inv_freq, pos, layout, r))
        assert torch.equal(y[..., r:], x[..., r:])


@pytest.mark.parametrize("pos", ["none", "int", "S32", "1S64", "BS32", "strided"])
def test_positions_in_every_form(pos):
    B, S, H, D = 3, 9, 4, 64
    rope = RotaryEmbedding(D, scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048}, device=DEV)
    q = _rand((B, H, S, D), F, 3)
    at = torch.arange(S, device=DEV)
    given, full = {
        "none": (None, at[None]), "int": (-5, at[None] - 5), "S32": (at.int() * 3, at[None] * 3), "1S64": (at[None] + 2**31, at[None] + 2**31),
        "BS32": ((at + torch.tensor([[4], [0], [900]], device=DEV)).int(),) * 2,
        "strided": ((at[:, None] * 2 + torch.tensor([[4, 0, 9]], device=DEV)).t(),) * 2,
    }[pos]
    y = rope(q, positions=given)
    _close(y, *_turn64(q, rope.inv_freq, full, "half", D, rope.attention_factor), rope.attention_factor)


def test_far_positions_keep_their_angle():
    # a float32 angle at position 2^20 + 1 would be off by up to 2^-5 of a radian
    rope = RotaryEmbedding(128)
    q = _rand((1, 1, 4, 128), F, 4)
    pos = torch.tensor([[2**20 + 1, 2**24 + 1, 2**30 + 1, 2**31 + 12345]], device=DEV)
    _close(rope(q, positions=pos), *_turn64(q, rope.inv_freq, pos, "half", 128))


@pytest.mark.parametrize("B,S,H", [(1, 1, 1), (1, 1, 41), (300, 1, 5), (1, 3000, 2), (2, 700, 33)])
def test_sizes_from_one_token_to_many(B, S, H):
    rope = RotaryEmbedding(128)
    q = _rand((B, H, S, 128), BF, 5, strided=True)
    _close(rope(q, positions=11), *_turn64(q, rope.inv_freq, torch.arange(S, device=DEV)[None] + 11, "half", 128))


def test_odd_addresses_and_strides():
    base = torch.randn(2, 3, 7, 200, device=DEV)
    for dtype in (BF, HF, F):
        for off in (0, 1, 2, 3, 4, 8):
            q = base.to(dtype)[:, :, ::2, off : off + 128]
            rope = RotaryEmbedding(128)
            _close(rope(q), *_turn64(q, rope.inv_freq, torch.arange(4, device=DEV)[None], "half", 128))
    q = torch.randn(2, 3, 128, 4, device=DEV).transpose(2, 3)  # channels not contiguous
    _close(RotaryEmbedding(128)(q), *_turn64(q, RotaryEmbedding(128).inv_freq, torch.arange(4, device=DEV)[None], "half", 128))
    q = torch.randn(1, 1, 1, 128, device=DEV).expand(3, 2, 4, 128)  # broadcast
    _close(RotaryEmbedding(128)(q), *_turn64(q, RotaryEmbedding(128).inv_freq, torch.arange(4, device=DEV)[None], "half", 128))


def test_empty_tensors():
    rope = RotaryEmbedding(64)
    for shape in ((0, 4, 3, 64), (2, 4, 0, 64), (2, 0, 3, 64)):
        assert rope(torch.empty(shape, device=DEV)).shape == shape


def test_inverse_turns_back():
    rope = RotaryEmbedding(96, rotary_dim=48, layout="interleaved")
    q = _rand((2, 3, 17, 96), F, 6)
    back = rope(rope(q, positions=1000), positions=1000, inverse=True)
    # two turns of 2^-20 (|a| + |b|) each, |a| below 8
    assert q.abs().max() < 8 and (back - q).abs().max().item() < 2.0**-15


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF, F])
def test_gradient_is_the_formula_and_the_difference_quotient(layout, dtype):
    D, r = 64, 32
    rope = RotaryEmbedding(D, rotary_dim=r, layout=layout, attention_factor=1.5)
    q, k = _rand((2, 4, 6, D), dtype, 7).requires_grad_(True), _rand((2, 2, 6, D), dtype, 8, strided=True).requires_grad_(True)
    pos = torch.randint(0, 5000, (2, 6), device=DEV)
    gq, gk = _rand((2, 4, 6, D), dtype, 9), _rand((2, 2, 6, D), dtype, 10)
    yq, yk = rope(q, k, pos)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for g, d in ((gq, dq), (gk, dk)):
        _close(d, *_turn64(g, rope.inv_freq, pos, layout, r, 1.5, -1.0), 1.5)
    if dtype == F:
        # the operation is linear: <g, f(x + e) - f(x)> = <df(g), e> up to the roundings of both sides
        e = _rand(tuple(q.shape), F, 11)
        with torch.no_grad():
            lhs = (gq.double() * (rope(q + e, positions=pos).double() - rope(q, positions=pos).double())).sum()
        rhs = (dq.double() * e.double()).sum()
        assert abs(float(lhs - rhs)) < 2.0**-18 * float((gq.abs().double() * (q.detach().abs() + e.abs()).double().amax()).sum())


def test_gradients_of_one_input_of_broadcast_grads_and_twice():
    rope = RotaryEmbedding(32)
    q, k = _rand((1, 2, 3, 32), F, 12).requires_grad_(True), _rand((1, 1, 3, 32), F, 13)
    yq, yk = rope(q, k)
    (d,) = torch.autograd.grad(yq.sum(), q, create_graph=True)
    _close(d, *_turn64(torch.ones_like(q), rope.inv_freq, torch.arange(3, device=DEV)[None], "half", 32, 1.0, -1.0))
    k2 = k.clone().requires_grad_(True)
    yq, yk = rope(q, k2)
    (dk,) = torch.autograd.grad(yk.sum(), k2)  # q's output is not used
    _close(dk, *_turn64(torch.ones_like(k2), rope.inv_freq, torch.arange(3, device=DEV)[None], "half", 32, 1.0, -1.0))
    # twice: f is linear, so the gradient of <df(g), w> with respect to g is f(w)
    g = torch.ones_like(q).requires_grad_(True)
    w = _rand((1, 2, 3, 32), F, 14)
    (d,) = torch.autograd.grad(rope(q), q, g, create_graph=True)
    (dd,) = torch.autograd.grad((d * w).sum(), g)
    _close(dd, *_turn64(w, rope.inv_freq, torch.arange(3, device=DEV)[None], "half", 32))


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("S,at", [(1, 0), (1, 351), (5, 40)])
def test_append_writes_its_rows_and_no_others(S, at, dtype):
    B, Hq, Hk, D, rows = 3, 8, 2, 128, 352
    rope = RotaryEmbedding(D, rotary_dim=64)
    q, k, v = _rand((B, Hq, S, D), dtype, 20), _rand((B, Hk, S, D), dtype, 21, strided=True), _rand((B, Hk, S, D), dtype, 22)
    kv = torch.randn(2, B, Hk, rows, D, device=DEV).to(dtype)
    if at + S > rows:
        at = rows - S
    before = kv.clone()
    pos = torch.randint(0, 9999, (B, S), device=DEV, dtype=torch.int32)
    y = rope.append(q, k, v, kv[0], kv[1], at, pos)
    _close(y, *_turn64(q, rope.inv_freq, pos, "half", 64))
    _close(kv[0, :, :, at : at + S], *_turn64(k, rope.inv_freq, pos, "half", 64))
    assert torch.equal(kv[1, :, :, at : at + S], v)
    keep = torch.ones(rows, dtype=torch.bool, device=DEV)
    keep[at : at + S] = False
    assert torch.equal(kv[:, :, :, keep], before[:, :, :, keep])


def test_append_refuses_shared_memory():
    rope = RotaryEmbedding(64)
    kv = torch.zeros(2, 1, 2, 8, 64, device=DEV)
    q, k = torch.zeros(1, 2, 1, 64, device=DEV), torch.zeros(1, 2, 1, 64, device=DEV)
    with pytest.raises(ValueError, match="share memory"):
        rope.append(q, kv[0, :, :, :1], k, kv[0], kv[1], 1)
    with pytest.raises(ValueError, match="different memory"):
        rope.append(q, k, k, kv[0], kv[0], 1)


def test_other_stream_and_graph_replay():
    rope = RotaryEmbedding(128, device=DEV)
    q, k = _rand((4, 8, 2, 128), BF, 30), _rand((4, 2, 2, 128), BF, 31)
    pos = torch.randint(0, 4096, (4, 2), device=DEV)
    want = rope(q, k, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rope(q, k, pos)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = rope(q, k, pos)
    pos.add_(17)
    q.mul_(2)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, rope(q, k, pos)))


def test_first_use_inside_a_capture_is_refused():
    rope = RotaryEmbedding(64)
    q = torch.zeros(1, 1, 1, 64, device=DEV)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="inside a graph capture"):
        with torch.cuda.graph(g):
            rope(q)


@pytest.mark.parametrize("b", [2, 4])
def test_cache_update_rotary_equals_rotating_first(b):
    from veloxquant_mlx_b200.cache import KVCacheConfig, KVCacheFactory

    def make():
        return KVCacheFactory.create(KVCacheConfig(method="kivi", head_dim=128, bit_width_inlier=b, residual_length=64, fused_sdpa_memory_bound=True))

    rope = RotaryEmbedding(128, base=500000.0)
    one, two = make(), make()
    n = 0
    for step, S in enumerate([70, 1, 1, 30] + [1] * 40 + [200, 1, 5]):
        q, k, v = (_rand((2, h, S, 128), HF, 100 * step + h, strided=True) for h in (8, 2, 2))
        q1, *_ = one.update_rotary(q, k, v, rope)
        q2, k2 = rope(q, k, n)
        two.update_and_fetch(k2, v)
        n += S
        assert torch.equal(q1, q2) and one.offset == two.offset == n and one._n_res == two._n_res and one._n_quantized == two._n_quantized
        assert torch.equal(one.fused_sdpa(q1[:, :, -1:].contiguous(), 0.09), two.fused_sdpa(q2[:, :, -1:].contiguous(), 0.09))
    assert all(torch.equal(x, y) for x, y in zip(one.state, two.state))


def test_offsets_past_32_bits():
    """More than 2^31 elements, in the tokens of one head and in the rows behind which an append goes."""
    S = (1 << 24) + 5
    x = torch.empty(1, 1, S, 136, dtype=BF, device=DEV)[..., :128]  # 2.3e9 elements apart
    tail = _rand((1, 1, 9, 128), BF, 40)
    x[:, :, -9:] = tail
    rope = RotaryEmbedding(128, rotary_dim=64)
    y = rope(x, positions=7)[:, :, -9:]
    pos = 7 + S - 9 + torch.arange(9, device=DEV)[None]
    _close(y, *_turn64(tail, rope.inv_freq, pos, "half", 64))
    assert torch.equal(y[..., 64:], tail[..., 64:])
    del x, y
    rows = (1 << 24) + 100
    res = torch.zeros(2, 1, 1, rows, 132, dtype=BF, device=DEV)[..., :128]
    q, k, v = (_rand((1, 1, 3, 128), BF, 41 + i) for i in range(3))
    rope.append(q, k, v, res[0], res[1], rows - 3, 5)
    _close(res[0, :, :, -3:], *_turn64(k, rope.inv_freq, 5 + torch.arange(3, device=DEV)[None], "half", 64))
    assert torch.equal(res[1, :, :, -3:], v) and not res[:, :, :, :1000].any() and not res[:, :, :, -200:-3].any()


def test_forward_and_gradient_inside_a_graph():
    rope = RotaryEmbedding(64, device=DEV)
    q, k = _rand((2, 4, 3, 64), F, 50).requires_grad_(True), _rand((2, 2, 3, 64), F, 51).requires_grad_(True)
    pos = torch.randint(0, 99, (2, 3), device=DEV)
    gq, gk = _rand((2, 4, 3, 64), F, 52), _rand((2, 2, 3, 64), F, 53)

    def step():
        yq, yk = rope(q, k, pos)
        return (yq, yk, *torch.autograd.grad((yq, yk), (q, k), (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    with torch.no_grad():
        q.mul_(3)
        gk.add_(1)
    pos.add_(100)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_the_same_tensor_twice_and_a_half_used_pair():
    rope = RotaryEmbedding(64)
    q = _rand((1, 2, 5, 64), F, 60).requires_grad_(True)
    a, b = rope(q, q, 3)
    assert torch.equal(a, b)
    (d,) = torch.autograd.grad((a, b), q, (torch.ones_like(a), torch.ones_like(b)))
    want, mag = _turn64(torch.ones_like(q), rope.inv_freq, 3 + torch.arange(5, device=DEV)[None], "half", 64, 1.0, -1.0)
    _close(d, 2 * want, 2 * mag)
    with torch.no_grad():
        assert not rope(q)[0].requires_grad


def test_update_rotary_of_a_cache_with_its_own_append():
    """kivi_sink replaces update_and_fetch: it gets rotated keys through it."""
    from veloxquant_mlx_b200.cache import KVCacheConfig, KVCacheFactory

    def make():
        return KVCacheFactory.create(KVCacheConfig(method="kivi_sink", head_dim=128, bit_width_inlier=4, residual_length=32, n_sink_tokens=2))

    rope, one, two = RotaryEmbedding(128), make(), make()
    n = 0
    for S in (50, 1, 1):
        q, k, v = (_rand((1, h, S, 128), HF, 70 + S + h) for h in (4, 2, 2))
        q1, k1, v1 = one.update_rotary(q, k, v, rope)
        q2, k2 = rope(q, k, n)
        k3, v3 = two.update_and_fetch(k2, v)
        n += S
        assert torch.equal(q1, q2) and torch.equal(k1, k3) and torch.equal(v1, v3)
