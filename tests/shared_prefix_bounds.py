"""softmax(scale q k) v over packed rows in 64 bits, with a bound on what the shared-prefix kernels may be off by.

h = 2^-11 (one rounding to float16, relative) and a = 2^-25 (the same below its normal range), f = 2^-24 (float32).
* Decoded in float32 (float16 data, and 8 bits): zero - BASE scale is rounded once, then one fused multiply-add, then float16:
  |err| <= h |v| + a + 2 f (|zero| + BASE scale), BASE = 128 (2 and 4 bits) or 32768.
* Decoded in half precision (bfloat16 data at 2 and 4 bits): scale is off by h scale or `scale_step` (a, or less where it is held as a
  multiple), zero by h |zero| + a, the fused multiply-add by h |v| + a:
  |err| <= (1 + h) (code (h scale + scale_step) + h |zero| + a) + h |v| + a.
* Exact rows: 0 in float16; bfloat16 has fewer bits than float16, so only a.
* A score: scale * (|q| . err_k + |err_q| . (|k| + err_k)) + (D + 4) f scale |q| . |k|, err_q = a for bfloat16; its exponent's argument is
  rounded twice more, f (4 |score| + 8) each; delta is the largest over the row's seen slots.
* A weight: a factor within exp(+-2 delta) (numerator and denominator), 2^-21 of the exponential, h as float16; `weight_step`, relative to
  the row's largest weight, is what float16's smallest step comes to.
* Sums in float32: n f. Output: one rounding, eps / 2 (and half of float16's smallest step)."""

from __future__ import annotations

import math

import torch

H, A, F = 2.0**-11, 2.0**-25, 2.0**-24


def numbers(rows, dtype, res_offset=0, scale_step=A):
    """Keys, their bound, values, their bound of a KiviRows: four [B, H, tokens, D] in 64 bits."""
    k_codes, k_scale, k_zero, v_codes, v_scale, v_zero, k_res, v_res = rows._tensors
    n, sb, D = rows.n_quant, rows.store_bits, rows.head_dim
    out = []
    for codes, scale, zero, exact, axis in ((k_codes, k_scale, k_zero, k_res, 2), (v_codes, v_scale, v_zero, v_res, 3)):
        val, err = [], []
        if n:
            at = torch.arange(D, device=codes.device)
            byte = codes[:, :, :n].long().repeat_interleave(8 // sb, 3)
            code = ((byte >> (sb * (at % (8 // sb)))) & (2**sb - 1)).double()
            rows_of = n // 32 if axis == 2 else n
            s, z = (t[:, :, :rows_of].double().repeat_interleave(32, axis) for t in (scale, zero))
            v = code * s + z
            val.append(v)
            if dtype == torch.bfloat16 and sb != 8:
                err.append((1 + H) * (code * (H * s + scale_step) + H * z.abs() + A) + H * v.abs() + A)
            else:
                err.append(H * v.abs() + A + 2 * F * (z.abs() + (32768 if sb == 8 else 128) * s))
        if rows.n_res:
            val.append(exact[:, :, res_offset : res_offset + rows.n_res].double())
            err.append(torch.full_like(val[-1], A if dtype == torch.bfloat16 else 0.0))
        out += [torch.cat(val, 2), torch.cat(err, 2)]
    return out


def expected(q, prefix, own, scale, *, causal=True, start=None, prefix_offset=0, own_offset=0, scale_step=A, weight_step=A):
    """(out, lse, bound on out, bound on lse) of kivi_shared_prefix_attend, in 64 bits."""
    B, Hq, S, D = q.shape
    parts = [[t.expand(B, -1, -1, -1) for t in numbers(prefix, q.dtype, prefix_offset, scale_step)]]
    if own is not None and len(own):
        parts.append(numbers(own, q.dtype, own_offset, scale_step))
    k, ek, v, ev = (torch.cat(t, 2).repeat_interleave(Hq // prefix.heads, 1) for t in zip(*parts))
    n, n_pre = k.shape[2], len(prefix)
    slot, r = torch.arange(n, device=q.device) - n_pre, torch.arange(S, device=q.device)
    seen = torch.ones(S, n, dtype=torch.bool, device=q.device)
    if causal:
        seen = (slot < 0) | (slot <= (n - n_pre) - S + r[:, None])
    seen = seen[None, None].expand(B, 1, S, n)
    if start is not None:
        seen = seen & ((slot < 0) | (slot >= start[:, None].long()))[:, None, None]
    nobody = ~seen.any(2)[:, :, :, None]  # slots that no row of the request sees may hold anything
    k, ek, v, ev = (t.masked_fill(nobody, 0.0) for t in (k, ek, v, ev))
    w, mag = q.double(), abs(scale)
    score = (w @ k.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
    size = score.masked_fill(~seen, 0.0).abs()
    delta = mag * (w.abs() @ ek.transpose(2, 3) + (D + 4) * F * (w.abs() @ k.abs().transpose(2, 3))) + F * (8 * size + 16)
    if q.dtype == torch.bfloat16:
        delta = delta + mag * A * (k.abs() + ek).sum(3)[:, :, None]
    delta = delta.masked_fill(~seen, 0.0).amax(3, keepdim=True)
    top = score.amax(3, keepdim=True)
    e = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(3, keepdim=True)
    p = e / total.masked_fill(total == 0, 1.0)
    out = p @ v
    big = v.abs() + ev
    tol = p @ ev + (p @ big) * (torch.expm1(2 * delta) + H + n * F + 2.0**-20) + weight_step * (seen.double() @ big) / total.masked_fill(total == 0, 1.0)
    tol = tol + torch.finfo(q.dtype).eps / 2 * (out.abs() + tol) + (A if q.dtype == torch.float16 else 0.0)
    lse = (top + torch.log(total))[..., 0]
    return out, lse, tol, delta[..., 0] + n * F + 2.0**-20 + 2.0**-22 * lse.abs().nan_to_num(0.0, 0.0, 0.0)


def compare(got, want):
    """``got``: (out, lse) of a call; ``want``: what :func:`expected` gives. A row that sees nothing is 0, -inf."""
    (out, lse), (o, l, tol, tol_l) = got, want
    off = ((out.double() - o).abs() - tol).max()
    assert bool(((out.double() - o).abs() <= tol).all()), f"off by {off.item():.3e} more than allowed; max err {(out.double() - o).abs().max().item():.3e}"
    empty = l == -math.inf
    assert bool((lse[empty] == -math.inf).all()) and not bool(out[empty].any())
    assert bool(((lse.double() - l).abs() <= tol_l)[~empty].all())
