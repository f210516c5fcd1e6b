"""Rotary positions: the step between a layer's projections and its cache.

``RotaryEmbedding`` holds the frequencies of one model and turns queries and keys in one launch
(half or interleaved layout, all or part of the head, frequencies scaled for long contexts).
It is differentiable: the gradient is the inverse turn. :meth:`RotaryEmbedding.append` is the
form of a decode step: rotated queries out, rotated keys and the values straight behind the
unquantized window of a KIVI cache (used by ``KIVIKVCache.update_rotary``).

The reference has no counterpart: its caches receive keys that the model has rotated.
"""

from __future__ import annotations

import math
from typing import Any

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import _DTYPE_CODE as _DTYPE_CODES
from ._lib import ROTARY_PACK, check, lib, require_cuda, stream_ptr

_LAYOUTS = ("half", "interleaved")
_NO_STRIDE = (0, 0, 0)
_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


_empty_like = torch.empty_like


def _empty(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor like ``x`` (empty_like costs a third of torch.empty, but keeps strides)."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


_BASE = 10000.0
# What each kind of scaling takes beside its name and the base; the second set says nothing about the frequencies.
_SCALING_KEYS = {
    "default": set(),
    "linear": {"factor"},
    "ntk": {"factor"},
    "llama3": {"factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"},
    "yarn": {"factor", "original_max_position_embeddings", "attention_factor", "beta_fast", "beta_slow", "mscale", "mscale_all_dim", "truncate"},
}
_NO_EFFECT = {"rope_type", "type", "rope_theta", "original_max_position_embeddings", "max_position_embeddings", "finetuned"}


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the stretches of memory from the first to the last element of ``a`` and ``b`` meet."""
    if not (a.numel() and b.numel()):
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))) for t in (a, b))
    return a0 < b1 and b0 < a1


def rotary_frequencies(rotary_dim: int, base: float | None = None, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """Angle per position of each of the ``rotary_dim / 2`` pairs (float64, on the host) and the
    factor on sine and cosine.

    Without ``scaling``: ``base ** (-2 i / rotary_dim)`` and 1. ``base`` defaults to ``scaling["rope_theta"]``, or to
    10000; one that contradicts ``rope_theta`` is refused. ``scaling["rope_type"]`` is one of

    * ``"default"``;
    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: ``base`` raised to ``base * factor ** (r / (r - 2))``, ``r = rotary_dim``;
    * ``"llama3"``: wavelengths above ``original_max_position_embeddings / low_freq_factor`` are
      stretched by ``factor``, those below ``.../ high_freq_factor`` are kept, a linear ramp (in the
      number of turns over the original context) between;
    * ``"yarn"``: the same between the pairs that make ``beta_slow`` (1) and ``beta_fast`` (32) turns
      over the original context, the ramp linear in the pair's index (rounded outwards unless
      ``truncate`` is false); the factor on sine and cosine is ``attention_factor``, by default
      ``m(mscale) / m(mscale_all_dim)`` where both are given (and not 0), else ``m(1)``, with
      ``m(x) = 0.1 x ln(factor) + 1`` (1 for a factor of at most 1).

    A key that is None counts as absent; one that the kind does not know is refused, so that nothing that would change
    the frequencies is passed over (``partial_rotary_factor`` is the business of :class:`RotaryEmbedding`).
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_frequencies: rotary_dim={rotary_dim} must be even and at least 2")
    scaling = {name: x for name, x in (scaling or {}).items() if x is not None}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _SCALING_KEYS:
        raise ValueError(f"rotary_frequencies: unknown rope_type {kind!r}")
    unknown = sorted(str(name) for name in scaling if name not in _SCALING_KEYS[kind] and name not in _NO_EFFECT)
    if unknown:
        raise ValueError(f"rotary_frequencies: rope_type {kind!r} does not take {', '.join(map(repr, unknown))}")
    theta = scaling.get("rope_theta")
    if base is None:
        base = _BASE if theta is None else float(theta)
    elif theta is not None and float(theta) != float(base):
        raise ValueError(f"rotary_frequencies: base={base} contradicts rope_theta={theta}")
    if not base > 0:
        raise ValueError(f"rotary_frequencies: base={base} must be positive")
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)

    def need(name):
        if name not in scaling:
            raise ValueError(f"rotary_frequencies: rope_type {kind!r} needs {name!r}")
        return float(scaling[name])

    if kind == "default":
        return base ** (-2.0 * pair / rotary_dim), 1.0
    factor = need("factor")
    if not factor > 0:
        raise ValueError(f"rotary_frequencies: factor={factor} must be positive")
    if kind == "ntk":
        if rotary_dim > 2:  # (a single pair turns by one radian a position whatever the base)
            base = base * factor ** (rotary_dim / (rotary_dim - 2.0))
        return base ** (-2.0 * pair / rotary_dim), 1.0
    freq = base ** (-2.0 * pair / rotary_dim)
    if kind == "linear":
        return freq / factor, 1.0
    old = need("original_max_position_embeddings")
    if not old > 0:
        raise ValueError(f"rotary_frequencies: original_max_position_embeddings={old} must be positive")
    if kind == "llama3":
        lo, hi = need("low_freq_factor"), need("high_freq_factor")
        if not hi > lo:
            raise ValueError(f"rotary_frequencies: high_freq_factor={hi} must exceed low_freq_factor={lo}")
        turns = old * freq / (2.0 * math.pi)
        keep = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
        return freq * (keep + (1.0 - keep) / factor), 1.0
    # yarn: the index of the pair that makes n turns over the original context
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    if not (fast > 0 and slow > 0 and base != 1):
        raise ValueError(f"rotary_frequencies: beta_fast={fast} and beta_slow={slow} must be positive, base={base} other than 1")
    at = lambda n: rotary_dim * math.log(old / (n * 2.0 * math.pi)) / (2.0 * math.log(base))  # noqa: E731
    lo, hi = at(fast), at(slow)
    if scaling.get("truncate", True):
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
    if hi == lo:
        hi += 0.001
    stretched = ((pair - lo) / (hi - lo)).clamp(0.0, 1.0)
    m = lambda x: 0.1 * x * math.log(factor) + 1.0 if factor > 1.0 else 1.0  # noqa: E731
    if "attention_factor" in scaling:
        att = float(scaling["attention_factor"])
    elif scaling.get("mscale") and scaling.get("mscale_all_dim"):
        att = m(float(scaling["mscale"])) / m(float(scaling["mscale_all_dim"]))
    else:
        att = m(1.0)
    return freq * ((1.0 - stretched) + stretched / factor), att


class RotaryEmbedding:
    """The rotary positions of one model.

    ``head_dim`` channels a head, of which the first ``rotary_dim`` (default: all) are turned, in
    pairs ``(c, c + rotary_dim/2)`` (``layout="half"``) or ``(2c, 2c+1)`` (``"interleaved"``).
    The frequencies are :func:`rotary_frequencies` of ``base`` and ``scaling``, or ``inv_freq``
    (``[rotary_dim/2]``, angle per position, taken in float64); ``attention_factor`` overrides the
    factor on sine and cosine. ``scaling["partial_rotary_factor"]`` stands for
    ``rotary_dim = int(head_dim * factor)``; a ``rotary_dim`` that contradicts it is refused.

    ``rope(q, k, positions)`` returns the turned ``q`` and ``k`` (``rope(q)`` one tensor) as new
    contiguous tensors: ``q [B, H_q, S, D]``, ``k [B, H_kv, S, D]`` in float16, bfloat16 or float32
    with any strides (heads in the projection's ``[B, S, H, D]`` order included). ``positions`` is an
    integer tensor ``[S]``, ``[1, S]`` or ``[B, S]`` on the same device, or an int: the position of token
    0, the others following (default 0). ``inverse=True`` turns the other way, times the same
    ``attention_factor``: the gradient. Products are float32, angles float64 (exact
    to float32 for positions up to 2**31 and beyond); one rounding to the tensors' type at the end.
    Derivatives flow through ``q`` and ``k`` in reverse mode (also twice) and forward mode
    (``torch.autograd.forward_ad``), not through positions or frequencies.

    The frequency table is put on a device at its first use there; make that use (or pass
    ``device=``) before a CUDA-graph capture. Copies and pickles keep the tables that lie on their device. Where a backward pass is captured, PyTorch's own rule
    holds: no graph that an earlier eager pass built over the same leaves may still be alive.
    """

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, base: float | None = None, layout: str = "half",
                 scaling: dict | None = None, inv_freq: Any = None, attention_factor: float | None = None, device=None) -> None:
        part = scaling.get("partial_rotary_factor") if scaling else None
        if part is not None:
            scaling = {name: x for name, x in scaling.items() if name != "partial_rotary_factor"}
            if rotary_dim is not None and int(rotary_dim) != int(head_dim * part):
                raise ValueError(f"RotaryEmbedding: rotary_dim={rotary_dim} contradicts partial_rotary_factor={part} of head_dim={head_dim}")
            rotary_dim = int(head_dim * part)
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if head_dim < 2 or rotary_dim < 2 or rotary_dim > head_dim or rotary_dim % 2:
            raise ValueError(f"RotaryEmbedding: rotary_dim={rotary_dim} must be even and in 2..head_dim={head_dim}")
        if layout not in _LAYOUTS:
            raise ValueError(f"RotaryEmbedding: layout must be one of {_LAYOUTS}, got {layout!r}")
        if inv_freq is None:
            freq, factor = rotary_frequencies(rotary_dim, base, scaling)
        else:
            if scaling is not None:
                raise ValueError("RotaryEmbedding: give inv_freq or scaling, not both")
            freq, factor = torch.as_tensor(inv_freq).detach().to(torch.float64, copy=True), 1.0  # (the caller may reuse theirs)
            if tuple(freq.shape) != (rotary_dim // 2,):
                raise ValueError(f"RotaryEmbedding: inv_freq must have shape ({rotary_dim // 2},), got {tuple(freq.shape)}")
        self.head_dim, self.rotary_dim, self.layout = int(head_dim), rotary_dim, layout
        self._layout_code = _LAYOUTS.index(layout)
        self._freq = freq  # (float64, where it was given)
        self.attention_factor = float(factor if attention_factor is None else attention_factor)
        self._turns: dict = {}  # device index -> turns per position of each pair
        if device is None and freq.is_cuda:
            device = freq.device
        if device is not None:
            self._turns_on(torch.device(device))

    def __setstate__(self, state) -> None:
        # (a load may have put the tables elsewhere than on the device they are for: those are made anew at their next use)
        turns = {i: t for i, t in state["_turns"].items() if t.is_cuda and t.device.index == i}
        self.__dict__.update(state, _turns=turns)

    @property
    def inv_freq(self) -> torch.Tensor:
        """Angle per position of each pair, float64 on the host."""
        return self._freq.to("cpu", copy=True)

    def _turns_on(self, device: torch.device) -> int:
        """The table's address on ``device``."""
        index = device.index if device.index is not None else torch.cuda.current_device()
        t = self._turns.get(index)
        if t is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("RotaryEmbedding: first use on a device inside a graph capture; pass device= or call it once before")
            with _lib.on_device(torch.device("cuda", index)):
                t = self._freq.to(torch.device("cuda", index)) / (2.0 * math.pi)
                torch.cuda.current_stream().synchronize()  # (any stream may read it from here on)
            self._turns[index] = t
        return t.data_ptr()

    # -- checks --------------------------------------------------------------------------
    def _check(self, fn, q, k):
        shape, dt = q.shape, q.dtype
        if len(shape) != 4 or shape[3] != self.head_dim:
            raise ValueError(f"{fn}: q must be [B, H, S, {self.head_dim}], got {tuple(shape)}")
        if dt not in _DTYPES:
            raise ValueError(f"{fn}: unsupported dtype {dt}; expected float16, bfloat16 or float32")
        if k is None:
            return
        ks = k.shape
        if len(ks) != 4 or ks[3] != self.head_dim:
            raise ValueError(f"{fn}: k must be [B, H, S, {self.head_dim}], got {tuple(ks)}")
        if ks[0] != shape[0] or ks[2] != shape[2] or k.dtype is not dt or k.device != q.device:
            raise ValueError(f"{fn}: q {tuple(shape)} {dt} on {q.device} and k {tuple(ks)} {k.dtype} on {k.device} must agree in "
                             "batch, tokens, dtype and device")

    def _check_append(self, q, k, v):
        fn = "RotaryEmbedding.append"
        self._check(fn, q, k)
        if v.shape != k.shape or v.dtype is not k.dtype or v.device != k.device:
            raise ValueError(f"{fn}: v {tuple(v.shape)} {v.dtype} must be like k {tuple(k.shape)} {k.dtype}")
        if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or (
                forward_ad._current_level >= 0 and _lib.carries_derivative(q, k, v)):
            raise ValueError(f"{fn}: not differentiable; rotate and append to the cache separately, or call it under torch.no_grad()")

    @staticmethod
    def _positions(fn, positions, B, S, device):
        """(tensor or None, stride_b, stride_s, offset)."""
        if positions is None:
            return None, 0, 0, 0
        if isinstance(positions, int):
            return None, 0, 0, positions
        if not isinstance(positions, torch.Tensor) or (positions.dtype is not torch.int64 and positions.dtype is not torch.int32):
            raise ValueError(f"{fn}: positions must be an int or an int32 / int64 tensor")
        shape, st = positions.shape, positions.stride()
        if len(shape) == 2 and shape[1] == S and (shape[0] == B or shape[0] == 1):
            sb = st[0] if shape[0] > 1 else 0
        elif len(shape) == 1 and shape[0] == S:
            sb = 0
        else:
            raise ValueError(f"{fn}: positions must be [{S}], [1, {S}] or [{B}, {S}], got {list(shape)}")
        if positions.device != device:
            raise ValueError(f"{fn}: positions are on {positions.device}, q on {device}")
        return positions, sb, st[-1], 0

    def _launch(self, fn, q, xs, q_out, k, ks, k_out, k_out_strides, v_ptr, Hv, vs, v_out, v_out_strides, positions, inverse) -> None:
        """``q`` (strides ``xs``) to the contiguous tensor ``q_out``; ``k`` turned and ``v`` copied to addresses
        (``k`` None and ``v_ptr`` 0: not given)."""
        B, Hq, S, D = q.shape
        dev = q.device
        if k is None:
            k_ptr = Hk = 0
        else:
            k_ptr, Hk = k.data_ptr(), k.shape[1]
        if positions is None or type(positions) is int:
            pos_ptr = psb = pss = 0
            pos_bytes, off = 8, positions or 0
        else:
            pos, psb, pss, off = self._positions(fn, positions, B, S, dev)
            pos_ptr, pos_bytes = (0, 8) if pos is None else (pos.data_ptr(), 8 if pos.dtype is torch.int64 else 4)
        index = dev.index
        turns = self._turns.get(index)
        row = S * D
        a = ROTARY_PACK.pack(
            q.data_ptr(), k_ptr, v_ptr, q_out.data_ptr(), k_out, v_out, xs[0], xs[1], xs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], Hq * row, row, D,
            k_out_strides[0], k_out_strides[1], k_out_strides[2], v_out_strides[0], v_out_strides[1], v_out_strides[2],
            Hq, Hk, Hv, _DTYPE_CODES[q.dtype], B, S, D, self.rotary_dim, self._layout_code, 1 if inverse else 0, pos_ptr, pos_bytes,
            self.attention_factor, psb, pss, off, self._turns_on(dev) if turns is None else turns.data_ptr())
        native = lib()
        if index == torch.cuda.current_device():  # (the usual case, without a context manager)
            status = native.vq_rotary(a, stream_ptr(dev))
        else:
            with _lib.on_device(dev):
                status = native.vq_rotary(a, stream_ptr(dev))
        if status:
            check(status, fn)

    # -- calls ---------------------------------------------------------------------------
    def __call__(self, q: torch.Tensor, k: torch.Tensor | None = None, positions=None, *, inverse: bool = False):
        fn = "RotaryEmbedding"
        self._check(fn, q, k)
        if forward_ad._current_level >= 0 or (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
            out = _Rotate.apply(self, positions, inverse, q, k)
        else:
            out = self._rotate(fn, q, k, positions, inverse)
        return out[0] if k is None else out

    def _rotate(self, fn, q, k, positions, inverse):
        if not q.is_cuda:
            require_cuda(q, f"{fn}: q")
        xs = q.stride()
        if xs[3] != 1:
            q = q.contiguous()
            xs = q.stride()
        yq = _empty_like(q) if q.is_contiguous() else _empty(q)
        if k is None:
            self._launch(fn, q, xs, yq, None, _NO_STRIDE, 0, _NO_STRIDE, 0, 0, _NO_STRIDE, 0, _NO_STRIDE, positions, inverse)
            return yq, None
        ks = k.stride()
        if ks[3] != 1:
            k = k.contiguous()
            ks = k.stride()
        yk = _empty_like(k) if k.is_contiguous() else _empty(k)
        _, H, S, D = k.shape
        row = S * D
        self._launch(fn, q, xs, yq, k, ks, yk.data_ptr(), (H * row, row, D), 0, 0, _NO_STRIDE, 0, _NO_STRIDE, positions, inverse)
        return yq, yk

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_res: torch.Tensor, v_res: torch.Tensor, tok_offset: int,
               positions=None) -> torch.Tensor:
        """Turn ``q [B,H_q,S,D]`` and ``k [B,H_kv,S,D]`` in one launch, writing the turned keys and
        ``v [B,H_kv,S,D]`` to rows ``[tok_offset, tok_offset + S)`` of ``k_res / v_res [B,H_kv,cap,D]``
        (the exact window of a KIVI cache: the rotating form of ``kernels.kivi_append``); returns the
        turned queries. The other rows stay as they are. Inputs must not lie within the memory that
        ``k_res`` / ``v_res`` span. Not differentiable."""
        fn = "RotaryEmbedding.append"
        self._check_append(q, k, v)
        B, H, S, D = k.shape
        for name, t in (("k_res", k_res), ("v_res", v_res)):
            shape, stride = t.shape, t.stride()
            if len(shape) != 4 or shape[0] != B or shape[1] != H or shape[3] != D or t.dtype is not k.dtype or t.device != k.device:
                raise ValueError(f"{fn}: {name} must be [{B}, {H}, rows, {D}] {k.dtype} on {k.device}, got {tuple(shape)} {t.dtype} on {t.device}")
            if stride[3] != 1 or stride[2] < D or not stride[0] or not stride[1]:
                raise ValueError(f"{fn}: the channels of {name} must be contiguous and its rows apart, got strides {stride}")
            if tok_offset < 0 or tok_offset + S > shape[2]:
                raise ValueError(f"{fn}: rows [{tok_offset}, {tok_offset + S}) exceed {name} ({shape[2]} rows)")
        require_cuda(q, f"{fn}: q")
        if q.stride(3) != 1:
            q = q.contiguous()
        if k.stride(3) != 1:
            k = k.contiguous()
        if v.stride(3) != 1:
            v = v.contiguous()
        if k_res.data_ptr() == v_res.data_ptr():
            raise ValueError(f"{fn}: k_res and v_res must be different memory")
        held = (k_res.untyped_storage().data_ptr(), v_res.untyped_storage().data_ptr())
        if q.untyped_storage().data_ptr() in held or k.untyped_storage().data_ptr() in held or v.untyped_storage().data_ptr() in held:
            # (one storage: views of different parts of it are fine)
            if any(_overlap(x, t) for x in (q, k, v) for t in (k_res, v_res)):
                raise ValueError(f"{fn}: q, k and v must not share memory with k_res / v_res")
        out = _empty(q)
        es = k.element_size()
        ks, vs = k_res.stride(), v_res.stride()
        self._launch(fn, q, q.stride(), out, k, k.stride(), k_res.data_ptr() + tok_offset * ks[2] * es, ks, v.data_ptr(), H, v.stride(),
                     v_res.data_ptr() + tok_offset * vs[2] * es, vs, positions, False)
        return out


def _turn(rope, positions, inverse, q, k):
    return rope._rotate("RotaryEmbedding", q, k, positions, inverse)


class _Rotate(torch.autograd.Function):
    """The turn as a differentiable operation: linear in q and k, its gradient is the inverse turn, its derivative along a
    direction the direction's own turn."""

    @staticmethod
    def forward(ctx, rope, positions, inverse, q, k):
        ctx.rope, ctx.inverse = rope, inverse
        ctx.set_materialize_grads(False)
        ctx.tensor_positions = isinstance(positions, torch.Tensor)
        if ctx.tensor_positions:
            ctx.save_for_backward(positions)
        else:
            ctx.positions = positions
        out = _turn(rope, positions, inverse, q, k)
        if forward_ad._current_level >= 0:
            ctx.tangent_positions = positions
            ctx.like = [None if y is None else (y.shape, y.dtype, y.device) for y in out]
        return out

    @staticmethod
    def jvp(ctx, _rope, _positions, _inverse, tq, tk):
        shapes, positions = ctx.like, ctx.tangent_positions
        # (a tangent may be torch's placeholder for zeros, which has no memory)
        tq, tk = (t.clone() if t is not None and t._is_zerotensor() else t for t in (tq, tk))
        if tq is not None:
            tq, tk = _Rotate.apply(ctx.rope, positions, ctx.inverse, tq, tk)
        elif tk is not None:
            tk = _Rotate.apply(ctx.rope, positions, ctx.inverse, tk, None)[0]
        return tuple(torch.zeros(like[0], dtype=like[1], device=like[2]) if t is None and like is not None else t for t, like in zip((tq, tk), shapes))

    @staticmethod
    def backward(ctx, gq, gk):
        positions = ctx.saved_tensors[0] if ctx.tensor_positions else ctx.positions
        need_q, need_k = ctx.needs_input_grad[3], ctx.needs_input_grad[4]
        gq, gk = gq if need_q else None, gk if need_k else None
        # (through the function again only where a second derivative may be asked for, in either mode)
        turn = _Rotate.apply if torch.is_grad_enabled() or forward_ad._current_level >= 0 else _turn
        if gq is not None:
            gq, gk = turn(ctx.rope, positions, not ctx.inverse, gq, gk)
        elif gk is not None:
            gk = turn(ctx.rope, positions, not ctx.inverse, gk, None)[0]
        return None, None, None, gq, gk


__all__ = ["RotaryEmbedding", "rotary_frequencies"]
