"""Attention of a batch that shares a prefix, over packed KIVI codes.

Many requests behind one system prompt: the prompt's packed keys and values exist once and are read
once per call for all requests (``kivi_shared_prefix_attend``), each request's own tokens follow in
a store of their own. ``SharedPrefixKIVICache`` is that pair behind the cache protocol: a prefilled
``KIVIKVCache`` of batch 1, forked for ``batch`` requests.

The reference has no counterpart: its prompt cache hands every request a copy.
"""

from __future__ import annotations

from typing import Any

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import KIVI_ROWS_PACK, SHARED_ATTEND_HEAD, SHARED_ATTEND_TAIL, check, lib, require_cuda, stream_ptr

_GROUP = 32


class KiviRows:
    """Keys and values of one packed KIVI store, checked once and passed to
    :func:`kivi_shared_prefix_attend` any number of times.

    ``k_codes / v_codes u8 [B,H_kv,cap,D*store_bits/8]``, ``k_scale / k_zero f32 [B,H_kv,cap/32,D]``,
    ``v_scale / v_zero f32 [B,H_kv,cap,D/32]`` (contiguous; all None: no packed tokens), of which the first
    ``n_quant`` (default: all) tokens are live; ``k_res / v_res [B,H_kv,rows,D]`` float16 or bfloat16
    (contiguous, or None) hold the exact rows that follow them, ``n_res`` of them (default: all) from row
    ``res_offset``. Group size 32, head_dim 64 or 128, 2-, 4- or 8-bit containers. The tensors are
    referenced, not copied."""

    def __init__(self, k_codes=None, k_scale=None, k_zero=None, v_codes=None, v_scale=None, v_zero=None, k_res=None, v_res=None, *,
                 group_size: int = 32, store_bits: int = 4, n_quant: int | None = None, n_res: int | None = None, res_offset: int = 0) -> None:
        fn = "KiviRows"
        if group_size != _GROUP:
            raise ValueError(f"{fn}: group_size={group_size} must be 32")
        if store_bits not in (2, 4, 8):
            raise ValueError(f"{fn}: store_bits={store_bits} must be 2, 4 or 8")
        packed = {"k_codes": k_codes, "k_scale": k_scale, "k_zero": k_zero, "v_codes": v_codes, "v_scale": v_scale, "v_zero": v_zero}
        given = [t is not None for t in packed.values()]
        if any(given) and not all(given):
            raise ValueError(f"{fn}: codes, scales and zeros come together, missing {[n for n, t in packed.items() if t is None]}")
        if (k_res is None) != (v_res is None):
            raise ValueError(f"{fn}: k_res and v_res come together")
        tensors = [(n, t) for n, t in (*packed.items(), ("k_res", k_res), ("v_res", v_res)) if t is not None]
        if not tensors:
            raise ValueError(f"{fn}: no tokens given")
        first = tensors[0][1]
        if first.ndim != 4:
            raise ValueError(f"{fn}: {tensors[0][0]} must be 4D, got {tuple(first.shape)}")
        B, H = first.shape[:2]
        if H < 1:
            raise ValueError(f"{fn}: at least one kv head expected, got {tuple(first.shape)}")
        D = k_res.shape[-1] if k_res is not None else k_codes.shape[3] * 8 // store_bits
        if D not in (64, 128):
            raise ValueError(f"{fn}: head_dim={D} must be 64 or 128")
        for name, t in tensors:
            if t.ndim != 4 or tuple(t.shape[:2]) != (B, H):
                raise ValueError(f"{fn}: {name} must be 4D with leading [{B}, {H}], got {tuple(t.shape)}")
            if not t.is_contiguous():
                raise ValueError(f"{fn}: {name} must be contiguous")
            if t.device != first.device:
                raise ValueError(f"{fn}: {name} is on {t.device}, {tensors[0][0]} on {first.device}")
        cap = cap_res = 0
        pointers, strides, res_stride = (0,) * 6, (0,) * 4, 0
        if k_codes is not None:
            rb = D * store_bits // 8
            if k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8 or k_codes.shape[3] != rb or v_codes.shape[3] != rb:
                raise ValueError(f"{fn}: k_codes / v_codes must be uint8 with rows of {rb} bytes, got {tuple(k_codes.shape)} / {tuple(v_codes.shape)}")
            if any(packed[n].dtype != torch.float32 for n in ("k_scale", "k_zero", "v_scale", "v_zero")):
                raise ValueError(f"{fn}: scales and zeros must be float32")
            cap = min(k_codes.shape[2], v_codes.shape[2])
            if k_scale.shape != k_zero.shape or k_scale.shape[3] != D:
                raise ValueError(f"{fn}: k_scale / k_zero must be equal [{B}, {H}, groups, {D}], got {tuple(k_scale.shape)} / {tuple(k_zero.shape)}")
            if v_scale.shape != v_zero.shape or v_scale.shape[3] != D // _GROUP:
                raise ValueError(f"{fn}: v_scale / v_zero must be equal [{B}, {H}, tokens, {D // _GROUP}], got {tuple(v_scale.shape)} / {tuple(v_zero.shape)}")
            if v_scale.shape[2] * v_scale.shape[3] % 4:
                raise ValueError(f"{fn}: v_scale / v_zero must hold an even number of tokens at head_dim 64, got {v_scale.shape[2]}")
            cap = min(cap, k_scale.shape[2] * _GROUP, v_scale.shape[2])
            pointers = tuple(t.data_ptr() for t in (k_codes, v_codes, k_scale, k_zero, v_scale, v_zero))
            if any(packed[n].data_ptr() % 16 for n in packed):
                raise ValueError(f"{fn}: codes, scales and zeros must be 16-byte aligned")
            if k_codes.shape[2] != v_codes.shape[2]:
                raise ValueError(f"{fn}: k_codes and v_codes must hold the same tokens, got {k_codes.shape[2]} and {v_codes.shape[2]}")
            strides = (k_codes.shape[2] * rb, v_codes.shape[2] * rb, k_scale.shape[2] * D, v_scale.shape[2] * (D // _GROUP))
        self.dtype = None
        if k_res is not None:
            if k_res.dtype not in (torch.float16, torch.bfloat16) or v_res.dtype != k_res.dtype or v_res.shape != k_res.shape:
                raise ValueError(f"{fn}: k_res / v_res must be equal float16 or bfloat16 shapes, got {tuple(k_res.shape)} {k_res.dtype} / "
                                 f"{tuple(v_res.shape)} {v_res.dtype}")
            if k_res.data_ptr() % 16 or v_res.data_ptr() % 16:
                raise ValueError(f"{fn}: k_res / v_res must be 16-byte aligned")
            cap_res = k_res.shape[2]
            self.dtype = k_res.dtype
            res_stride = cap_res * D
        self.batch, self.heads, self.head_dim, self.store_bits, self.device = B, H, D, store_bits, first.device
        self._cap, self._cap_res, self._pointers, self._strides = cap, cap_res, pointers, (*strides, res_stride)
        self._tensors = (k_codes, k_scale, k_zero, v_codes, v_scale, v_zero, k_res, v_res)  # (kept alive)
        self._grad = any(t is not None and t.requires_grad for t in self._tensors)
        self._k_res_ptr, self._v_res_ptr = (0, 0) if k_res is None else (k_res.data_ptr(), v_res.data_ptr())
        self.resize(cap // _GROUP * _GROUP if n_quant is None else n_quant, cap_res - res_offset if n_res is None else n_res, res_offset)

    def resize(self, n_quant: int, n_res: int, res_offset: int = 0) -> None:
        """Another number of live tokens over the same buffers."""
        if n_quant < 0 or n_quant % _GROUP or n_quant > self._cap:
            raise ValueError(f"KiviRows: n_quant={n_quant} must be a multiple of 32 within the {self._cap} packed tokens held")
        if n_res < 0 or res_offset < 0 or res_offset + n_res > self._cap_res:
            raise ValueError(f"KiviRows: rows [{res_offset}, {res_offset + n_res}) exceed the exact rows ({self._cap_res})")
        skip = res_offset * self.head_dim * 2
        res = (self._k_res_ptr + skip, self._v_res_ptr + skip) if n_res else (0, 0)
        self._args = KIVI_ROWS_PACK.pack(*self._pointers, *res, *self._strides, n_quant, n_res)
        self.n_quant, self.n_res, self._res_offset = n_quant, n_res, res_offset

    def __reduce__(self):
        # (copies and pickles refer to their own tensors' memory, not to this object's)
        return _rows_again, (self._tensors, self.store_bits, self.n_quant, self.n_res, self._res_offset)

    def __len__(self) -> int:
        return self.n_quant + self.n_res


def _rows_again(tensors, store_bits, n_quant, n_res, res_offset):
    return KiviRows(*tensors, store_bits=store_bits, n_quant=n_quant, n_res=n_res, res_offset=res_offset)


_EMPTY = bytes(KIVI_ROWS_PACK.size)


def kivi_shared_prefix_attend(q: torch.Tensor, prefix: KiviRows, own: KiviRows | None, scale: float, *, causal: bool = True,
                              own_start: torch.Tensor | None = None, out: torch.Tensor | None = None, return_lse: bool = False,
                              variant: int = 0, n_splits: int = 0):
    """Attention of ``q [B,H_q,S_q,D]`` (float16 or bfloat16) over one ``prefix`` that all ``B`` requests
    share (``KiviRows`` of batch 1) followed by each request's ``own`` tokens (of batch ``B``, or None).
    Returns ``[B,H_q,S_q,D]`` in q's type; with ``return_lse`` also the natural log of each row's softmax sum
    ``f32 [B,H_q,S_q]``.

    Every query row sees the whole prefix. ``causal=True``: of the ``n`` own tokens row ``r`` sees the slots
    ``<= n - S_q + r``; ``causal=False``: all. ``own_start`` (``int32 [B]`` on the device): own slots before
    ``own_start[b]`` are padding and are not seen (a batch padded on the left). Their values, exact rows and key groups
    of padding alone may hold anything; padding keys that share a packed group of 32 with live tokens set its scale
    and zero and have to be finite and of ordinary size. A row that sees nothing gives zeros and ``lse`` -inf. An
    infinite or NaN value reaches every row of its request, seen or hidden by ``causal``.

    The prefix is read once for all query rows of a kv head. Decoded keys and values, the exact rows and q
    enter the tensor cores as float16 also for bfloat16 (so they must lie within +-65504; small ones keep 2^-25 absolute, and
    decoded bfloat16 ones of 2 and 4 bits 2^-20: bfloat16 values below about 2^-12 lose accuracy, 1.3 % at 1e-5, 14 % at
    1e-6), softmax and sums are float32. ``variant`` 1 / 2 force the warp-tile / the tensor-memory kernel for the prefix (2: ``scale`` > 0). Not
    differentiable: tensors that carry a derivative (either mode) are refused. A call takes ``4 (D + 2)`` bytes for
    each output row and split of either part from torch's allocator (at least two: 68 MB for 65,536 rows of 128).
    """
    fn = "kivi_shared_prefix_attend"
    if q.ndim != 4:
        raise ValueError(f"{fn}: q must be 4D, got {tuple(q.shape)}")
    B, H, S_q, D = q.shape
    dt = q.dtype
    if dt is not torch.float16 and dt is not torch.bfloat16:
        raise ValueError(f"{fn}: q must be float16 or bfloat16, got {dt}")
    if not isinstance(prefix, KiviRows) or not (own is None or isinstance(own, KiviRows)):
        raise ValueError(f"{fn}: prefix and own must be KiviRows")
    if prefix.batch != 1:
        raise ValueError(f"{fn}: the prefix must have batch 1, got {prefix.batch}")
    H_kv, bits = prefix.heads, prefix.store_bits
    dev = q.device
    for st in (prefix,) if own is None else (prefix, own):
        if st.head_dim != D or st.heads != H_kv or st.store_bits != bits:
            raise ValueError(f"{fn}: {'prefix' if st is prefix else 'own'} has {st.heads} heads of {st.head_dim} at {st.store_bits} bits; {H_kv} of {D} at "
                             f"{bits} expected")
        if st.device != dev:
            raise ValueError(f"{fn}: {'prefix' if st is prefix else 'own'} is on {st.device}, q on {dev}")
        if st.n_res and st.dtype is not dt:
            raise ValueError(f"{fn}: the exact rows of {'prefix' if st is prefix else 'own'} are {st.dtype}, q is {dt}")
    if own is not None and own.batch != B:
        raise ValueError(f"{fn}: own has batch {own.batch}, q {B}")
    if H % H_kv:
        raise ValueError(f"{fn}: H_q={H} must be a multiple of H_kv={H_kv}")
    if causal and own is not None and 0 < len(own) < S_q:
        raise ValueError(f"{fn}: {S_q} causal query rows but only {len(own)} own tokens")
    if own_start is not None:
        if own_start.dtype is not torch.int32 or tuple(own_start.shape) != (B,) or own_start.device != dev or not own_start.is_contiguous():
            raise ValueError(f"{fn}: own_start must be a contiguous int32 [{B}] tensor on {dev}, got {own_start.dtype} {tuple(own_start.shape)}")
    if (torch.is_grad_enabled() and (q.requires_grad or prefix._grad or (own is not None and own._grad))) or (
            forward_ad._current_level >= 0 and _lib.carries_derivative(q, *prefix._tensors, *(() if own is None else own._tensors))):
        raise ValueError(f"{fn}: not differentiable (q, exact rows, scales or zeros carry a derivative; call it under torch.no_grad())")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=dt, device=dev)
    elif out.shape != q.shape or out.dtype is not dt or out.device != dev or not out.is_contiguous():
        raise ValueError(f"{fn}: out must be a contiguous {tuple(q.shape)} {dt} tensor on {dev}")
    require_cuda(q, f"{fn}: q")
    if q.numel() == 0:
        return (out, q.new_empty((B, H, S_q), dtype=torch.float32)) if return_lse else out
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    if out.data_ptr() % 16:
        raise ValueError(f"{fn}: out must be 16-byte aligned")
    lse = torch.empty((B, H, S_q), dtype=torch.float32, device=dev) if return_lse else None
    head = SHARED_ATTEND_HEAD.pack(q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), 0 if own_start is None else own_start.data_ptr(),
                                   0 if dt is torch.float16 else 1, B, H, H_kv, S_q, D, bits, _GROUP, scale, _lib.VQ_ATTEND_CAUSAL if causal else 0)
    head += prefix._args + (_EMPTY if own is None else own._args)
    native = lib()
    with _lib.on_device(dev):
        need = native.vq_kivi_shared_attend_workspace_bytes(head + SHARED_ATTEND_TAIL.pack(0, 0, variant, n_splits))
        # (from torch's allocator at every call: calls on other streams and captured graphs have their own)
        ws = q.new_empty(need // 2 + 8)
        check(native.vq_kivi_shared_attend(head + SHARED_ATTEND_TAIL.pack(ws.data_ptr(), need, variant, n_splits), stream_ptr(dev)), fn)
    return out if lse is None else (out, lse)


from .cache import KIVIKVCache, KVCacheConfig, QuantizerConfigError  # noqa: E402
from .core import StandaloneProtocol  # noqa: E402


class SharedPrefixKIVICache(StandaloneProtocol):
    """``batch`` requests behind one prefilled prompt: a ``KIVIKVCache`` of batch 1 (the prefix, which is
    referenced and stays usable) and a ``KIVIKVCache`` for the requests' own tokens, of the prefix's bits,
    group size and residual length.

    Always memory-bound: ``update_and_fetch`` takes ``[batch,H_kv,S,D]`` and returns zero-length sentinels,
    ``fused_sdpa`` attends. ``offset`` counts the prefix. ``trim`` reaches back to the end of the prefix, not into
    it; ``reset`` drops the own tokens. ``own_start``: see :meth:`set_own_start`. The prefix may grow after the fork
    (the fork keeps the tokens it had); after it was trimmed, reset or reloaded the fork refuses to attend.
    Requires head_dim 64 or 128, group size 32, 2 to 8 bits, float16 or bfloat16."""

    def __init__(self, prefix: KIVIKVCache, batch: int, *, own_start=None) -> None:
        who = "SharedPrefixKIVICache"
        if type(prefix) is not KIVIKVCache:
            raise QuantizerConfigError(f"{who}: the prefix must be a KIVIKVCache, got {type(prefix).__name__}")
        if batch < 1:
            raise QuantizerConfigError(f"{who}: batch={batch} must be >= 1")
        if prefix.offset == 0 or prefix._k_res is None:
            raise QuantizerConfigError(f"{who}: the prefix is empty")
        if prefix._shape_bhd[0] != 1:
            raise QuantizerConfigError(f"{who}: the prefix must have batch 1, got {prefix._shape_bhd[0]}")
        if prefix._head_dim not in (64, 128) or prefix._group_size != _GROUP or prefix._sb not in (2, 4, 8):
            raise QuantizerConfigError(f"{who}: needs head_dim 64 or 128, group size 32 and 2 to 8 bits, got head_dim {prefix._head_dim}, group size "
                                       f"{prefix._group_size}, {prefix._b} bits")
        if prefix._k_res.dtype not in (torch.float16, torch.bfloat16):
            raise QuantizerConfigError(f"{who}: needs a float16 or bfloat16 prefix, got {prefix._k_res.dtype}")
        self._prefix, self._batch, self._head_dim = prefix, int(batch), prefix._head_dim
        self._memory_bound = True
        self._n_prefix = prefix.offset
        self._rollbacks = prefix._rollbacks
        nq = prefix._n_quantized
        kr, vr = (t.clone(memory_format=torch.contiguous_format) for t in prefix._live_res())  # (the window moves on; the packed store does not)
        packed = (prefix._k_codes, prefix._k_scale, prefix._k_zero, prefix._v_codes, prefix._v_scale, prefix._v_zero) if nq else (None,) * 6
        self._prefix_rows = KiviRows(*packed, kr, vr, group_size=_GROUP, store_bits=prefix._sb, n_quant=nq)
        self.own = KIVIKVCache(KVCacheConfig(method="kivi", head_dim=prefix._head_dim, bit_width_inlier=prefix._b, kivi_group_size=_GROUP,
                                             residual_length=prefix._residual_length, fused_sdpa_memory_bound=True))
        self._own_rows, self._own_version = None, -1
        self._start_host = None
        self._start = None
        if own_start is not None:
            self.set_own_start(own_start)

    def set_own_start(self, own_start) -> None:
        """Number of padding tokens at the front of each request's own tokens (a sequence of ``batch`` ints >= 0,
        or None): they take slots but are never seen, and positions count from the first token after them. Their
        keys go through the quantizer: they have to be finite and of ordinary size (see
        :func:`kivi_shared_prefix_attend`). It stays set over :meth:`reset` and :meth:`trim`."""
        if own_start is None:
            self._start_host = self._start = None
            return
        host = [int(x) for x in own_start]
        if len(host) != self._batch or min(host) < 0:
            raise ValueError(f"SharedPrefixKIVICache: own_start must be {self._batch} ints >= 0")
        self._start_host = host
        self._start = torch.tensor(host, dtype=torch.int32, device=self._prefix_rows.device)

    # -- protocol ----------------------------------------------------------------------
    @property
    def offset(self) -> int:
        return self._n_prefix + self.own.offset

    @property
    def prefix_length(self) -> int:
        return self._n_prefix

    def _check_block(self, keys, fn) -> None:
        want = (self._batch, self._prefix_rows.heads)
        if keys.ndim != 4 or tuple(keys.shape[:2]) != want:
            raise ValueError(f"SharedPrefixKIVICache.{fn}: keys must be [{want[0]}, {want[1]}, S, {self._head_dim}], got {tuple(keys.shape)}")
        if keys.dtype is not self._prefix_rows.dtype or keys.device != self._prefix_rows.device:
            raise ValueError(f"SharedPrefixKIVICache.{fn}: keys are {keys.dtype} on {keys.device}, the prefix {self._prefix_rows.dtype} on {self._prefix_rows.device}")

    def update_and_fetch(self, keys: torch.Tensor, values: torch.Tensor):
        self._check_block(keys, "update_and_fetch")
        return self.own.update_and_fetch(keys, values)

    def update_rotary(self, q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, rope: Any, positions=None):
        """``KIVIKVCache.update_rotary`` on the own tokens; the default positions follow the prefix and skip
        each request's padding."""
        self._check_block(keys, "update_rotary")
        if positions is None:
            first, S = self.offset, keys.shape[2]
            positions = first
            if self._start is not None:
                positions = torch.arange(first, first + S, dtype=torch.int32, device=keys.device) - self._start[:, None]
        return self.own.update_rotary(q, keys, values, rope, positions)

    def fused_sdpa(self, q: torch.Tensor, scale: float, *, causal: bool = True, sliding_window: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of ``q [batch,H_q,S_q,D]`` over the prefix and each request's own tokens (see
        :func:`kivi_shared_prefix_attend`)."""
        if sliding_window:
            raise ValueError("SharedPrefixKIVICache.fused_sdpa: sliding_window is not supported")
        if self._prefix._rollbacks != self._rollbacks:
            raise RuntimeError("SharedPrefixKIVICache.fused_sdpa: the prefix was trimmed, reset or reloaded after the fork")
        if q.ndim == 4 and q.shape[0] != self._batch:
            raise ValueError(f"SharedPrefixKIVICache.fused_sdpa: q has batch {q.shape[0]}, the cache {self._batch}")
        own, rows = self.own, None
        if own.offset:
            nq = own._n_quantized
            if self._own_version != (own._version, nq > 0):
                packed = (own._k_codes, own._k_scale, own._k_zero, own._v_codes, own._v_scale, own._v_zero) if nq else (None,) * 6
                self._own_rows = KiviRows(*packed, own._k_res, own._v_res, group_size=_GROUP, store_bits=own._sb, n_quant=0, n_res=0)
                self._own_version = (own._version, nq > 0)
            rows = self._own_rows
            rows.resize(nq, own._n_res, own._res_lo)
        return kivi_shared_prefix_attend(q, self._prefix_rows, rows, scale, causal=causal, own_start=self._start, out=out)

    def trim(self, n: int) -> int:
        return self.own.trim(n)

    def is_trimmable(self) -> bool:
        return True

    def empty(self) -> bool:
        return False

    def size(self) -> int:
        return self.offset

    def _reset_tokens(self) -> None:
        self.own.reset()

    def check_status(self) -> None:
        """See ``KIVIKVCache.check_status``."""
        self.own.check_status()

    @property
    def nbytes(self) -> int:
        """The own tokens' live bytes; the shared prefix counts once, in its own cache."""
        return self.own.nbytes


__all__ = ["KiviRows", "kivi_shared_prefix_attend", "SharedPrefixKIVICache"]
