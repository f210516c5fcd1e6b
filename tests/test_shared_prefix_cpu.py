"""Refusals of the shared-prefix attention and its cache, before the device is looked at."""

from __future__ import annotations

import pytest
import torch

from veloxquant_mlx_b200 import VQLibraryError
from veloxquant_mlx_b200.kernels import KiviRows, kivi_shared_prefix_attend


def _store(B=1, H=2, n=64, r=5, D=128, bits=4, dtype=torch.float16, **kw):
    t = dict(k_codes=torch.zeros(B, H, n, D * bits // 8, dtype=torch.uint8), k_scale=torch.zeros(B, H, n // 32, D), k_zero=torch.zeros(B, H, n // 32, D),
             v_codes=torch.zeros(B, H, n, D * bits // 8, dtype=torch.uint8), v_scale=torch.zeros(B, H, n, D // 32), v_zero=torch.zeros(B, H, n, D // 32),
             k_res=torch.zeros(B, H, r, D, dtype=dtype), v_res=torch.zeros(B, H, r, D, dtype=dtype), store_bits=bits)
    t.update(kw)
    return t


def test_rows_count_and_resize():
    r = KiviRows(**_store(n=96, r=7))
    assert (len(r), r.n_quant, r.n_res, r.batch, r.heads, r.head_dim, r.store_bits) == (103, 96, 7, 1, 2, 128, 4)
    r.resize(32, 2, 5)
    assert len(r) == 34
    for bad in ((33, 0, 0), (128, 0, 0), (-32, 0, 0), (0, 8, 0), (0, 3, 5), (0, -1, 0), (0, 1, -1)):
        with pytest.raises(ValueError, match="KiviRows"):
            r.resize(*bad)
    only = {k: v for k, v in _store().items() if k.endswith("_res")}
    assert len(KiviRows(**only)) == 5
    assert len(KiviRows(**{k: v for k, v in _store().items() if not k.endswith("_res")})) == 64


@pytest.mark.parametrize("change,what", [
    (dict(group_size=64), "group_size"), (dict(store_bits=1), "store_bits"), (dict(k_scale=None), "missing"), (dict(k_res=None), "together"),
    (dict(k_codes=torch.zeros(1, 2, 64, 64)), "uint8"), (dict(k_codes=torch.zeros(1, 2, 64, 32, dtype=torch.uint8)), "rows of 64 bytes"),
    (dict(v_codes=torch.zeros(1, 2, 32, 64, dtype=torch.uint8)), "same tokens"), (dict(k_scale=torch.zeros(1, 2, 2, 128).half()), "float32"),
    (dict(k_scale=torch.zeros(1, 2, 2, 64)), "k_scale"), (dict(v_zero=torch.zeros(1, 2, 64, 2)), "v_scale"), (dict(k_zero=torch.zeros(2, 2, 2, 128)), "leading"),
    (dict(k_res=torch.zeros(1, 2, 5, 128)), "equal float16"), (dict(v_res=torch.zeros(1, 2, 4, 128).half()), "equal float16"),
    (dict(v_codes=torch.zeros(1, 2, 64, 128, dtype=torch.uint8)[..., ::2]), "contiguous"), (dict(n_quant=96), "n_quant"), (dict(n_res=6), "exceed"),
    (dict(k_res=torch.zeros(1, 2, 5, 96).half(), v_res=torch.zeros(1, 2, 5, 96).half()), "head_dim"),
])
def test_bad_stores_are_refused(change, what):
    with pytest.raises(ValueError, match=what):
        KiviRows(**{**_store(), **change})


def test_bad_calls_are_refused_and_a_cpu_tensor_loudly():
    prefix, own = KiviRows(**_store()), KiviRows(**_store(B=3, n=0, r=4))
    q = torch.zeros(3, 8, 1, 128, dtype=torch.float16)
    call = lambda q=q, p=prefix, o=own, **kw: kivi_shared_prefix_attend(q, p, o, 0.1, **kw)  # noqa: E731
    for kw, what in [
        (dict(q=q[0]), "4D"), (dict(q=q.float()), "float16 or bfloat16"), (dict(p=own), "batch 1"), (dict(p=None), "KiviRows"), (dict(o=q), "KiviRows"),
        (dict(q=q[:2]), "own has batch 3"), (dict(q=q[:, :7]), "multiple of"), (dict(q=q.bfloat16()), "exact rows of prefix"),
        (dict(q=q[..., :64].contiguous()), "expected"), (dict(o=KiviRows(**_store(B=3, bits=2))), "expected"), (dict(o=KiviRows(**_store(B=3, H=1))), "expected"),
        (dict(q=q.expand(3, 8, 5, 128)), "5 causal query rows but only 4"), (dict(own_start=torch.zeros(3)), "own_start"),
        (dict(own_start=torch.zeros(2, dtype=torch.int32)), "own_start"), (dict(out=torch.zeros(3, 8, 1, 128)), "out must be"),
        (dict(q=q.clone().requires_grad_(True)), "not differentiable"),
    ]:
        with pytest.raises(ValueError, match=what):
            call(**kw)
    with pytest.raises(VQLibraryError):
        call()


def test_a_fork_needs_a_prefilled_kivi_cache_of_batch_one():
    from veloxquant_mlx_b200.cache import DenseKVCache, KIVIKVCache, QuantizerConfigError
    from veloxquant_mlx_b200.shared_prefix import SharedPrefixKIVICache

    with pytest.raises(QuantizerConfigError, match="must be a KIVIKVCache"):
        SharedPrefixKIVICache(DenseKVCache(), 4)
    c = object.__new__(KIVIKVCache)  # (the constructor asks for a device; only the checks run here)
    c.offset, c._k_res = 0, None
    with pytest.raises(QuantizerConfigError, match="batch=0"):
        SharedPrefixKIVICache(c, 0)
    with pytest.raises(QuantizerConfigError, match="empty"):
        SharedPrefixKIVICache(c, 4)
    c.offset, c._k_res, c._shape_bhd = 9, torch.zeros(2, 2, 9, 128), (2, 2, 128)
    with pytest.raises(QuantizerConfigError, match="batch 1"):
        SharedPrefixKIVICache(c, 4)
    c._shape_bhd, c._head_dim, c._group_size, c._sb, c._b = (1, 2, 96), 96, 32, 4, 4
    with pytest.raises(QuantizerConfigError, match="head_dim 64 or 128"):
        SharedPrefixKIVICache(c, 4)
    c._head_dim = 128
    with pytest.raises(QuantizerConfigError, match="float16 or bfloat16"):
        SharedPrefixKIVICache(c, 4)


def test_struct_sizes_match_header(tmp_path):
    import ctypes
    import os
    import subprocess

    from veloxquant_mlx_b200 import _lib

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include "vqb200.h"\nint main(){printf("%zu %zu %zu\\n",sizeof(vq_rotary_args),sizeof(vq_kivi_rows),'
                   'sizeof(vq_shared_attend_args));return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == [ctypes.sizeof(t) for t in (_lib.RotaryArgs, _lib.KiviRowsArgs, _lib.SharedAttendArgs)]
    # the packed forms that the wrappers pass: the same bytes as the structures, field by field
    for fmt, cls in ((_lib.ROTARY_PACK, _lib.RotaryArgs), (_lib.KIVI_ROWS_PACK, _lib.KiviRowsArgs)):
        assert fmt.size == ctypes.sizeof(cls)
    assert _lib.SHARED_ATTEND_HEAD.size == _lib.SharedAttendArgs.prefix.offset
    assert _lib.SHARED_ATTEND_HEAD.size + 2 * _lib.KIVI_ROWS_PACK.size == _lib.SharedAttendArgs.workspace.offset
    assert _lib.SHARED_ATTEND_HEAD.size + 2 * _lib.KIVI_ROWS_PACK.size + _lib.SHARED_ATTEND_TAIL.size == ctypes.sizeof(_lib.SharedAttendArgs)
    r = _lib.RotaryArgs.from_buffer_copy(_lib.ROTARY_PACK.pack(*range(1, 37), 37.0, 38, 39, 40, 41))
    assert list(r.x) == [1, 2, 3] and list(r.y_stride) == list(range(16, 25)) and list(r.heads) == [25, 26, 27] and r.dtype == 28
    assert (r.B, r.S, r.D, r.rotary_dim, r.layout, r.inverse, r.positions, r.pos_bytes) == (29, 30, 31, 32, 33, 34, 35, 36)
    assert (r.factor, r.pos_stride_b, r.pos_stride_s, r.pos_offset, r.turns) == (37.0, 38, 39, 40, 41)
    k = _lib.KiviRowsArgs.from_buffer_copy(_lib.KIVI_ROWS_PACK.pack(*range(1, 16)))
    assert (k.k_codes, k.v_res, k.k_codes_stride_bh, k.res_stride_bh, k.n_quant, k.n_res) == (1, 8, 9, 13, 14, 15)


def test_value_scales_whose_slabs_would_be_off_16_bytes_are_refused():
    """head_dim 64 has two scales a token: with an odd number of tokens the next head's would start 8 bytes off."""
    from veloxquant_mlx_b200 import _lib

    odd = dict(v_scale=torch.zeros(1, 2, 65, 2), v_zero=torch.zeros(1, 2, 65, 2))
    with pytest.raises(ValueError, match="even number of tokens"):
        KiviRows(**{**_store(D=64), **odd})
    good = KiviRows(**_store(D=64))._args
    head = _lib.SHARED_ATTEND_HEAD.pack(64, 64, 0, 0, 0, 1, 2, 2, 1, 64, 4, 32, 0.1, 0)
    tail = _lib.SHARED_ATTEND_TAIL.pack(0, 0, 0, 0)
    need = _lib.lib().vq_kivi_shared_attend_workspace_bytes
    assert need(head + good + bytes(_lib.KIVI_ROWS_PACK.size) + tail) > 0
    fields = list(_lib.KIVI_ROWS_PACK.unpack(good))
    assert fields[11] == 128  # v_param_stride_bh
    fields[11] = 130
    assert need(head + _lib.KIVI_ROWS_PACK.pack(*fields) + bytes(_lib.KIVI_ROWS_PACK.size) + tail) == 0
