"""Copies (copy, deepcopy, pickle) of packed stores, KIVI caches and forks read and write memory of their own."""

from __future__ import annotations

import copy
import io
import pickle

import pytest
import torch

from veloxquant_mlx_b200 import _lib
from veloxquant_mlx_b200.kernels import KiviRows


def _addresses(rows):
    return [0 if t is None else t.data_ptr() for t in rows._tensors]


def _store(B=1, n=64, r=5):
    return dict(k_codes=torch.zeros(B, 2, n, 64, dtype=torch.uint8), k_scale=torch.zeros(B, 2, n // 32, 128), k_zero=torch.zeros(B, 2, n // 32, 128),
                v_codes=torch.zeros(B, 2, n, 64, dtype=torch.uint8), v_scale=torch.zeros(B, 2, n, 4), v_zero=torch.zeros(B, 2, n, 4),
                k_res=torch.zeros(B, 2, r, 128, dtype=torch.float16), v_res=torch.zeros(B, 2, r, 128, dtype=torch.float16))


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
@pytest.mark.parametrize("part", ["all", "packed", "exact"])
def test_a_store_points_at_its_own_tensors(part, again):
    t = _store()
    t = {n: x for n, x in t.items() if part == "all" or n.endswith("_res") == (part == "exact")}
    rows = KiviRows(**t, n_quant=32 if part != "exact" else 0, n_res=2 if part != "packed" else 0, res_offset=3 if part != "packed" else 0)
    other = again(rows)
    kc, ks, kz, vc, vs, vz, kr, vr = _addresses(other)
    skip = 3 * 128 * 2 if part != "packed" else 0
    assert _lib.KIVI_ROWS_PACK.unpack(other._args)[:8] == (kc, vc, ks, kz, vs, vz, kr + skip, vr + skip)
    assert (other.n_quant, other.n_res, len(other)) == (rows.n_quant, rows.n_res, len(rows))
    if again is not copy.copy:
        assert not set(_addresses(other)) & (set(_addresses(rows)) - {0})
    other.resize(0, other.n_res, other._res_offset)
    assert rows.n_quant == (32 if part != "exact" else 0)


@pytest.mark.gpu
def test_a_copied_fork_goes_its_own_way():
    from veloxquant_mlx_b200.cache import KVCacheConfig, KVCacheFactory
    from veloxquant_mlx_b200.rotary import RotaryEmbedding
    from veloxquant_mlx_b200.shared_prefix import SharedPrefixKIVICache

    rope = RotaryEmbedding(128)

    def block(B, S, seed):
        g = torch.Generator("cuda").manual_seed(seed)
        return [torch.randn(B, h, S, 128, device="cuda", generator=g).half() for h in (8, 2, 2)]

    def step(c, seed):
        q = c.update_rotary(*block(4, 1, seed), rope)[0]
        return c.fused_sdpa(q, 0.09)

    def run(cut):
        first = KVCacheFactory.create(KVCacheConfig(method="kivi", head_dim=128, bit_width_inlier=4, residual_length=32, fused_sdpa_memory_bound=True))
        first.update_rotary(*block(1, 90, 1), rope)
        fork = SharedPrefixKIVICache(first, 4)
        outs = [step(fork, s) for s in range(2, cut)]
        return fork, outs

    for cut in (5, 50):  # before and after own tokens were packed
        fork, _ = run(cut)
        ends = [copy.deepcopy(fork), None, fork]
        buffer = io.BytesIO()
        torch.save(fork, buffer)
        buffer.seek(0)
        ends[1] = torch.load(buffer, weights_only=False)
        got = []
        for way, c in enumerate(ends):  # three continuations, step by step in turn
            got.append([step(c, 1000 * way + s) for s in range(40)])
        for way in range(3):
            plain, _ = run(cut)
            want = [step(plain, 1000 * way + s) for s in range(40)]
            assert all(torch.equal(a, b) for a, b in zip(got[way], want))
        del fork, ends[0]


@pytest.mark.gpu
@pytest.mark.parametrize("method", ["kivi", "kivi_sink"])
def test_a_copied_cache_goes_its_own_way(method):
    from veloxquant_mlx_b200.cache import KVCacheConfig, KVCacheFactory

    def block(S, seed):
        g = torch.Generator("cuda").manual_seed(seed)
        return [torch.randn(1, 2, S, 128, device="cuda", generator=g).half() for _ in range(2)]

    def run(seeds):
        c = KVCacheFactory.create(KVCacheConfig(method=method, head_dim=128, bit_width_inlier=4, residual_length=32, fused_sdpa_memory_bound=True))
        c.update_and_fetch(*block(90, 1))
        for s in seeds:
            c.update_and_fetch(*block(1, s))
        return c

    one = run(range(2, 50))
    two = copy.deepcopy(one)
    for s in range(40):
        one.update_and_fetch(*block(1, 100 + s))
        two.update_and_fetch(*block(1, 200 + s))
    for c, base in ((one, 100), (two, 200)):
        want = run([*range(2, 50), *range(base, base + 40)])
        assert all(torch.equal(a, b) for a, b in zip(c.state, want.state))
