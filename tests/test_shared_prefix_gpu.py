"""Attention behind a shared packed prefix on the GPU against softmax(q k) v in 64 bits.

Tolerance, per output element, with u = 2^-11 (one rounding to float16) and everything else computed in 64 bits:
* keys: code*scale+zero carries 2^-9 * 2^-24 * 2^15 ... at most 2^-9 of a quantization step at 8 bits (2^-17 at 2 and 4 bits),
  then one rounding to float16, so a key channel is off by at most u |k| + 2^-9 * step + 2^-25; a query rounds to
  float16 only where bfloat16 leaves half's normal range (2^-25). A score is then off by
  delta = scale * sum_d |q_d| (u |k_d| + 2^-9 step_d + 2^-25) + 2^-25 |k_d| ..., plus float32 accumulation, (D + 4) 2^-24 scale sum |q_d k_d|;
* weights: a factor within exp(+-2 delta) (numerator and denominator), one rounding to float16 (u, and half's
  smallest step: weights below 2^-25 of the largest vanish), the exponential itself 2^-20;
* values: like keys; sums in float32 over n tokens, n 2^-24;
* output: one rounding, eps / 2.
|err| <= sum p |v| (exp(2 delta) - 1 + 2 u + n 2^-24 + 2^-19) + 2^-9 max step + 2^-25 sum |v| / sum of 2^(s - max) + eps / 2 |out|."""

from __future__ import annotations

import math

import pytest
import torch

from veloxquant_mlx_b200 import kernels
from veloxquant_mlx_b200.kernels import KiviRows, kivi_shared_prefix_attend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def make_store(B, H, D, bits, n_quant, n_res, dtype, seed, spare=0, loud=True):
    """A store and what it stands for in 64 bits: keys, values, quantization step of each."""
    g = _gen(seed)
    k = torch.randn(B, H, n_quant + n_res, D, device=DEV, generator=g)
    if loud:
        k = k * (1 + 4 * (torch.rand(1, H, 1, D, device=DEV, generator=g) < 0.05))
    k, v = k.to(dtype), torch.randn(B, H, n_quant + n_res, D, device=DEV, generator=g).to(dtype)
    t = {}
    if n_quant:
        t["k_codes"], t["k_scale"], t["k_zero"] = kernels.kivi_quantize(k[:, :, :n_quant], -2, 32, bits)
        t["v_codes"], t["v_scale"], t["v_zero"] = kernels.kivi_quantize(v[:, :, :n_quant], -1, 32, bits)
        if spare:  # capacity behind the live tokens, holding garbage
            def more(x, rows, junk):
                return torch.cat([x, torch.full((B, H, rows, x.shape[3]), junk, dtype=x.dtype, device=DEV)], 2)
            nan = float("nan")
            t = {n: more(x, spare // 32 if n in ("k_scale", "k_zero") else spare, 255 if x.dtype == torch.uint8 else nan) for n, x in t.items()}
    if n_res or not n_quant:
        t["k_res"], t["v_res"] = k[:, :, n_quant:].contiguous(), v[:, :, n_quant:].contiguous()
    rows = KiviRows(**t, store_bits=kernels.storage_bits(bits), n_quant=n_quant)
    return rows, dense_of(t, kernels.storage_bits(bits), n_quant, D, B, H)


def dense_of(t, sb, nq, D, B, H):
    out = []
    for name in "kv":
        parts, steps = [], []
        if nq:
            byte = t[name + "_codes"][:, :, :nq].long().repeat_interleave(8 // sb, 3)
            code = (byte >> (sb * (torch.arange(D, device=DEV) % (8 // sb)))) & (2**sb - 1)
            if name == "k":
                sc, ze = (t[name + p][:, :, : nq // 32].double().repeat_interleave(32, 2) for p in ("_scale", "_zero"))
            else:
                sc, ze = (t[name + p][:, :, :nq].double().repeat_interleave(32, 3) for p in ("_scale", "_zero"))
            parts.append(code * sc + ze)
            steps.append(sc)
        if t.get(name + "_res") is not None:
            parts.append(t[name + "_res"].double())
            steps.append(torch.zeros_like(parts[-1]))
        out += [torch.cat(parts, 2), torch.cat(steps, 2)]
    return out  # k, k steps, v, v steps


def reference(q, pre, own, scale, causal=True, start=None):
    """(out, lse, tolerance without the output's rounding) in 64 bits; a row that sees nothing is 0, -inf."""
    B, Hq, S, D = q.shape
    H = pre[0].shape[1]
    k, ks, v, vs = (torch.cat([p.expand(B, -1, -1, -1), o], 2) if own is not None else p.expand(B, -1, -1, -1) for p, o in zip(pre, own or pre))
    n_pre, n = pre[0].shape[2], k.shape[2]
    n_own = n - n_pre
    rep = Hq // H
    k, ks, v, vs = (x.repeat_interleave(rep, 1) for x in (k, ks, v, vs))
    slot = torch.arange(n, device=DEV) - n_pre
    r = torch.arange(S, device=DEV)
    seen = (slot[None] < 0) | (slot[None] <= n_own - S + r[:, None]) if causal else torch.ones(S, n, dtype=torch.bool, device=DEV)
    seen = seen[None, None].expand(B, 1, S, n)
    if start is not None:
        seen = seen & ((slot < 0) | (slot >= start[:, None].long()))[:, None, None]
    w = q.double()
    dead = ~seen.any(2, keepdim=True)[:, :, 0, :, None] if n else None  # slots nobody sees may hold NaN
    if n:
        k, v, ks, vs = (x.masked_fill(dead, 0.0) for x in (k, v, ks, vs))
    score = (w @ k.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
    u = 2.0**-11
    err_k = u * k.abs() + 2.0**-9 * ks + 2.0**-25
    delta = (w.abs() @ err_k.transpose(2, 3) + 2.0**-25 * k.abs().sum(3)[:, :, None] + (D + 4) * 2.0**-24 * (w.abs() @ k.abs().transpose(2, 3))) * scale
    delta = delta.masked_fill(~seen, 0.0).amax(3, keepdim=True) if n else torch.zeros(B, Hq, S, 1, device=DEV, dtype=torch.float64)
    top = score.amax(3, keepdim=True) if n else torch.full((B, Hq, S, 1), -math.inf, device=DEV, dtype=torch.float64)
    safe = top.masked_fill(top == -math.inf, 0.0)
    e = torch.exp(score - safe)
    total = e.sum(3, keepdim=True)
    p = e / total.masked_fill(total == 0, 1.0)
    out = p @ v
    tol = (p @ v.abs()) * (torch.expm1(2 * delta) + 2 * u + n * 2.0**-24 + 2.0**-19)
    if n:
        # a packed record may keep a maximum of its own part that lies up to 8 powers of two below a later one
        tol = tol + p @ (2.0**-9 * vs) + 2.0**-25 * (seen.double() @ v.abs()) / total.masked_fill(total == 0, 1.0) + 2.0**-25
    lse = (top + torch.log(total))[..., 0]
    return out, lse, tol, delta[..., 0]


def check(q, pre, own, scale, start=None, causal=True, **kw):
    (prows, pd), (orows, od) = pre, own if own is not None else (None, None)
    got, lse = kivi_shared_prefix_attend(q, prows, orows, scale, causal=causal, own_start=start, return_lse=True, **kw)
    kernels.attend_status()
    want, wlse, tol, delta = reference(q, pd, od, scale, causal, start)
    tol = tol + torch.finfo(q.dtype).eps / 2 * (want.abs() + tol) + (2.0**-25 if q.dtype == HF else 0)
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), f"off by {off.max().item():.3e} more than allowed; max err {(got.double() - want).abs().max().item():.3e}"
    empty = wlse == -math.inf
    assert bool((lse[empty] == -math.inf).all()) and bool((got.masked_select(empty[..., None].expand_as(got)) == 0).all())
    # lse: the scores' error, the sum's, and its own rounding
    assert bool(((lse.double() - wlse).abs()[~empty] <= (delta + 2.0**-16 + 2.0**-22 * wlse.abs())[~empty]).all())
    return got


CASES = [
    # B, Hq, Hk, S, D, bits, dtype, pre_q, pre_r, own_q, own_r
    (1, 1, 1, 1, 128, 4, HF, 32, 0, 0, 1),
    (3, 8, 2, 1, 128, 4, HF, 64, 7, 0, 40),
    (3, 8, 2, 1, 128, 4, BF, 64, 7, 32, 33),
    (5, 10, 2, 1, 128, 2, HF, 320, 77, 64, 130),
    (2, 4, 4, 1, 128, 8, BF, 96, 0, 32, 1),
    (2, 16, 2, 3, 128, 3, HF, 128, 31, 32, 5),
    (2, 8, 1, 17, 128, 4, BF, 544, 128, 96, 160),
    (7, 2, 2, 1, 64, 4, HF, 416, 33, 64, 129),
    (2, 12, 4, 2, 64, 2, BF, 64, 1, 32, 2),
    (2, 8, 4, 5, 64, 8, HF, 64, 1, 0, 5),
    (40, 8, 2, 1, 128, 4, BF, 1024, 100, 32, 20),
    (70, 4, 1, 1, 128, 4, HF, 640, 0, 0, 1),
    (9, 8, 1, 4, 128, 8, BF, 2048, 5, 32, 9),
    (3, 8, 2, 40, 128, 4, BF, 640, 3, 160, 77),     # own tokens on the tensor-memory kernel, one and two row tiles
    (2, 8, 2, 9, 128, 2, HF, 512, 0, 0, 40),
    (2, 4, 4, 130, 64, 4, HF, 32, 9, 256, 130),
    (1, 6, 1, 43, 128, 8, BF, 0, 0, 128, 128),
]


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_against_64_bits(case, variant):
    B, Hq, Hk, S, D, bits, dtype, pq, pr, oq, orr = case
    q = torch.randn(B, Hq, S, D, device=DEV, generator=_gen(1)).to(dtype)
    if not pq + pr and variant == 2:
        with pytest.raises(ValueError, match="needs a prefix"):
            kivi_shared_prefix_attend(q, make_store(1, Hk, D, bits, 0, 0, dtype, 2)[0], None, 0.1, variant=2)
        return
    check(q, make_store(1, Hk, D, bits, pq, pr, dtype, 2, spare=32), make_store(B, Hk, D, bits, oq, orr, dtype, 3, spare=64), D**-0.5, variant=variant)


@pytest.mark.parametrize("S", [1, 4, 33, 84])
@pytest.mark.parametrize("causal", [True, False])
def test_padding_on_the_left_and_what_it_holds(S, causal):
    B, H, D, n_own = 6, 2, 128, 64 + 20
    start = torch.tensor([0, 1, 31, 33, 70, n_own + 50], dtype=torch.int32, device=DEV)
    q = torch.randn(B, 4, S, D, device=DEV, generator=_gen(4)).to(HF)
    own = make_store(B, H, D, 4, 64, 20, HF, 5)
    check(q, make_store(1, H, D, 4, 96, 3, HF, 6), own, D**-0.5, start=start, causal=causal)
    # the padding slots hold infinities and NaN: value rows, whole key groups, exact rows
    t = own[0]._tensors
    for b, s in enumerate(start.tolist()):
        s = min(s, n_own)
        t[4][b, :, : min(s, 64)] = float("nan")
        t[5][b, :, : min(s, 64)] = float("inf")
        t[1][b, :, : min(s, 64) // 32] = float("nan")
        t[6][b, :, : max(0, s - 64)] = float("inf")
        t[7][b, :, : max(0, s - 64)] = float("nan")
    pads = torch.arange(n_own, device=DEV)[None, :, None] < start[:, None, None]
    od = [x.masked_fill(pads[:, None], 0.0) for x in dense_of(dict(zip(("k_codes", "k_scale", "k_zero", "v_codes", "v_scale", "v_zero", "k_res", "v_res"), t)),
                                                             4, 64, D, B, H)]
    check(q, make_store(1, H, D, 4, 96, 3, HF, 6), (own[0], od), D**-0.5, start=start, causal=causal)


def test_rows_that_see_nothing_give_zeros():
    B, H, D = 3, 2, 128
    none = KiviRows(k_res=torch.empty(1, H, 0, D, dtype=HF, device=DEV), v_res=torch.empty(1, H, 0, D, dtype=HF, device=DEV))
    zero = [torch.zeros(1, H, 0, D, dtype=torch.float64, device=DEV)] * 4
    q = torch.randn(B, 4, 2, D, device=DEV, generator=_gen(7)).to(HF)
    start = torch.tensor([0, 9, 40], dtype=torch.int32, device=DEV)
    check(q, (none, zero), make_store(B, H, D, 4, 0, 10, HF, 8), D**-0.5, start=start)
    out, lse = kivi_shared_prefix_attend(q, none, None, 0.1, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())


def test_prefix_alone_and_wide_scores():
    q = 30 * torch.randn(4, 8, 1, 128, device=DEV, generator=_gen(9)).to(BF)
    for n in ((32, 0), (0, 1), (256, 160)):
        check(q, make_store(1, 2, 128, 4, *n, BF, 10), None, 128**-0.5)


def test_a_later_token_outweighs_all_before_it():
    # the running maximum rises at every group, and at the last token by far
    B, H, D = 40, 1, 128
    k = torch.randn(1, H, 320, D, device=DEV, generator=_gen(11)) * 0.1
    q = torch.randn(B, 1, 1, D, device=DEV, generator=_gen(12))
    ramp = torch.linspace(0, 3, 320, device=DEV)[None, None, :, None]
    k = (k + ramp * q.mean((0, 1))[None, None] * 6).half()
    v = torch.randn(1, H, 320, D, device=DEV, generator=_gen(13)).half()
    t = {}
    t["k_codes"], t["k_scale"], t["k_zero"] = kernels.kivi_quantize(k[:, :, :288], -2, 32, 4)
    t["v_codes"], t["v_scale"], t["v_zero"] = kernels.kivi_quantize(v[:, :, :288], -1, 32, 4)
    t["k_res"], t["v_res"] = k[:, :, 288:].contiguous(), v[:, :, 288:].contiguous()
    pre = (KiviRows(**t), dense_of(t, 4, 288, D, 1, H))
    for variant in (1, 2):
        check(q.half(), pre, None, 0.5, variant=variant)


@pytest.mark.parametrize("variant", [1, 2])
def test_long_prefix_and_many_rows(variant):
    q = torch.randn(24, 8, 2, 128, device=DEV, generator=_gen(14)).to(BF)
    check(q, make_store(1, 2, 128, 4, 8192, 77, BF, 15), make_store(24, 2, 128, 4, 64, 40, BF, 16), 128**-0.5, variant=variant)


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("splits", [1, 2, 5, 17, 64])
def test_every_number_of_splits(splits, variant):
    q = torch.randn(12, 8, 1, 128, device=DEV, generator=_gen(17)).to(HF)
    check(q, make_store(1, 2, 128, 4, 2080, 9, HF, 18), make_store(12, 2, 128, 4, 32, 1, HF, 19), 128**-0.5, n_splits=splits, variant=variant)


def test_strided_queries_given_output_other_stream_and_repeat():
    B = 9
    q = torch.randn(B, 1, 8, 128, device=DEV, generator=_gen(20)).to(HF).transpose(1, 2)
    pre, own = make_store(1, 2, 128, 4, 256, 9, HF, 21), make_store(B, 2, 128, 4, 32, 8, HF, 22)
    want = check(q, pre, own, 0.1)
    out = torch.full((B, 8, 1, 128), 7.0, dtype=HF, device=DEV)
    assert kivi_shared_prefix_attend(q, pre[0], own[0], 0.1, out=out) is out and torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(4):  # two streams at once
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(kivi_shared_prefix_attend(q, pre[0], own[0], 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    with pytest.raises(ValueError, match="16-byte aligned"):
        kivi_shared_prefix_attend(q, pre[0], own[0], 0.1, out=torch.empty(B * 8 * 128 + 1, dtype=HF, device=DEV)[1:].view(B, 8, 1, 128))


def test_two_captured_graphs_replayed_at_once():
    pre, own = make_store(1, 2, 128, 4, 1024, 9, HF, 23), make_store(20, 2, 128, 4, 32, 8, HF, 24)
    qs = [torch.randn(20, 8, 1, 128, device=DEV, generator=_gen(25 + i)).to(HF) for i in range(2)]
    want = [kivi_shared_prefix_attend(q, pre[0], own[0], 0.1) for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kivi_shared_prefix_attend(q, pre[0], own[0], 0.1))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_one_request_equals_the_packed_decode_attention():
    """A batch of one behind a prefix of its own is the plain decode attention over the same tokens."""
    from veloxquant_mlx_b200.cache import KVCacheConfig, KVCacheFactory
    from veloxquant_mlx_b200.shared_prefix import SharedPrefixKIVICache

    cfg = KVCacheConfig(method="kivi", head_dim=128, bit_width_inlier=4, residual_length=32, fused_sdpa_memory_bound=True)
    one = KVCacheFactory.create(cfg)
    g = _gen(30)
    k, v = (torch.randn(1, 2, 320, 128, device=DEV, generator=g).half() for _ in range(2))
    one.update_and_fetch(k, v)
    fork = SharedPrefixKIVICache(one, 1)
    k1, v1, q = (torch.randn(1, h, 1, 128, device=DEV, generator=g).half() for h in (2, 2, 8))
    fork.update_and_fetch(k1, v1)
    a = fork.fused_sdpa(q, 0.09)
    one.update_and_fetch(k1, v1)  # the prefix goes on; the fork keeps the 320 tokens it had
    b = one.fused_sdpa(q, 0.09)
    # both within the framework's attention tolerance of the same softmax (the last group may be packed in one of them only)
    assert one._n_quantized == 288 and (a.float() - b.float()).abs().max() < 4e-3
    assert torch.equal(fork.fused_sdpa(q, 0.09), a) and fork.offset == 321 and fork.prefix_length == 320
    one.trim(5)
    with pytest.raises(RuntimeError, match="trimmed"):
        fork.fused_sdpa(q, 0.09)


@pytest.mark.parametrize("pad", [None, [0, 3, 17, 40, 2]])
def test_decoding_a_forked_batch_step_by_step(pad):
    """Prompt, fork, the requests' own prompts, then single tokens: rotary append and attention, as a serving loop runs them."""
    from veloxquant_mlx_b200.cache import KVCacheConfig, KVCacheFactory
    from veloxquant_mlx_b200.rotary import RotaryEmbedding
    from veloxquant_mlx_b200.shared_prefix import SharedPrefixKIVICache

    B, H, Hk, D = 5, 8, 2, 128
    cfg = KVCacheConfig(method="kivi", head_dim=D, bit_width_inlier=4, residual_length=64, fused_sdpa_memory_bound=True)
    rope = RotaryEmbedding(D, base=500000.0)
    g = _gen(40)
    rand = lambda b, h, s: torch.randn(b, h, s, D, device=DEV, generator=g).to(BF)  # noqa: E731
    first = KVCacheFactory.create(cfg)
    first.update_rotary(rand(1, H, 200), rand(1, Hk, 200), rand(1, Hk, 200), rope)
    cache = SharedPrefixKIVICache(first, B, own_start=pad)
    plain = KVCacheFactory.create(cfg)  # the own tokens alone, rotated by hand
    start = torch.tensor(pad or [0] * B, device=DEV)
    n = 0
    pre_dense = dense_of(dict(zip(("k_codes", "k_scale", "k_zero", "v_codes", "v_scale", "v_zero"), cache._prefix_rows._tensors[:6]))
                         | {"k_res": cache._prefix_rows._tensors[6], "v_res": cache._prefix_rows._tensors[7]}, 4, cache._prefix_rows.n_quant, D, 1, Hk)
    for S in [45, 1, 1, 1] + [1] * 80:
        q, k, v = rand(B, H, S), rand(B, Hk, S), rand(B, Hk, S)
        q1, ks, vs = cache.update_rotary(q, k, v, rope)
        assert ks.shape == (B, Hk, 0, D) and vs.shape == (B, Hk, 0, D)
        pos = 200 + n + torch.arange(S, device=DEV)[None] - start[:, None]
        q2, k2 = rope(q, k, pos)
        assert torch.equal(q1, q2)
        plain.update_and_fetch(k2, v)
        n += S
        assert cache.offset == 200 + n and len(cache) == 200 + n
        out = cache.fused_sdpa(q1, D**-0.5)
        if S > 1 or n % 20 == 0:
            st = plain.state
            own_dense = dense_of(dict(zip(("k_codes", "k_scale", "k_zero", "v_codes", "v_scale", "v_zero", "k_res", "v_res"), st[:8])), 4, plain._n_quantized, D, B, Hk)
            want, _, tol, _ = reference(q2, pre_dense, own_dense, D**-0.5, True, start if pad else None)
            tol = tol + 2.0**-9 * 2 * (want.abs() + tol)  # (bfloat16: eps / 2 = 2^-8)
            assert bool(((out.double() - want).abs() <= tol).all())
    assert cache.trim(1000) == n and cache.offset == 200
    alone = cache.fused_sdpa(q1, D**-0.5, causal=False)
    assert torch.equal(alone, kivi_shared_prefix_attend(q1, cache._prefix_rows, None, D**-0.5))
    cache.reset()
    assert cache.offset == 200 and cache.nbytes >= 0
    cache.check_status()


def test_a_fork_of_a_transformers_cache_continues_a_prompt():
    pytest.importorskip("transformers")
    from transformers import LlamaConfig, LlamaForCausalLM

    from veloxquant_mlx_b200.cache import KVCacheConfig
    from veloxquant_mlx_b200.integration import fork_hf_cache, make_hf_cache, patch_hf_for_fused_sdpa

    torch.manual_seed(0)
    model = LlamaForCausalLM(LlamaConfig(hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                         vocab_size=64, max_position_embeddings=512)).to(DEV, torch.float16).eval()
    patch_hf_for_fused_sdpa(model)
    cfg = KVCacheConfig(method="kivi", head_dim=64, bit_width_inlier=8, residual_length=32, fused_sdpa_memory_bound=True)
    prompt = torch.randint(0, 64, (1, 90), device=DEV)
    asks = torch.randint(0, 64, (3, 4), device=DEV)
    with torch.no_grad():
        cache = make_hf_cache(model, cfg)
        model(prompt, past_key_values=cache, use_cache=True)
        fork = fork_hf_cache(cache, 3)
        together = [model(asks[:, i : i + 1], past_key_values=fork, use_cache=True).logits[:, -1] for i in range(4)]
        for b in range(3):  # each request alone over its own copy of the prompt
            alone = make_hf_cache(model, cfg)
            model(prompt, past_key_values=alone, use_cache=True)
            for i in range(4):
                got = model(asks[b : b + 1, i : i + 1], past_key_values=alone, use_cache=True).logits[0, -1]
                assert fork.get_seq_length() == 94
                # 8-bit codes of the same tokens; the alone cache packs a group that the fork still holds exactly
                assert (got.float() - together[i][b].float()).abs().max() < 0.05 * got.float().abs().max() + 0.05


def test_exact_rows_past_32_bits():
    rows, D = (1 << 24) + 64, 128  # 2.1e9 elements a slab; the second request's begin behind it
    k = torch.empty(2, 1, rows, D, dtype=HF, device=DEV)
    v = torch.empty(2, 1, rows, D, dtype=HF, device=DEV)
    small = [torch.randn(2, 1, 40, D, device=DEV, generator=_gen(50 + i)).half() for i in range(2)]
    k[:, :, -50:-10], v[:, :, -50:-10] = small
    own = KiviRows(k_res=k, v_res=v, n_res=40, res_offset=rows - 50)
    dense = []
    for t in small:
        dense += [t.double(), torch.zeros_like(t, dtype=torch.float64)]
    pre = make_store(1, 1, D, 4, 64, 3, HF, 52)
    for S in (1, 36):
        q = torch.randn(2, 2, S, D, device=DEV, generator=_gen(53)).half()
        check(q, pre, (own, dense), D**-0.5)
        check(q, pre, (own, dense), D**-0.5, variant=2)


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_constant_groups_and_large_offsets(variant, dtype):
    """Groups without spread (scale at its floor) and keys far from zero: code * scale + zero must not lose the zero."""
    B, H, D = 40, 1, 128
    k = (100 + torch.randn(1, H, 256, D, device=DEV, generator=_gen(60))).to(dtype)
    k[:, :, :32] = 3.0
    v = (-50 + torch.randn(1, H, 256, D, device=DEV, generator=_gen(61))).to(dtype)
    v[:, :, 40:50] = 7.0
    t = {}
    t["k_codes"], t["k_scale"], t["k_zero"] = kernels.kivi_quantize(k, -2, 32, 4)
    t["v_codes"], t["v_scale"], t["v_zero"] = kernels.kivi_quantize(v, -1, 32, 4)
    q = 0.05 * torch.randn(B, 1, 1, D, device=DEV, generator=_gen(62)).to(dtype)
    check(q, (KiviRows(**t), dense_of(t, 4, 256, D, 1, H)), None, 0.1, variant=variant)


def test_a_nan_that_is_seen_stays_in_its_rows():
    q = torch.randn(40, 2, 1, 128, device=DEV, generator=_gen(70)).half()
    q[3, 1] = float("nan")
    pre, own = make_store(1, 1, 128, 4, 512, 9, HF, 71), make_store(40, 1, 128, 4, 32, 5, HF, 72)
    own[0]._tensors[7][9, 0, 2, 5] = float("nan")  # a value of request 9
    for variant in (1, 2):
        out = kivi_shared_prefix_attend(q, pre[0], own[0], 0.1, variant=variant)
        bad = out.isnan()
        assert bool(bad[3, 1].all()) and bool(bad[9, :, :, 5].all())
        bad[3, 1] = False
        bad[9, :, :, 5] = False
        assert not bool(bad.any())


def test_a_wait_that_runs_out_is_reported_once():
    """The bounded waits' error path: a barrier that nothing arms, waited for behind the work (which stays right)."""
    from veloxquant_mlx_b200 import VQLibraryError

    q = torch.randn(40, 2, 1, 128, device=DEV, generator=_gen(80)).half()
    pre = make_store(1, 1, 128, 4, 512, 9, HF, 81)
    want = kivi_shared_prefix_attend(q, pre[0], None, 0.1, variant=2)
    kernels.attend_status()
    assert kernels.tune("shared_wait_test", 1) == 0
    out = kivi_shared_prefix_attend(q, pre[0], None, 0.1, variant=2)
    with pytest.raises(VQLibraryError, match="TIMEOUT.*shared"):
        kernels.attend_status()
    kernels.attend_status()
    assert torch.equal(out, want) and kernels.tune("shared_wait_test", 0) == 0


@pytest.mark.parametrize("B,H,G,n_pre,n_own,Sq", [(3, 8, 8, 96, 5, 4), (40, 2, 2, 4096, 1, 1), (9, 1, 16, 20000, 40, 1), (2, 4, 4, 300, 290, 40)])
def test_parts_that_end_in_either_order(B, H, G, n_pre, n_own, Sq):
    """The own tokens' kernel runs beside the prefix's and may be done long before or long after it; one and two row
    tiles, one token tile for two streams, own tokens on tcgen05 too. Twenty calls in a row give the same bits."""
    pre, _ = make_store(1, H, 128, 4, n_pre // 32 * 32, n_pre % 32, BF, 90)
    own, _ = make_store(B, H, 128, 4, n_own // 32 * 32, n_own % 32, BF, 91)
    q = torch.randn(B, H * G, Sq, 128, device=DEV, generator=_gen(92)).to(BF)
    first = kivi_shared_prefix_attend(q, pre, own, 0.088, variant=2)
    warp_tiles = kivi_shared_prefix_attend(q, pre, own, 0.088, variant=1)
    # (two roundings of the weights and of the output apart, on values of at most about 4: 4 (2 * 2^-11 + 2 * 2^-8) < 0.04)
    assert float((first.float() - warp_tiles.float()).abs().max()) < 0.04
    for _ in range(20):
        assert torch.equal(kivi_shared_prefix_attend(q, pre, own, 0.088, variant=2), first)
    kernels.attend_status()
