"""Cases and plain forms of the rotary-position operators and of the attention of a batch that shares a prefix.

``run`` makes one pass: with ``own`` through the package's public entry points, without it through
elementary torch operations in 32 bits (angles in 64), rounded once at the end. ``exact`` is the
definition of the same outputs in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
GROUP = 32  # tokens of a key group, channels of a value group
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    def rope(name, kind, B, S, Hq, Hk, D, rdim, layout, dtype, far, scaled, strided):
        return dict(name=name, op="rope", kind=kind, B=B, S=S, Hq=Hq, Hk=Hk, D=D, rdim=rdim, layout=layout, dtype=dtype, far=far,
                    scaled=scaled, strided=strided)

    def attend(name, B, Sq, Hq, Hk, D, bits, dtype, pre_q, pre_r, own_q, own_r, pad):
        return dict(name=name, op="attend", B=B, Sq=Sq, Hq=Hq, Hk=Hk, D=D, bits=bits, dtype=dtype, pre_q=pre_q, pre_r=pre_r,
                    own_q=own_q, own_r=own_r, pad=pad)

    return [
        # one request's next token: queries and keys of one position, where only latency counts
        rope("rope-decode-one", "apply", 1, 1, 32, 8, 128, 128, "half", "bf16", 4096, False, False),
        # a decode batch whose requests stand at different positions of a context scaled to a million tokens
        rope("rope-decode-far", "apply", 64, 1, 40, 8, 128, 128, "half", "f16", 1 << 20, True, False),
        # a prompt of odd length, heads still in the projection's [B, S, H, D] order
        rope("rope-prompt-strided", "apply", 4, 8191, 32, 8, 128, 128, "half", "bf16", 16384, False, True),
        # a training step of an interleaved layout that rotates part of the head: outputs and gradients
        rope("rope-train-partial", "train", 2, 2048, 16, 16, 80, 32, "interleaved", "f32", 4096, False, False),
        # the decode step of a cache: rotate, and put the rotated keys and the values behind the unquantized window
        rope("rope-append-batch", "append", 64, 1, 32, 8, 128, 128, "half", "bf16", 32768, False, False),
        # a few requests right behind a short system prompt
        attend("prefix-short", 4, 1, 32, 8, 128, 4, "f16", 256, 64, 0, 40, 0),
        # a serving batch behind a prompt of 8K tokens
        attend("prefix-8k", 16, 1, 32, 8, 128, 4, "bf16", 8064, 128, 96, 140, 0),
        # the large serving batch: 64 requests, 32K shared tokens, a few hundred of their own
        attend("prefix-32k", 64, 1, 32, 8, 128, 4, "bf16", 32640, 128, 512, 150, 0),
        # 2-bit codes, an odd batch, five heads to a kv head, own tokens padded on the left to one length
        attend("prefix-padded-2bit", 23, 1, 40, 8, 128, 2, "f16", 12288, 77, 256, 130, 300),
        # four drafted tokens a request are verified at once, 8-bit codes
        attend("prefix-draft", 8, 4, 32, 8, 128, 8, "bf16", 16384, 0, 32, 133, 0),
        # the requests' own prompts are run behind the shared one: many query rows
        attend("prefix-prompts", 8, 256, 32, 8, 128, 4, "bf16", 8064, 128, 224, 160, 100),
        # a small head without grouped heads
        attend("prefix-d64", 96, 1, 8, 8, 64, 4, "f16", 4096, 33, 64, 129, 0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.4:
        kind = rng.choice(["apply", "apply", "train", "append"])
        dtype = rng.choice(["bf16", "f16", "f32"])
        D = rng.choice([64, 80, 96, 128, 128, 256])
        rdim = rng.choice([D, D, D // 2, 32])
        Hk = rng.choice([1, 4, 8, 16])
        Hq = Hk * rng.choice([1, 2, 4, 5])
        B = _log_int(rng, 1, 96)
        most = max(1, (1 << 25) // (B * (Hq + Hk) * D))  # elements of queries and keys
        S = 1 if rng.random() < 0.3 or most < 2 else _log_int(rng, 1, min(16384, most))
        if kind == "append":
            S = min(S, 64)
        return dict(op="rope", kind=kind, B=B, S=S, Hq=Hq, Hk=Hk, D=D, rdim=rdim, layout=rng.choice(["half", "interleaved"]), dtype=dtype,
                    far=_log_int(rng, max(S, 64), 1 << 20), scaled=rng.random() < 0.4, strided=rng.random() < 0.5)
    Hk = rng.choice([1, 4, 8])
    G = rng.choice([1, 2, 4, 5, 8])
    D = rng.choice([64, 128, 128])
    B = _log_int(rng, 1, 96)
    pre_q = GROUP * _log_int(rng, 1, 1020) if rng.random() < 0.95 else 0
    pre_r = rng.randint(0 if pre_q else 1, 160)
    Sq = 1 if rng.random() < 0.6 else _log_int(rng, 2, 256)
    most = (8 * 256 * 32 * 8192) // max(1, B * Hk * G * (pre_q + pre_r))  # query rows x shared tokens
    Sq = max(1, min(Sq, most))
    own_q = GROUP * rng.randint(0, 24)
    own_r = rng.randint(max(1, Sq - own_q), max(160, Sq))
    return dict(op="attend", B=B, Sq=Sq, Hq=Hk * G, Hk=Hk, D=D, bits=rng.choice([2, 4, 4, 8]), dtype=rng.choice(["bf16", "f16"]),
                pre_q=pre_q, pre_r=pre_r, own_q=own_q, own_r=own_r, pad=rng.choice([0, 0, own_q + own_r - 1]))


# ---------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------
def _frequencies(case):
    """Angle per position of each pair, in 64 bits, and the factor on sine and cosine: plain, or with the low
    frequencies stretched for a long context (a ramp between two wavelengths)."""
    half = case["rdim"] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64) * 2.0 / case["rdim"])
    if not case["scaled"]:
        return f, 1.0
    wave, old, factor, lo, hi = 2 * math.pi / f, 8192.0, 8.0, 1.0, 4.0
    ramp = ((old / wave - lo) / (hi - lo)).clamp(0, 1)
    return f * (ramp + (1 - ramp) / factor), 0.1 * math.log(factor) + 1.0


def _prepare_rope(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    B, S, D, dt = case["B"], case["S"], case["D"], DTYPES[case["dtype"]]

    def rand(H, strided):
        if strided:
            return torch.randn(B, S, H, D, generator=g, device=DEV, dtype=torch.float32).to(dt).transpose(1, 2)
        return torch.randn(B, H, S, D, generator=g, device=DEV, dtype=torch.float32).to(dt)

    freq, factor = _frequencies(case)
    start = torch.randint(0, case["far"] - S + 1, (B, 1), generator=g, device=DEV)
    s = {"case": case, "q": rand(case["Hq"], case["strided"]), "k": rand(case["Hk"], case["strided"]), "freq": freq.to(DEV), "factor": factor,
         "pos": start + torch.arange(S, device=DEV)}
    if case["kind"] == "train":
        s["gq"], s["gk"] = rand(case["Hq"], False), rand(case["Hk"], False)
        s["q"].requires_grad_(True)
        s["k"].requires_grad_(True)
    if case["kind"] == "append":
        # the window of unquantized rows: the new ones go behind row `at`, the rows after them stay
        s["v"] = rand(case["Hk"], case["strided"])
        rows = 2 * (128 + GROUP) + GROUP
        s["at"] = int(torch.randint(0, rows - S + 1, (1,), generator=torch.Generator().manual_seed(seed)))
        s["k_res"] = torch.randn(B, case["Hk"], rows, D, generator=g, device=DEV, dtype=torch.float32).to(dt)
        s["v_res"] = torch.randn(B, case["Hk"], rows, D, generator=g, device=DEV, dtype=torch.float32).to(dt)
    if own:
        from veloxquant_mlx_b200 import rotary

        s["rope"] = rotary.RotaryEmbedding(D, rotary_dim=case["rdim"], layout=case["layout"], inv_freq=s["freq"], attention_factor=factor)
    return s


def _angles(s, wide):
    turn = s["pos"].double()[:, None, :, None] * s["freq"]  # [B, 1, S, pairs], 64 bits: positions go to a million
    c, n = torch.cos(turn) * s["factor"], torch.sin(turn) * s["factor"]
    return (c, n) if wide else (c.float(), n.float())


def _pairs(x, layout, rdim):
    x = x[..., :rdim]
    return (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else (x[..., : rdim // 2], x[..., rdim // 2 :])


def _turned(x, c, n, layout, rdim):
    """Rotated in 32 bits (64 where the angles are), rounded once."""
    dt = x.dtype if c.dtype == torch.float32 else torch.float64
    w = x.to(c.dtype)
    a, b = _pairs(w, layout, rdim)
    ya, yb = a * c - b * n, b * c + a * n
    y = torch.stack((ya, yb), -1).flatten(-2) if layout == "interleaved" else torch.cat((ya, yb), -1)
    return torch.cat((y, w[..., rdim:]), -1).to(dt) if rdim < x.shape[-1] else y.to(dt)


def _run_rope(s):
    case = s["case"]
    q, k = s["q"], s["k"]
    if own:
        rope = s["rope"]
        if case["kind"] == "append":
            return [rope.append(q, k, s["v"], s["k_res"], s["v_res"], s["at"], s["pos"]), s["k_res"], s["v_res"]]
        yq, yk = rope(q, k, s["pos"])
        if case["kind"] == "train":
            return [yq, yk, *torch.autograd.grad((yq, yk), (q, k), (s["gq"], s["gk"]))]
        return [yq, yk]
    lay, r = case["layout"], case["rdim"]
    with torch.no_grad():
        c, n = _angles(s, False)
        yq, yk = _turned(q, c, n, lay, r), _turned(k, c, n, lay, r)
        if case["kind"] == "train":  # the gradient turns back
            return [yq, yk, _turned(s["gq"], c, -n, lay, r), _turned(s["gk"], c, -n, lay, r)]
        if case["kind"] == "append":
            at = s["at"]
            s["k_res"][:, :, at : at + case["S"]] = yk
            s["v_res"][:, :, at : at + case["S"]] = s["v"]
            return [yq, s["k_res"], s["v_res"]]
    return [yq, yk]


def _exact_rope(s):
    """Each pair as a complex number times factor * exp(i * position * frequency)."""
    case, r = s["case"], s["case"]["rdim"]
    turn = torch.polar(torch.full_like(s["freq"], s["factor"]).expand(*s["pos"].shape, -1).contiguous(), s["pos"].double()[..., None] * s["freq"])
    turn = turn[:, None]

    def times(x, t):
        x = x.detach().double()
        if case["layout"] == "interleaved":
            z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * t
            y = torch.view_as_real(z).reshape(*x.shape[:-1], r)
        else:
            z = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2 : r].contiguous()) * t
            y = torch.cat((z.real, z.imag), -1)
        return torch.cat((y, x[..., r:]), -1)

    out = [times(s["q"], turn), times(s["k"], turn)]
    if case["kind"] == "train":
        out += [times(s["gq"], turn.conj()), times(s["gk"], turn.conj())]
    if case["kind"] == "append":
        at, k_res, v_res = s["at"], s["k_res"].double(), s["v_res"].double()
        k_res[:, :, at : at + case["S"]] = out[1]
        v_res[:, :, at : at + case["S"]] = s["v"].double()
        out = [out[0], k_res, v_res]
    return out


def _work_rope(case):
    rows = case["B"] * case["S"]
    el = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    n = rows * (case["Hq"] + case["Hk"]) * case["D"]
    values = rows * case["Hk"] * case["D"] if case["kind"] == "append" else 0
    twice = 2 if case["kind"] == "train" else 1
    return {"bytes": twice * 2 * el * (n + values) + 8 * rows, "flops": twice * 3 * n * case["rdim"] / case["D"]}


# ---------------------------------------------------------------------------------------------
# attention of a batch that shares a prefix, over packed codes
# ---------------------------------------------------------------------------------------------
def _packed(x, axis, bits):
    """Codes (packed along the channels, lowest bits first), scales and zeros of groups of 32 along `axis`."""
    B, H, S, D = x.shape
    w = x.float()
    w = w.reshape(B, H, S // GROUP, GROUP, D) if axis == 2 else w.reshape(B, H, S, D // GROUP, GROUP)
    at = 3 if axis == 2 else 4
    lo, hi = w.amin(at, keepdim=True), w.amax(at, keepdim=True)
    scale = ((hi - lo) / (2**bits - 1)).clamp_min(1e-8)
    code = ((w - lo) / scale).round().clamp(0, 2**bits - 1).reshape(B, H, S, D * bits // 8, 8 // bits).int()
    code = (code << (bits * torch.arange(8 // bits, device=x.device, dtype=torch.int32))).sum(-1).to(torch.uint8)
    return code, scale.squeeze(at), lo.squeeze(at)


def _prepare_attend(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    B, H, D, dt, bits = case["B"], case["Hk"], case["D"], DTYPES[case["dtype"]], case["bits"]
    loud = 1.0 + 4.0 * (torch.rand(1, H, 1, D, generator=g, device=DEV) < 0.04)  # key channels that stand out

    def store(b, n_q, n_r):
        k = (torch.randn(b, H, n_q + n_r, D, generator=g, device=DEV) * loud).to(dt)
        v = torch.randn(b, H, n_q + n_r, D, generator=g, device=DEV).to(dt)
        kc, ks, kz = _packed(k[:, :, :n_q], 2, bits)
        vc, vs, vz = _packed(v[:, :, :n_q], 3, bits)
        return {"k_codes": kc, "k_scale": ks, "k_zero": kz, "v_codes": vc, "v_scale": vs, "v_zero": vz, "k_res": k[:, :, n_q:].contiguous(),
                "v_res": v[:, :, n_q:].contiguous()}

    s = {"case": case, "scale": D**-0.5, "q": torch.randn(B, case["Hq"], case["Sq"], D, generator=g, device=DEV).to(dt),
         "prefix": store(1, case["pre_q"], case["pre_r"]), "mine": store(B, case["own_q"], case["own_r"]), "start": None}
    if case["pad"]:  # the first own slot that is a token of request b
        s["start"] = torch.tensor([b * 37 % (case["pad"] + 1) for b in range(B)], dtype=torch.int32, device=DEV)
    if own:
        from veloxquant_mlx_b200 import kernels

        s["rows"] = [kernels.KiviRows(**s[name], group_size=GROUP, store_bits=bits) for name in ("prefix", "mine")]
    return s


def _values_of(st, bits, name, wide):
    """Keys or values of a store as numbers, [B, H, tokens, D]: code * scale + zero, then the exact rows."""
    codes, scale, zero, exact = (st[name + part].to(wide) if part != "_codes" else st[name + part] for part in ("_codes", "_scale", "_zero", "_res"))
    B, H, S, _ = codes.shape
    D = exact.shape[3]
    c = ((codes[..., None].int() >> (bits * torch.arange(8 // bits, device=codes.device, dtype=torch.int32))) & (2**bits - 1)).reshape(B, H, S, D).to(wide)
    if name == "k":
        c = (c.reshape(B, H, S // GROUP, GROUP, D) * scale[:, :, :, None] + zero[:, :, :, None]).reshape(B, H, S, D)
    else:
        c = (c.reshape(B, H, S, D // GROUP, GROUP) * scale[..., None] + zero[..., None]).reshape(B, H, S, D)
    return torch.cat((c, exact), 2)


def _visible(s):
    """[B, 1, Sq, own tokens]: own slot t of request b is seen by query row r where start[b] <= t <= tokens - Sq + r."""
    case = s["case"]
    n = case["own_q"] + case["own_r"]
    t, r = torch.arange(n, device=DEV), torch.arange(case["Sq"], device=DEV)
    seen = (t <= (n - case["Sq"] + r)[:, None])[None, None]
    return seen if s["start"] is None else seen & (t >= s["start"][:, None])[:, None, None]


def _run_attend(s):
    case, q = s["case"], s["q"]
    if own:
        from veloxquant_mlx_b200 import kernels

        return kernels.kivi_shared_prefix_attend(q, *s["rows"], s["scale"], causal=True, own_start=s["start"])
    B, H, G, Sq, D, bits = case["B"], case["Hk"], case["Hq"] // case["Hk"], case["Sq"], case["D"], case["bits"]
    w = q.float() * s["scale"]
    k, v = (_values_of(s["prefix"], bits, name, torch.float32)[0] for name in "kv")  # [H, shared, D]
    ko, vo = (_values_of(s["mine"], bits, name, torch.float32) for name in "kv")  # [B, H, own, D]
    n = k.shape[1]
    shared = (w.reshape(B, H, G * Sq, D).transpose(0, 1).reshape(H, -1, D) @ k.transpose(1, 2)).reshape(H, B, G * Sq, n).transpose(0, 1)
    mine = (w.reshape(B, H, G * Sq, D) @ ko.transpose(2, 3)).reshape(B, H * G, Sq, -1)
    mine = mine.masked_fill(~_visible(s), -math.inf).reshape(B, H, G * Sq, -1)
    top = torch.maximum(shared.amax(3, keepdim=True), mine.amax(3, keepdim=True))
    shared, mine = torch.exp(shared - top), torch.exp(mine - top)
    total = shared.sum(3, keepdim=True) + mine.sum(3, keepdim=True)
    out = (shared.transpose(0, 1).reshape(H, -1, n) @ v).reshape(H, B, G * Sq, D).transpose(0, 1) + mine @ vo
    return (out / total).reshape(q.shape).to(q.dtype)


def _wide(st, bits, name):
    """Keys or values of one kv head's store in 64 bits, [B, tokens, D], code by code from its byte."""
    codes, exact_rows = st[name + "_codes"][:, 0], st[name + "_res"][:, 0].double()
    byte = codes.double().repeat_interleave(8 // bits, 2)
    place = torch.arange(exact_rows.shape[2], device=DEV) % (8 // bits)
    code = torch.remainder(torch.floor(byte / 2.0 ** (bits * place)), 2.0**bits)
    along = 1 if name == "k" else 2  # a key group is 32 tokens of a channel, a value group 32 channels of a token
    scale, zero = (st[name + part][:, 0].double().repeat_interleave(GROUP, along) for part in ("_scale", "_zero"))
    return torch.cat((code * scale + zero, exact_rows), 1)


def _softmax_64(q, k, v, ko, vo, first):
    """softmax(q k / sqrt(D)) v over the shared tokens and request's own ones; q [m, G, Sq, D], `first` [m]."""
    n, Sq, n_own = k.shape[0], q.shape[2], ko.shape[1]
    score = torch.cat((torch.einsum("bgsd,td->bgst", q, k), torch.einsum("bgsd,btd->bgst", q, ko)), 3) / math.sqrt(q.shape[3])
    slot = torch.arange(n_own, device=DEV)
    last = n_own - Sq + torch.arange(Sq, device=DEV)
    hidden = (slot < first[:, None, None]) | (slot > last[:, None])
    score[..., n:] = torch.where(hidden[:, None], -math.inf, score[..., n:])
    p = torch.softmax(score, 3)
    return torch.einsum("bgst,td->bgsd", p[..., :n], v) + torch.einsum("bgst,btd->bgsd", p[..., n:], vo)


def _work_attend(case):
    B, H, D, Sq, bits = case["B"], case["Hk"], case["D"], case["Sq"], case["bits"]
    # a packed token: key and value codes, its share of the key group's scales and zeros, its own value scales and zeros
    packed, exact = 2 * D * bits // 8 + 8 * D // GROUP + 8 * D // GROUP, 2 * D * 2
    pads = [b * 37 % (case["pad"] + 1) for b in range(B)]
    n_own = case["own_q"] + case["own_r"]
    stored = H * (case["pre_q"] * packed + case["pre_r"] * exact)
    seen = 0
    for p in pads:
        stored += H * (max(0, case["own_q"] - p) * packed + min(case["own_r"], n_own - p) * exact)
        seen += sum(max(0, n_own - Sq + r + 1 - p) for r in range(Sq))
    scores = case["Hq"] * (B * Sq * (case["pre_q"] + case["pre_r"]) + seen)
    return {"bytes": stored + 2 * 2 * B * case["Hq"] * Sq * D, "flops": 4 * D * scores}


# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    return _prepare_rope(case, seed) if case["op"] == "rope" else _prepare_attend(case, seed)


def run(state):
    return _run_rope(state) if state["case"]["op"] == "rope" else _run_attend(state)


def work(case):
    return _work_rope(case) if case["op"] == "rope" else _work_attend(case)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s)
    G, B, bits = case["Hq"] // case["Hk"], case["B"], case["bits"]
    first = torch.zeros(B, dtype=torch.int64, device=DEV) if s["start"] is None else s["start"].long()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    # one kv head, and at most 2^28 scores, at a time
    some = max(1, min(B, (1 << 28) // (G * case["Sq"] * sum(case[n] for n in ("pre_q", "pre_r", "own_q", "own_r")))))
    for h in range(case["Hk"]):
        prefix, mine = ({name: t[:, h : h + 1] for name, t in s[of].items()} for of in ("prefix", "mine"))
        k, v = _wide(prefix, bits, "k")[0], _wide(prefix, bits, "v")[0]
        ko, vo = _wide(mine, bits, "k"), _wide(mine, bits, "v")
        for b in range(0, B, some):
            e = slice(b, b + some)
            out[e, h * G : (h + 1) * G] = _softmax_64(s["q"][e, h * G : (h + 1) * G].double(), k, v, ko[e], vo[e], first[e])
    return out
