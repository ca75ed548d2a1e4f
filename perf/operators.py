"""Cases, plain forms and 64-bit values of the operators of a decode step around the quantized KV cache.

Three operators run together in one step of a layer:

* rotary positions applied to the new query and key rows (`apply_rotary`);
* products of a few activation rows with a 4-bit group-scaled weight
  (`PackedWeight.matvec`), the step's projections;
* attention of every sequence of a batch over one shared prompt prefix, merged
  with the attention state of its own tokens (`prefix_attention`).

A case is a dict of plain values.  `own` chooses the framework's kernels; else
`run` computes the same from elementary torch operations in fp32.
"""

import importlib
import math

import numpy as np
import torch

own = False

_PKG = "care-kv-sparse-residual-correction-for-low-bit-kv-cache-quantization_b200"
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _ck():
    return importlib.import_module(_PKG)


# ── cases ─────────────────────────────────────────────────────────────────
def _rotary(batch, tokens, heads, kv_heads, dim, rotary_dim, layout, scaling, start, inverse, dtype):
    return dict(op="rotary", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                rotary_dim=rotary_dim, layout=layout, scaling=scaling, start=start, inverse=inverse, dtype=dtype)


def _w4(rows, k, n, group, dtype):
    return dict(op="w4", rows=rows, k=k, n=n, group=group, dtype=dtype)


def _prefix(rows, heads, kv_heads, dim, tokens, ragged, tail, dtype):
    return dict(op="prefix", rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, tokens=tokens, ragged=ragged,
                tail=tail, dtype=dtype)


def listed():
    return [
        # one new token of one sequence, TinyLlama shape: only latency counts
        dict(_rotary(1, 1, 32, 4, 64, 64, "half", "none", 511, False, "f16"), name="rotary one token"),
        # a prompt of 4096 tokens for 4 sequences (Mistral-7B heads), positions stretched past the trained length
        dict(_rotary(4, 4096, 32, 8, 128, 128, "half", "yarn", 0, False, "bf16"), name="rotary prompt yarn"),
        # the backward pass (inverse rotation) of an odd-length batch, interleaved pairs on part of the head, fp32
        dict(_rotary(3, 1021, 40, 40, 128, 96, "interleaved", "linear", 7, True, "f32"),
             name="rotary backward partial"),
        # output projection of one token (Llama-2-7B hidden size)
        dict(_w4(1, 4096, 4096, 32, "f16"), name="w4 1x4096x4096"),
        # FFN up projection of one token (Llama-2-13B shape)
        dict(_w4(1, 5120, 13824, 64, "bf16"), name="w4 1x5120x13824"),
        # FFN up projection of a batch of 16 sequences (Mistral-7B shape)
        dict(_w4(16, 4096, 14336, 32, "bf16"), name="w4 16x4096x14336"),
        # FFN down projection of a batch of 64 (Llama-2-13B shape)
        dict(_w4(64, 13824, 5120, 64, "f16"), name="w4 64x13824x5120"),
        # one sequence on a short prefix, GQA with 8 queries per kv head: the smallest call
        dict(_prefix(1, 32, 4, 64, 512, False, False, "f16"), name="prefix 1 on 512"),
        # 16 sequences on one long document (Mistral-7B heads)
        dict(_prefix(16, 32, 8, 128, 32768, False, True, "bf16"), name="prefix 16 on 32768"),
        # 32 sequences, MHA (Llama-2-7B), each seeing its own share of the prefix, some none of it
        dict(_prefix(32, 32, 32, 128, 4096, True, True, "f16"), name="prefix 32 on 4096 ragged"),
        # 64 sequences, MHA (Llama-2-13B), a prefix that ends inside a tile
        dict(_prefix(64, 40, 40, 128, 8191, False, True, "bf16"), name="prefix 64 on 8191"),
        # 2048 prompt tokens of the sequences' own against the prefix in one call: products bound it
        dict(_prefix(2048, 32, 8, 128, 8192, False, True, "bf16"), name="prefix 2048 on 8192"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotary", "w4", "prefix"))
    if op == "rotary":
        dim = rng.choice((64, 80, 128))
        kv = rng.choice((1, 2, 4, 8, 32))
        heads = kv * rng.choice((1, 2, 4, 5, 8) if kv < 32 else (1,))
        batch = _log(rng, 1, 32)
        tokens = _log(rng, 1, max(1, 16384 * 40 // (batch * (heads + kv))))
        rd = dim if rng.random() < 0.6 else 2 * rng.randint(4, dim // 2)
        return _rotary(batch, tokens, heads, kv, dim, rd, rng.choice(("half", "interleaved")),
                       rng.choice(("none", "linear", "ntk", "yarn")), _log(rng, 1, 100000), rng.random() < 0.3,
                       rng.choice(("f16", "bf16", "f32")) if batch * tokens * (heads + kv) * dim < 4e7
                       else rng.choice(("f16", "bf16")))
    if op == "w4":
        group = rng.choice((32, 64, 128))
        k = group * _log(rng, 1, 13824 // group)
        n = _log(rng, 64, 14336)
        return _w4(_log(rng, 1, 64), k, n, group, rng.choice(("f16", "bf16", "bf16", "f32")))
    kv = rng.choice((1, 2, 4, 8, 32, 40))
    heads = kv * (rng.choice((1, 2, 4, 7, 8)) if kv <= 8 else 1)
    dim = rng.choice((64, 128))
    most = 2048 * 32 * 8192 * 128   # the largest listed product
    tokens = min(_log(rng, 1, 32768), 40 * 8192 * 128 // (kv * dim))
    rows = _log(rng, 1, max(1, min(2048, most // (heads * tokens * dim))))
    return _prefix(rows, heads, kv, dim, tokens, rng.random() < 0.4, rng.random() < 0.6, rng.choice(("f16", "bf16")))


# ── inputs ────────────────────────────────────────────────────────────────
_BASE, _TRAINED, _FACTOR = 10000.0, 4096, 8.0


def _theta(rd, scaling):
    """Radians per position of each pair (float64) and the attention factor."""
    i = np.arange(rd // 2, dtype=np.float64)
    base = _BASE * _FACTOR ** (rd / (rd - 2)) if scaling == "ntk" else _BASE
    th = base ** (-2 * i / rd)
    if scaling == "linear":
        return th / _FACTOR, 1.0
    if scaling == "yarn":
        def pair(turns):
            return rd * math.log(_TRAINED / (turns * 2 * math.pi)) / (2 * math.log(_BASE))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rd - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return th / _FACTOR * ramp + th * (1 - ramp), 0.1 * math.log(_FACTOR) + 1.0
    return th, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "rotary":
        b, t, d = case["batch"], case["tokens"], case["dim"]
        th, factor = _theta(case["rotary_dim"], case["scaling"])
        # pair i turns by freq[i] / 2^64 of a full circle per position
        freq = torch.tensor([round(x / (2 * math.pi) * 2.0 ** 64) for x in th], dtype=torch.int64, device="cuda")
        start = torch.randint(0, 32, (b, 1), device="cuda", generator=g) + case["start"]
        return dict(case=case, q=randn(b, t, case["heads"], d).to(dt), k=randn(b, t, case["kv_heads"], d).to(dt),
                    positions=start + torch.arange(t, device="cuda"), freq=freq, factor=factor)
    if case["op"] == "w4":
        n, k, gs = case["n"], case["k"], case["group"]
        w = randn(n, k // gs, gs) / math.sqrt(k)
        scale = (w.abs().amax(-1) / 7).to(dt)
        codes = (w / scale.float().unsqueeze(-1)).round_().clamp_(-8, 7).to(torch.int32).view(n, k)
        packed = ((codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)).to(torch.uint8)
        st = dict(case=case, x=randn(case["rows"], k).to(dt), packed=packed, scale=scale)
        if own:   # the weight in the kernels' layout, made once when a model is loaded
            st["weight"] = _ck().PackedWeight(packed, scale, gs)
        return st
    r, h, kv, d, n = (case[x] for x in ("rows", "heads", "kv_heads", "dim", "tokens"))
    k = randn(kv, n, d)
    k[:, :, :4] *= 20   # outlier channels, as trained keys have them
    st = dict(case=case, q=randn(r, h, d).to(dt), k=k.to(dt), v=randn(kv, n, d).to(dt), lengths=None, tail=None)
    if case["ragged"]:
        st["lengths"] = _lengths(case)[torch.randperm(r, device="cuda", generator=g)]
    if case["tail"]:
        lse = 8 + 4 * randn(r, h)
        lse[torch.randperm(r, device="cuda", generator=g)[: r // 8]] = -math.inf   # no token of their own yet
        o = torch.where(lse.unsqueeze(-1) > -math.inf, 0.3 * randn(r, h, d), 0.0)
        st["tail"] = (o.to(dt), lse)
    return st


def _lengths(case):
    """Visible prefix tokens of the sequences, from all of them down to none."""
    r, n = case["rows"], case["tokens"]
    return n - (torch.arange(r, device="cuda", dtype=torch.int32) * n) // max(1, r - 1)


# ── one pass ──────────────────────────────────────────────────────────────
def run(st):
    case = st["case"]
    if own:
        ck = _ck()
        if case["op"] == "rotary":
            return ck.apply_rotary(st["q"], st["k"], st["positions"], st["freq"], layout=case["layout"],
                                   attention_factor=st["factor"], inverse=case["inverse"])
        if case["op"] == "w4":
            return st["weight"].matvec(st["x"])
        return ck.prefix_attention(st["q"], st["k"], st["v"], lengths=st["lengths"], tail=st["tail"],
                                   return_lse=True)
    return {"rotary": _plain_rotary, "w4": _plain_w4, "prefix": _plain_prefix}[case["op"]](st)


def _plain_rotary(st):
    case = st["case"]
    # the product wraps at 2^64 = one turn; its top 32 bits as a signed half-turn fraction
    turn = (st["positions"].unsqueeze(-1) * st["freq"]) >> 32
    ang = turn.float() * (math.pi * 2.0 ** -31)
    cos, sin = torch.cos(ang) * st["factor"], torch.sin(ang) * st["factor"]
    if case["inverse"]:
        sin = -sin
    cos, sin = cos.unsqueeze(2), sin.unsqueeze(2)   # [batch, tokens, 1, pairs]
    rd = case["rotary_dim"]

    def turn_rows(x):
        r = x[..., :rd].float()
        if case["layout"] == "half":
            a, b = r[..., : rd // 2], r[..., rd // 2:]
            y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        return torch.cat((y.to(x.dtype), x[..., rd:]), -1)
    return turn_rows(st["q"]), turn_rows(st["k"])


def _plain_w4(st):
    case = st["case"]
    p = st["packed"].to(torch.int32)
    codes = torch.stack((p & 15, p >> 4), -1).flatten(1)
    codes = (codes ^ 8) - 8
    w = codes.float().view(case["n"], -1, case["group"]) * st["scale"].float().unsqueeze(-1)
    return (st["x"].float() @ w.view(case["n"], case["k"]).t()).to(st["x"].dtype)


def _plain_prefix(st):
    q, k, v = st["q"], st["k"], st["v"]
    (r, h, d), (kv, n, _) = q.shape, k.shape
    qg = q.float().view(r, kv, h // kv, d).transpose(0, 1).reshape(kv, -1, d)
    s = (qg / math.sqrt(d)) @ k.float().transpose(1, 2)   # [kv, r * group, n]
    if st["lengths"] is not None:
        hide = torch.arange(n, device=s.device) >= st["lengths"].unsqueeze(-1)
        s = s.view(kv, r, -1, n).masked_fill_(hide[None, :, None], -math.inf).view(kv, -1, n)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m > -math.inf, m, 0.0)
    p = s.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p @ v.float()) / torch.where(l > 0, l, 1.0)
    o = o.view(kv, r, -1, d).transpose(0, 1).reshape(r, h, d)
    lse = (m + torch.log(l)).view(kv, r, -1).transpose(0, 1).reshape(r, h)
    if st["tail"] is not None:
        ot, lt = st["tail"]
        top = torch.maximum(lse, lt)
        top = torch.where(top > -math.inf, top, 0.0)
        a, b = torch.exp(lse - top), torch.exp(lt - top)
        total = a + b
        wa, wb = (x / torch.where(total > 0, total, 1.0) for x in (a, b))
        o = o * wa.unsqueeze(-1) + ot.float() * wb.unsqueeze(-1)
        lse = top + torch.log(total)
    return o.to(q.dtype), lse


# ── what a pass cannot do without ─────────────────────────────────────────
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "rotary":
        tok = case["batch"] * case["tokens"]
        x = tok * (case["heads"] + case["kv_heads"])
        return dict(bytes=2 * x * case["dim"] * e + tok * 8, flops=3 * x * case["rotary_dim"])
    if case["op"] == "w4":
        m, k, n = case["rows"], case["k"], case["n"]
        return dict(bytes=n * k / 2 + n * k / case["group"] * e + m * (k + n) * e, flops=2 * m * n * k)
    r, h, kv, d, n = (case[x] for x in ("rows", "heads", "kv_heads", "dim", "tokens"))
    seen = sum(n - i * n // max(1, r - 1) for i in range(r)) if case["ragged"] else r * n
    return dict(bytes=2 * kv * n * d * e + (3 if case["tail"] else 2) * r * h * d * e
                + (8 if case["tail"] else 4) * r * h + (4 * r if case["ragged"] else 0), flops=4 * seen * h * d)


# ── the definitions in 64 bits ────────────────────────────────────────────
def exact(case, seed):
    st = prepare(case, seed)
    return {"rotary": _exact_rotary, "w4": _exact_w4, "prefix": _exact_prefix}[case["op"]](case, st)


def _exact_rotary(case, st):
    th, factor = _theta(case["rotary_dim"], case["scaling"])
    ang = torch.remainder(st["positions"].double()[..., None, None] * torch.from_numpy(th).cuda(), 2 * math.pi)
    z = torch.polar(torch.full_like(ang, factor), -ang if case["inverse"] else ang)
    half = case["rotary_dim"] // 2
    out = []
    for x in (st["q"].double(), st["k"].double()):
        first = torch.arange(half, device="cuda") * (1 if case["layout"] == "half" else 2)
        second = first + (half if case["layout"] == "half" else 1)
        w = torch.complex(x[..., first], x[..., second]) * z
        x = x.clone()
        x[..., first], x[..., second] = w.real, w.imag
        out.append(x)
    return tuple(out)


def _exact_w4(case, st):
    n, k, gs = case["n"], case["k"], case["group"]
    signed = st["packed"].view(torch.int8).double()
    high = torch.floor(signed / 16)
    low = signed - 16 * high
    low = torch.where(low > 7, low - 16, low)
    w = torch.empty(n, k, dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = low, high
    w *= st["scale"].double().repeat_interleave(gs, 1)
    return st["x"].double() @ w.T


def _exact_prefix(case, st):
    r, h, kv, d, n = (case[x] for x in ("rows", "heads", "kv_heads", "dim", "tokens"))
    group = h // kv
    out = torch.zeros(r, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((r, h), -math.inf, dtype=torch.float64, device="cuda")
    seen = torch.full((r,), n, device="cuda") if st["lengths"] is None else st["lengths"]
    some = seen > 0
    hide = torch.arange(n, device="cuda") >= seen[some].unsqueeze(-1)
    for j in range(h):
        s = (st["q"][some, j].double() @ st["k"][j // group].double().T / math.sqrt(d)).masked_fill_(hide, -math.inf)
        lse[some, j] = torch.logsumexp(s, -1)
        out[some, j] = torch.softmax(s, -1) @ st["v"][j // group].double()
    if st["tail"] is not None:
        both = torch.stack((lse, st["tail"][1].double()))
        any_ = both.amax(0) > -math.inf
        weight = torch.softmax(torch.where(any_, both, 0.0), 0)
        out = torch.where(any_.unsqueeze(-1), weight[0, ..., None] * out + weight[1, ..., None] * st["tail"][0].double(),
                          0.0)
        lse = torch.logsumexp(both, 0)
    return out, lse
