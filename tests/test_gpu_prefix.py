"""Attention over a shared prefix against 64-bit softmax (GPU).

Tolerance, per element: with d = head_dim 2^-24 scale sum |q| |k| the largest
error of an fp32 score, a weight is off by a factor 1 +- (2 d + 4e-6), plus half
an ulp of the 16-bit type where weights enter the matrix product in it; the
result is rounded once: |error| <= half ulp |o| + (half ulp + 2 d + 4e-6) sum p |v|.
The log-sum-exp is off by at most d + 4e-6 (1 + |lse|).
"""

import ctypes
import math

import pytest
import torch

from conftest import load_pkg

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def pkg():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_pkg()


def reference(q, k, v, scale, lengths, tail):
    """(o, sum p |v|, lse, d) in float64, shaped [n, Hq, ...]."""
    n, hq, D = q.shape
    hkv, N, _ = k.shape
    g = hq // hkv
    kd, vd = k.double().repeat_interleave(g, 0), v.double().repeat_interleave(g, 0)
    qd = q.double().transpose(0, 1)
    seen = torch.full((n,), N, device=q.device) if lengths is None else lengths.long().clamp(0, N)
    top = int(seen.max()) if n else 0
    kd, vd = kd[:, :top], vd[:, :top]
    s = scale * qd @ kd.transpose(1, 2)                                   # [Hq, n, top]
    hide = torch.arange(top, device=q.device) >= seen.unsqueeze(-1)
    s = s.masked_fill(hide, -math.inf)
    d = (D * 2.0 ** -24 * scale * (qd.abs() @ kd.abs().transpose(1, 2))).masked_fill(hide, 0.0)
    d = d.amax(-1) if top else torch.zeros(hq, n, dtype=torch.float64, device=q.device)
    lse = torch.logsumexp(s, -1) if top else torch.full((hq, n), -math.inf, dtype=torch.float64, device=q.device)
    p = torch.exp(s - torch.where(lse > -math.inf, lse, 0.0).unsqueeze(-1))
    o, size = p @ vd, p @ vd.abs()
    o, size, lse, d = (x.transpose(0, 1) for x in (o, size, lse, d))
    if tail is not None:
        to, tl = tail[0].double(), tail[1].double()
        both = torch.logaddexp(lse, tl)
        ref = torch.where(both > -math.inf, both, 0.0)
        a, b = torch.exp(lse - ref).unsqueeze(-1), torch.exp(tl - ref).unsqueeze(-1)
        to = torch.where(b > 0, to, 0.0)
        o, size, lse = a * o + b * to, a * size + b * to.abs(), both
    return o, size, lse, d


def check(got, lse, q, k, v, dtype, scale=None, lengths=None, tail=None):
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    o, size, ref_lse, d = reference(q, k, v, scale, lengths, tail)
    h = HALF_ULP[dtype]
    tol = h * o.abs() + (h + 2 * d.unsqueeze(-1) + 4e-6) * size + (2.0 ** -24 if dtype == "f16" else 1e-30)
    err = (got.double() - o).abs()
    assert got.dtype == q.dtype and bool((err <= tol).all()), float((err - tol).max())
    some = ref_lse > -math.inf
    assert torch.equal(lse > -math.inf, some)
    off = (lse.double() - ref_lse)[some].abs()
    assert bool((off <= (d + 4e-6 * (1 + ref_lse.abs()))[some]).all()), float(off.max())
    assert bool((got[~some] == 0).all())


def inputs(n, hq, hkv, D, N, dtype, seed=0, outliers=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(n, hq, D, device="cuda", generator=g)
    k = torch.randn(hkv, N, D, device="cuda", generator=g)
    if outliers:
        k[..., : max(1, D // 32)] *= 8
    v = torch.randn(hkv, N, D, device="cuda", generator=g)
    return q.to(DT[dtype]), k.to(DT[dtype]), v.to(DT[dtype])


def own_state(n, hq, D, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    o = (0.3 * torch.randn(n, hq, D, device="cuda", generator=g)).to(DT[dtype])
    lse = 3 + 4 * torch.randn(n, hq, device="cuda", generator=g)
    lse[::3] = -math.inf
    o[::3] = float("nan")     # a state of no tokens may hold anything
    return o, lse


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,hq,hkv", [(1, 4, 4), (1, 8, 1), (3, 14, 2), (17, 8, 2), (33, 32, 4), (130, 3, 3),
                                      (300, 8, 1)])
def test_sizes(dtype, D, n, hq, hkv):
    ck = pkg()
    for N in (1, 2, 31, 64, 127, 128, 129, 255, 300, 513, 1100):
        q, k, v = inputs(n, hq, hkv, D, N, dtype, N)
        o, lse = ck.prefix_attention(q, k, v, return_lse=True)
        check(o, lse, q, k, v, dtype)
        tail = own_state(n, hq, D, dtype)
        o, lse = ck.prefix_attention(q, k, v, tail=tail, return_lse=True, scale=0.05)
        check(o, lse, q, k, v, dtype, scale=0.05, tail=tail)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,hq,hkv,D", [(40, 4, 2, 128), (200, 8, 2, 64), (9, 40, 40, 128), (300, 6, 2, 128)])
def test_lengths(dtype, n, hq, hkv, D):
    """Rows that see part of the prefix, none of it, or more than there is; what no row sees may hold NaN."""
    ck = pkg()
    for N, top in ((5, 3), (128, 128), (129, 128), (700, 389), (700, 700), (384, 257)):
        q, k, v = inputs(n, hq, hkv, D, N, dtype, N)
        g = torch.Generator(device="cuda").manual_seed(7)
        lengths = torch.randint(0, top + 1, (n,), device="cuda", generator=g, dtype=torch.int32)
        lengths[0], lengths[-1] = top, 0
        if n > 4:
            lengths[1] = -3
        clean = (k.clone(), v.clone())
        k[:, top:] = float("nan")
        v[:, top:] = float("inf")
        for tail in (None, own_state(n, hq, D, dtype)):
            o, lse = ck.prefix_attention(q, k, v, lengths=lengths, tail=tail, return_lse=True)
            check(o, lse, q, *clean, dtype, lengths=lengths, tail=tail)
    # more than there is: the whole prefix
    q, k, v = inputs(n, hq, hkv, D, 200, dtype)
    o, lse = ck.prefix_attention(q, k, v, lengths=torch.full((n,), 10 ** 6, dtype=torch.int32, device="cuda"),
                                 return_lse=True)
    check(o, lse, q, k, v, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_tokens(dtype):
    ck = pkg()
    q, k, v = inputs(6, 4, 2, 64, 0, dtype)
    o, lse = ck.prefix_attention(q, k, v, return_lse=True)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    tail = own_state(6, 4, 64, dtype)
    o, lse = ck.prefix_attention(q, k, v, tail=tail, return_lse=True)
    check(o, lse, q, k, v, dtype, tail=tail)
    q, k, v = inputs(5, 4, 2, 64, 300, dtype)
    zero = torch.zeros(5, dtype=torch.int32, device="cuda")
    o, lse = ck.prefix_attention(q, k, v, lengths=zero, return_lse=True)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    assert ck.prefix_attention(q[:0], k, v).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_head_dims(dtype):
    ck = pkg()
    for D in (1, 24, 80, 96, 200, 256):
        q, k, v = inputs(11, 6, 3, D, 150, dtype, D)
        o, lse = ck.prefix_attention(q, k, v, return_lse=True)
        check(o, lse, q, k, v, dtype)


def test_strides_streams_and_out():
    """Token-major K / V, views into a fused projection, another stream, a given output."""
    ck = pkg()
    for D in (64, 128):
        n, hq, hkv, N = 21, 8, 2, 333
        g = torch.Generator(device="cuda").manual_seed(D)
        kv = torch.randn(N, 2 * hkv * D, device="cuda", generator=g).to(torch.bfloat16)
        k = kv[:, : hkv * D].view(N, hkv, D).transpose(0, 1)
        v = kv[:, hkv * D:].view(N, hkv, D).transpose(0, 1)
        q = torch.randn(n, (hq + 3) * D, device="cuda", generator=g).to(torch.bfloat16)[:, D:(hq + 1) * D].view(n, hq, D)
        o, lse = ck.prefix_attention(q, k, v, return_lse=True)
        check(o, lse, q, k, v, "bf16")
        out = torch.empty(n, hq, D, device="cuda", dtype=torch.bfloat16)
        assert ck.prefix_attention(q, k, v, out=out) is out
        assert torch.equal(out, o)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = ck.prefix_attention(q, k, v)
        s.synchronize()
        assert torch.equal(other, o)
        # rows that start at odd elements, and channels that are not adjacent
        odd = torch.randn(1 + hkv * N * D, device="cuda", generator=g).to(torch.bfloat16)[1:].view(hkv, N, D)
        o, lse = ck.prefix_attention(q, odd, odd, return_lse=True)
        check(o, lse, q, odd, odd, "bf16")
        kt = torch.randn(hkv, D, N, device="cuda", generator=g).to(torch.bfloat16).transpose(1, 2)
        qt = torch.randn(D, hq, n, device="cuda", generator=g).to(torch.bfloat16).permute(2, 1, 0)
        o, lse = ck.prefix_attention(qt, kt, k, return_lse=True)
        check(o, lse, qt, kt, k, "bf16")
        # one kv head broadcast to several
        kb = k[:1].expand(4, N, D)
        o, lse = ck.prefix_attention(q, kb, kb, return_lse=True)
        check(o, lse, q, kb, kb, "bf16")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_growing_maximum(dtype):
    """Scores that rise (or fall) steadily by tens along the prefix: the running maximum moves at every tile."""
    ck = pkg()
    for D in (64, 128):
        n, hq, hkv, N = 7, 8, 2, 1500
        q, k, v = inputs(n, hq, hkv, D, N, dtype, 3, outliers=False)
        q[..., 0] = 4.0
        ramp = torch.linspace(-60, 60, N, device="cuda")
        for r in (ramp, ramp.flip(0)):
            k[..., 0] = r.to(k.dtype)
            for lengths in (None, torch.arange(n, device="cuda", dtype=torch.int32) * 200):
                o, lse = ck.prefix_attention(q, k, v, scale=1.0, lengths=lengths, return_lse=True)
                check(o, lse, q, k, v, dtype, scale=1.0, lengths=lengths)


def test_scores_of_the_types_lowest_value():
    """Keys that push scores to the type's lowest value weigh nothing; a prefix of only such keys is an even mean."""
    ck = pkg()
    for dtype in ("f16", "bf16"):
        n, hq, hkv, D, N = 5, 4, 2, 64, 200
        q, k, v = inputs(n, hq, hkv, D, N, dtype, 5, outliers=False)
        q[..., 0] = 1.0
        k[..., 1:] = 0
        k[..., 0] = 0
        k[:, 50:150, 0] = torch.finfo(DT[dtype]).min
        o, lse = ck.prefix_attention(q, k, v, scale=1.0, return_lse=True)
        check(o, lse, q, k, v, dtype, scale=1.0)
        k[..., 0] = torch.finfo(torch.float16).min
        o, lse = ck.prefix_attention(q, k, v, scale=1.0, return_lse=True)
        check(o, lse, q, k, v, dtype, scale=1.0)


def test_shared_prefix_object():
    ck = pkg()
    q, k, v = inputs(4, 8, 2, 64, 100, "f16")
    sp = ck.SharedPrefix(2)
    assert sp.tokens is None
    sp.set(0, k, v)
    sp.set(1, v, k)
    assert sp.tokens == 100 and sp.memory_bytes() == 4 * k.numel() * 2
    assert torch.equal(sp.attend(1, q), ck.prefix_attention(q, v, k))
    with pytest.raises(ValueError, match="layer 0 holds 90"):
        sp.set(0, k[:, :90], v[:, :90])
    with pytest.raises(ValueError, match="has not been set"):
        ck.SharedPrefix(1).attend(0, q)


def test_refusals():
    ck = pkg()
    q, k, v = inputs(4, 8, 2, 64, 100, "f16")
    with pytest.raises(ValueError, match="query heads"):
        ck.prefix_attention(q[:, :7], k, v)
    with pytest.raises(ValueError, match="expected"):
        ck.prefix_attention(q, k.float(), v)
    with pytest.raises(ValueError, match="do not fit"):
        ck.prefix_attention(q, k, v[:, :50])
    with pytest.raises(ValueError, match="lengths"):
        ck.prefix_attention(q, k, v, lengths=torch.ones(4, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="tail"):
        ck.prefix_attention(q, k, v, tail=(q, torch.zeros(4, 8, device="cuda").half()))
    with pytest.raises(RuntimeError, match="CUDA"):
        ck.prefix_attention(q.cpu(), k, v)
    with pytest.raises(ck._lib.CareKVError, match="unsupported"):
        big = torch.zeros(1, 1, 512, device="cuda")
        ck.prefix_attention(big, big, big)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,hq,hkv,D,N", [
    (1200, 40, 40, 64, 300),     # more tiles than SMs: whole tiles first, the rest shared
    (700, 64, 64, 128, 520),
    (20, 100, 100, 64, 8192),    # tiles do not divide the SMs: CTAs cross from one tile into the next
    (3, 90, 90, 128, 5000),
    (5, 148, 148, 64, 640)])     # a tile per SM
def test_shares_of_the_prefix(dtype, n, hq, hkv, D, N):
    """Every way the prefix is cut over CTAs, with all tokens seen and with ragged lengths and own states."""
    ck = pkg()
    q, k, v = inputs(n, hq, hkv, D, N, dtype, n + hq)
    o, lse = ck.prefix_attention(q, k, v, return_lse=True)
    check(o, lse, q, k, v, dtype)
    g = torch.Generator(device="cuda").manual_seed(N)
    lengths = torch.randint(0, N + 1, (n,), device="cuda", generator=g, dtype=torch.int32)
    lengths[0] = 0
    tail = own_state(n, hq, D, dtype)
    o, lse = ck.prefix_attention(q, k, v, lengths=lengths, tail=tail, return_lse=True)
    check(o, lse, q, k, v, dtype, lengths=lengths, tail=tail)


def test_result_must_not_overlap_its_inputs():
    ck = pkg()
    buf = torch.randn(3, 4, 8, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.randn(2, 50, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        ck.prefix_attention(buf[0], k, k, out=buf[0])
    want = ck.prefix_attention(buf[0], k, k)
    assert torch.equal(ck.prefix_attention(buf[0], k, k, out=buf[1]), want)      # neighbours in one buffer are fine
    none = torch.empty(0, 8, 64, device="cuda", dtype=torch.bfloat16)
    assert ck.prefix_attention(none, k, k, out=torch.empty_like(none)).shape == (0, 8, 64)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,hq,hkv,D,N", [(1, 4, 4, 64, 300), (40, 8, 2, 128, 512),     # tiles that a CTA holds whole
                                          (700, 64, 64, 128, 200), (20, 8, 8, 64, 3000)])   # ... with shared ones; shared
def test_results_and_workspaces_on_16_byte_boundaries(dtype, n, hq, hkv, D, N):
    """A result, and (through the C entry) a workspace, that starts 16 bytes past a 32-byte boundary: the same bits."""
    ck = pkg()
    q, k, v = inputs(n, hq, hkv, D, N, dtype, N)
    tail = own_state(n, hq, D, dtype)
    want, want_lse = ck.prefix_attention(q, k, v, tail=tail, return_lse=True)
    check(want, want_lse, q, k, v, dtype, tail=tail)
    buf = torch.zeros(8 + q.numel() + 8, device="cuda", dtype=DT[dtype])
    out = buf[8:8 + q.numel()].view(n, hq, D)
    assert out.data_ptr() % 32 == 16
    ck.prefix_attention(q, k, v, tail=tail, out=out)
    assert torch.equal(out, want) and not buf[:8].any() and not buf[-8:].any()
    L = ck._lib
    prefix = L.PREFIX_PACK(k.data_ptr(), v.data_ptr(), N * D, D, N * D, D, hkv, N, D, L.F16 if dtype == "f16" else L.BF16)
    need = ctypes.c_size_t(0)
    L.check(L.lib().carekv_prefix_workspace_bytes(prefix, n, hq, ctypes.byref(need)), "workspace")
    ws = torch.zeros(need.value + 32, device="cuda", dtype=torch.uint8)
    assert ws.data_ptr() % 32 == 0
    lse = torch.empty_like(want_lse)
    L.check(L.lib().carekv_prefix_attention(prefix, q.data_ptr(), hq * D, D, n, hq, 1 / math.sqrt(D), None,
                                            tail[0].data_ptr(), tail[1].data_ptr(), out.data_ptr(), lse.data_ptr(),
                                            ws.data_ptr() + 16, need.value, torch.cuda.current_stream().cuda_stream),
            "prefix")
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert not ws[:16].any() and not ws[need.value + 16:].any()


@pytest.mark.parametrize("n,hq,hkv,D,N", [(9, 4, 4, 64, 300), (9, 4, 4, 128, 4000), (300, 2, 2, 64, 700),
                                          (300, 2, 2, 128, 260)])
def test_hidden_tokens_weigh_nothing(n, hq, hkv, D, N):
    """The type's largest values in tokens that a row does not see leave no trace in it."""
    ck = pkg()
    q, k, v = inputs(n, hq, hkv, D, N, "bf16", 11)
    half = N // 2 + 3
    lengths = torch.full((n,), half, dtype=torch.int32, device="cuda")
    lengths[1::2] = N
    clean = v.clone()
    v[:, half:] = torch.finfo(torch.bfloat16).max / N
    v[:, half:, ::2] *= -1
    o, lse = ck.prefix_attention(q, k, v, lengths=lengths, return_lse=True)
    some = torch.arange(0, n, 2, device="cuda")
    check(o[some], lse[some], q[some], k, clean, "bf16", lengths=lengths[some])


def test_far_scores_weigh_nothing():
    """Visible tokens whose weight is below 2^-150 of the largest one's leave no trace, whatever their values."""
    ck = pkg()
    for n, hq in ((5, 4), (300, 2)):
        D, N = 64, 256
        q, k, v = inputs(n, hq, hq, D, N, "bf16", 12, outliers=False)
        q[..., 0], k[..., 0] = 1.0, 0.0
        k[:, 1::2, 0] = -1000.0
        v[:, 1::2] = 1e38
        o, lse = ck.prefix_attention(q, k, v, scale=1.0, return_lse=True)
        v[:, 1::2] = 0
        check(o, lse, q, k, v, "bf16", scale=1.0)


def test_inputs_that_require_a_gradient_are_refused():
    """The operator has no backward pass: it says so instead of dropping a gradient."""
    ck = pkg()
    q, k, v = inputs(3, 4, 2, 64, 40, "f32")
    tail = own_state(3, 4, 64, "f32")
    args = dict(q=q, k=k, v=v)
    for name in args:
        bad = dict(args, **{name: args[name].clone().requires_grad_()})
        with pytest.raises(RuntimeError, match="backward"):
            ck.prefix_attention(**bad)
        with torch.no_grad():
            assert torch.equal(ck.prefix_attention(**bad), ck.prefix_attention(q, k, v))
    for i in range(2):
        bad = tuple(t.clone().requires_grad_() if j == i else t for j, t in enumerate(tail))
        with pytest.raises(RuntimeError, match="backward"):
            ck.prefix_attention(q, k, v, tail=bad)


def test_result_over_the_own_state():
    """`out` may be the own state's output itself; at another place over it, its log-sum-exp or the lengths it is refused."""
    ck = pkg()
    for n, N in ((6, 200), (6, 3000), (300, 700)):      # whole tiles, shared tiles, both
        q, k, v = inputs(n, 8, 2, 64, N, "f16")
        o, lse = own_state(n, 8, 64, "f16")
        lengths = torch.full((n,), N, dtype=torch.int32, device="cuda")
        want = ck.prefix_attention(q, k, v, tail=(o, lse))
        buf = torch.empty(n + 1, 8, 64, device="cuda", dtype=torch.float16)
        buf[:n] = o
        with pytest.raises(ValueError, match="overlap"):
            ck.prefix_attention(q, k, v, tail=(buf[:n], lse), out=buf[1:])
        assert torch.equal(ck.prefix_attention(q, k, v, tail=(buf[:n], lse), out=buf[:n]), want)
        over = torch.empty(q.numel(), device="cuda", dtype=torch.float16)
        state = over.view(torch.float32)[:n * 8].view(n, 8)
        with pytest.raises(ValueError, match="overlap"):
            ck.prefix_attention(q, k, v, tail=(o, state), out=over.view(q.shape))
        with pytest.raises(ValueError, match="overlap"):
            ck.prefix_attention(q, k, v, lengths=over.view(torch.int32)[:n], out=over.view(q.shape))
        with pytest.raises(ValueError, match="overlap"):
            odd = torch.empty(2 * q.numel(), device="cuda", dtype=torch.float16)
            ck.prefix_attention(odd[4:4 + q.numel()].view(q.shape), k, v, out=odd[:q.numel()].view(q.shape))
        ck.prefix_attention(q, k, v, lengths=lengths, out=buf[:n])


def test_shared_prefix_holds_its_own_values():
    """A later write to the tensors given to set() does not change the prefix; a layer can be set anew, to another
    length too where no other layer holds one."""
    ck = pkg()
    q, k, v = inputs(4, 8, 2, 64, 100, "f16")
    sp = ck.SharedPrefix(1)
    sp.set(0, k, v)
    want = sp.attend(0, q)
    k.zero_()
    v.zero_()
    assert torch.equal(sp.attend(0, q), want)
    _, k, v = inputs(4, 8, 2, 64, 60, "f16", 3)
    sp.set(0, k, v)
    assert sp.tokens == 60 and torch.equal(sp.attend(0, q), ck.prefix_attention(q, k, v))
    sp.set(0, k.float().requires_grad_(), v.float())
    assert not sp.layer(0)[0].requires_grad


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_many_rows_on_a_long_prefix(dtype):
    ck = pkg()
    for n, hq, hkv, D, N in ((300, 4, 2, 128, 5003), (260, 2, 2, 64, 9000)):
        q, k, v = inputs(n, hq, hkv, D, N, dtype, n)
        o, lse = ck.prefix_attention(q, k, v, return_lse=True)
        check(o, lse, q, k, v, dtype)


def test_results_repeat_and_run_in_a_graph():
    """The same bits at every call, and from a captured graph (also with other values in the same tensors)."""
    ck = pkg()
    for n, hq, hkv, D, N in ((2, 8, 2, 64, 300), (20, 8, 8, 128, 3000), (300, 4, 2, 128, 3000)):
        q, k, v = inputs(n, hq, hkv, D, N, "bf16", 5)
        tail = own_state(n, hq, D, "bf16")
        want = ck.prefix_attention(q, k, v, tail=tail, return_lse=True)
        for _ in range(20):
            got = ck.prefix_attention(q, k, v, tail=tail, return_lse=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, lse = ck.prefix_attention(q, k, v, tail=tail, return_lse=True)
        graph.replay()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        q.neg_()
        graph.replay()
        assert not torch.equal(o, want[0])
        got = ck.prefix_attention(q, k, v, tail=tail, return_lse=True)
        assert torch.equal(o, got[0]) and torch.equal(lse, got[1])
