"""Rotary positions against the formula in 64 bits (GPU).

Tolerance: the result is rounded once to the dtype (relative 2^-9 for bf16,
2^-12 for fp16) after fp32 arithmetic on cos / sin whose angle is exact to
2^-24 of half a turn: |error| <= half ulp |y| + 2e-6 factor (|a| + |b|).
"""

import math

import pytest
import torch

from conftest import load_pkg

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # of a value, at most


def pkg():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_pkg()


def turned(x, positions, theta, layout, factor, inverse):
    """x [..., H, D] float64, positions [...]: the rotation, and |a| + |b| per element."""
    half = theta.numel()
    ang = torch.remainder(positions.double().unsqueeze(-1) * theta, 2 * math.pi).unsqueeze(-2)
    c, s = torch.cos(ang) * factor, torch.sin(ang) * factor * (-1 if inverse else 1)
    i = torch.arange(half, device=x.device)
    ia, ib = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = x[..., ia], x[..., ib]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


def theta_of(freq):
    return freq.double() * (2 * math.pi / 2.0 ** 64)


def check(got, x, positions, freq, layout, factor, inverse, dtype):
    ref, size = turned(x.double(), positions, theta_of(freq), layout, factor, inverse)
    err = (got.double() - ref).abs()
    tol = HALF_ULP[dtype] * ref.abs() + 2e-6 * factor * size + (2.0 ** -24 if dtype == "f16" else 0.0)
    assert got.dtype == x.dtype and bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rd", [(64, 64), (128, 128), (128, 96), (80, 20), (80, 34), (12, 6), (256, 256), (7, 2)])
def test_against_formula(dtype, layout, D, rd):
    ck = pkg()
    g = torch.Generator(device="cuda").manual_seed(D * 1000 + rd)
    freq, factor = ck.rotary_frequencies(rd, device="cuda")
    for B, T, Hq, Hk in ((1, 1, 1, 1), (1, 1, 32, 4), (2, 37, 6, 2), (3, 5, 3, 0)):
        q = torch.randn(B, T, Hq, D, device="cuda", generator=g).to(DT[dtype])
        k = torch.randn(B, T, Hk, D, device="cuda", generator=g).to(DT[dtype])
        pos = torch.randint(-5, 200000, (B, T), device="cuda", generator=g)
        yq, yk = ck.apply_rotary(q, k, pos, freq, layout=layout)
        check(yq, q, pos, freq, layout, factor, False, dtype)
        if Hk:
            check(yk, k, pos, freq, layout, factor, False, dtype)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_frequencies_and_far_positions(scaling):
    """Scaled frequencies against their formulas; a position of 2^20 keeps its digits."""
    ck = pkg()
    rd, base, s, L = 128, 10000.0, 4.0, 4096
    freq, factor = ck.rotary_frequencies(rd, base, scaling, s, L, device="cuda")
    i = torch.arange(rd // 2, dtype=torch.float64)
    th = (base * s ** (rd / (rd - 2)) if scaling == "ntk" else base) ** (-2 * i / rd)
    want_factor = 1.0
    if scaling == "linear":
        th = th / s
    if scaling == "yarn":
        want_factor = 0.1 * math.log(s) + 1
        turns = L * th / (2 * math.pi)       # pairs above 32 turns keep theta, below 1 turn are slowed by s
        assert torch.equal(theta_of(freq).cpu()[turns > 33], th[turns > 33]) or \
            float((theta_of(freq).cpu()[turns > 33] / th[turns > 33] - 1).abs().max()) < 1e-15
        slow = turns < 0.9
        assert float((theta_of(freq).cpu()[slow] * s / th[slow] - 1).abs().max()) < 1e-9
        mid = theta_of(freq).cpu() / th
        assert bool((mid[1:] <= mid[:-1] + 1e-12).all())
    else:
        assert float((theta_of(freq).cpu() / th - 1).abs().max()) < 1e-12
    assert factor == pytest.approx(want_factor)
    q = torch.randn(1, 3, 2, rd, device="cuda")
    pos = torch.tensor([2 ** 20, -2 ** 20, 0], device="cuda")
    yq, none = ck.apply_rotary(q, None, pos, freq, attention_factor=factor)
    assert none is None
    check(yq, q, pos, freq, "half", factor, False, "f32")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_outputs_and_positions(layout):
    """Transposed and fused views, int32 and broadcast positions, strided outputs."""
    ck = pkg()
    g = torch.Generator(device="cuda").manual_seed(3)
    B, T, Hq, Hk, D = 2, 19, 8, 2, 64
    freq, _ = ck.rotary_frequencies(48, device="cuda")
    qkv = torch.randn(B, T, (Hq + 2 * Hk) * D, device="cuda", generator=g).to(torch.bfloat16)
    q = qkv[..., : Hq * D].view(B, T, Hq, D)
    k = qkv[..., Hq * D:(Hq + Hk) * D].view(B, T, Hk, D)
    pos = torch.arange(T, device="cuda", dtype=torch.int32) + 11
    yq = torch.empty(B, Hq, T, D, device="cuda", dtype=torch.bfloat16)
    yk = torch.empty(B, Hk, T, D, device="cuda", dtype=torch.bfloat16)
    ck.apply_rotary(q, k, pos, freq, layout=layout, out=(yq.transpose(1, 2), yk.transpose(1, 2)))
    full = pos.expand(B, T)
    check(yq.transpose(1, 2), q, full, freq, layout, 1.0, False, "bf16")
    check(yk.transpose(1, 2), k, full, freq, layout, 1.0, False, "bf16")
    # rows that start at odd elements take the single-element path
    odd = torch.randn(1 + 7 * 3 * D, device="cuda", generator=g).half()[1:].view(7, 3, D)
    y, _ = ck.apply_rotary(odd, None, pos[:7], freq, layout=layout)
    check(y, odd, pos[:7], freq, layout, 1.0, False, "f16")
    # unit stride on another axis
    t = torch.randn(5, D, 3, device="cuda", generator=g).transpose(1, 2)
    y, _ = ck.apply_rotary(t, None, pos[:5], freq, layout=layout)
    check(y, t, pos[:5], freq, layout, 1.0, False, "f32")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient(layout):
    """backward = the inverse rotation: against the formula's gradient and differences."""
    ck = pkg()
    g = torch.Generator(device="cuda").manual_seed(5)
    T, H, D = 5, 2, 16
    freq, _ = ck.rotary_frequencies(12, device="cuda")
    pos = torch.randint(0, 9000, (T,), device="cuda", generator=g)
    q = torch.randn(T, H, D, device="cuda", generator=g, requires_grad=True)
    k = torch.randn(T, 1, D, device="cuda", generator=g, requires_grad=True)
    wq, wk = torch.randn(T, H, D, device="cuda", generator=g), torch.randn(T, 1, D, device="cuda", generator=g)
    yq, yk = ck.apply_rotary(q, k, pos, freq, layout=layout, attention_factor=1.25)
    ((yq * wq).sum() + (yk * wk).sum()).backward()
    check(q.grad, wq, pos, freq, layout, 1.25, True, "f32")
    check(k.grad, wk, pos, freq, layout, 1.25, True, "f32")
    # the map is linear: a central difference is exact up to rounding
    for j in range(D):
        e = torch.zeros_like(q)
        e[2, 1, j] = 0.5
        with torch.no_grad():
            up = ck.apply_rotary(q + e, None, pos, freq, layout=layout, attention_factor=1.25)[0]
            dn = ck.apply_rotary(q - e, None, pos, freq, layout=layout, attention_factor=1.25)[0]
        diff = float(((up - dn).double() * wq.double()).sum())
        assert diff == pytest.approx(float(q.grad[2, 1, j]), abs=2e-5)
    # only one of the two takes part in the loss
    q2 = q.detach().clone().requires_grad_()
    y2, _ = ck.apply_rotary(q2, k.detach(), pos, freq, layout=layout)
    (y2 * wq).sum().backward()
    check(q2.grad, wq, pos, freq, layout, 1.0, True, "f32")


def test_empty_other_stream_and_refusals():
    ck = pkg()
    freq, _ = ck.rotary_frequencies(64, device="cuda")
    e, _ = ck.apply_rotary(torch.empty(0, 4, 64, device="cuda"), None, torch.empty(0, dtype=torch.int64, device="cuda"),
                           freq)
    assert e.shape == (0, 4, 64)
    q = torch.randn(4, 2, 64, device="cuda")
    pos = torch.arange(4, device="cuda")
    want, _ = ck.apply_rotary(q, None, pos, freq)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, _ = ck.apply_rotary(q, None, pos, freq)
    s.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="positions"):
        ck.apply_rotary(q, None, pos.float(), freq)
    with pytest.raises(ValueError, match="positions"):
        ck.apply_rotary(q, None, pos[:3], freq)
    with pytest.raises(ValueError, match="layout"):
        ck.apply_rotary(q, None, pos, freq, layout="pairs")
    with pytest.raises(ValueError, match="rotary channels"):
        ck.apply_rotary(q[..., :32], None, pos, freq)
    with pytest.raises(ValueError, match="share storage"):
        ck.apply_rotary(q, None, pos, freq, out=(q, None))
    with pytest.raises(ValueError, match="dtype|expected"):
        ck.apply_rotary(q, q.half(), pos, freq)
    with pytest.raises(RuntimeError, match="CUDA"):
        ck.apply_rotary(q.cpu(), None, pos, freq)
    with pytest.raises(ck._lib.CareKVError):
        ck.apply_rotary(torch.randn(1, 1, 512, device="cuda"), None, pos[:1], freq)
    with pytest.raises(ValueError, match="rotary_dim"):
        ck.rotary_frequencies(7)
    with pytest.raises(ValueError, match="original_max_position"):
        ck.rotary_frequencies(8, scaling="yarn", factor=2.0)


def test_no_tokens_into_a_given_result():
    ck = pkg()
    freq, _ = ck.rotary_frequencies(64, device="cuda")
    q = torch.empty(0, 4, 64, device="cuda", dtype=torch.float16)
    y, _ = ck.apply_rotary(q, None, torch.empty(0, device="cuda", dtype=torch.int64), freq,
                           out=(torch.empty_like(q), None))
    assert y.shape == q.shape


def test_positions_changed_before_backward():
    """A gradient belongs to the positions and frequencies of its forward pass: changing them in place is an error."""
    ck = pkg()
    freq, _ = ck.rotary_frequencies(16, device="cuda")
    for changed in ("positions", "freq"):
        q = torch.randn(5, 2, 16, device="cuda", requires_grad=True)
        pos, f = torch.arange(5, device="cuda"), freq.clone()
        y, _ = ck.apply_rotary(q, None, pos, f)
        (pos if changed == "positions" else f).add_(1)
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_second_derivative(layout):
    """The gradient is linear in the output's gradient and can be differentiated by it: the forward turn again."""
    ck = pkg()
    freq, _ = ck.rotary_frequencies(12, device="cuda")
    pos = torch.arange(4, device="cuda") * 31
    q = torch.randn(4, 3, 16, device="cuda", requires_grad=True)
    w = torch.randn(4, 3, 16, device="cuda", requires_grad=True)
    u = torch.randn(4, 3, 16, device="cuda")
    y, _ = ck.apply_rotary(q, None, pos, freq, layout=layout, attention_factor=1.25)
    (dq,) = torch.autograd.grad((y * w).sum(), q, create_graph=True)
    check(dq.detach(), w.detach(), pos, freq, layout, 1.25, True, "f32")
    (dw,) = torch.autograd.grad((dq * u).sum(), w)
    check(dw, u, pos, freq, layout, 1.25, False, "f32")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_results_in_one_buffer(layout):
    """Results beside each other in one buffer (also the inputs' own, at other elements) are written in place; results
    that meet each other, the inputs, the positions or themselves are refused."""
    ck = pkg()
    g = torch.Generator(device="cuda").manual_seed(8)
    B, T, Hq, Hk, D = 2, 7, 4, 2, 64
    freq, _ = ck.rotary_frequencies(D, device="cuda")
    pos = torch.arange(T, device="cuda")
    q, k = (torch.randn(B, T, h, D, device="cuda", generator=g) for h in (Hq, Hk))
    want = ck.apply_rotary(q, k, pos, freq, layout=layout)

    def same(out, q_=q, k_=k):
        got = ck.apply_rotary(q_, k_, pos, freq, layout=layout, out=out)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    fused = torch.empty(B, T, Hq + Hk, D, device="cuda")
    same((fused[:, :, :Hq], fused[:, :, Hq:]))
    major = torch.empty(B, Hq + Hk, T, D, device="cuda")
    same((major[:, :Hq].transpose(1, 2), major[:, Hq:].transpose(1, 2)))
    wide = torch.empty(B, T, 2 * (Hq + Hk), D, device="cuda")     # inputs, then results, of every token
    wide[:, :, :Hq], wide[:, :, Hq:Hq + Hk] = q, k
    same((wide[:, :, Hq + Hk:2 * Hq + Hk], wide[:, :, 2 * Hq + Hk:]), wide[:, :, :Hq], wide[:, :, Hq:Hq + Hk])
    flat = torch.empty(2, q.numel(), device="cuda")
    flat[0] = q.flatten()
    same((flat[1].view(q.shape), torch.empty_like(k)), flat[0].view(q.shape))
    bad = [(fused[:, :, :Hq], fused[:, :, Hq - 1:-1]),                               # one head of both
           (fused[:, :, :Hq], fused[:, :, :Hk]),
           (torch.empty(B, T, 1, D, device="cuda").expand(B, T, Hq, D), torch.empty_like(k)),   # meets itself
           (q, torch.empty_like(k)), (torch.empty_like(q), k),
           (torch.empty_like(q), q[:, :, :Hk])]
    for out in bad:
        with pytest.raises(ValueError, match="overlap|share storage"):
            ck.apply_rotary(q, k, pos, freq, layout=layout, out=out)
    room = torch.zeros(q.numel(), device="cuda")
    with pytest.raises(ValueError, match="overlap|share storage"):
        ck.apply_rotary(q, k, room.view(torch.int64)[:T], freq, layout=layout, out=(room.view(q.shape), torch.empty_like(k)))


def test_yarn_ramp():
    """Every pair's frequency: theta (1 - r) + theta / s r, r rising from the pair that turns beta_fast times to the one
    that turns beta_slow times within the trained range (their indices rounded outwards)."""
    ck = pkg()
    for rd, base, s, L, fast, slow in ((128, 10000.0, 8.0, 4096, 32.0, 1.0), (64, 500000.0, 4.0, 8192, 16.0, 2.0)):
        freq, factor = ck.rotary_frequencies(rd, base, "yarn", s, L, beta_fast=fast, beta_slow=slow)
        assert factor == pytest.approx(0.1 * math.log(s) + 1)
        at = [rd / 2 * math.log(L / (2 * math.pi * t)) / math.log(base) for t in (fast, slow)]
        lo, hi = math.floor(at[0]), math.ceil(at[1])
        assert 0 < lo < hi < rd // 2
        for i, f in enumerate(theta_of(freq).tolist()):
            r = min(max((i - lo) / (hi - lo), 0.0), 1.0)
            theta = base ** (-2 * i / rd)
            assert f == pytest.approx(theta * (1 - r) + theta / s * r, rel=1e-12)
