"""4-bit weight products against 64-bit sums (GPU).

Tolerance: codes and activations enter exactly; what rounds is the fp32 sum
of the K products (at most K 2^-24 sum |w| |x|, each partial sum once) and the
result's own dtype (half an ulp).
"""

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


def weight(n, k, group, dtype, seed=0):
    """Random packed rows, scales, and the weight they stand for (float64)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), device="cuda", generator=g)
    scale = (0.01 + 0.1 * torch.rand(n, k // group, device="cuda", generator=g)).to(DT[dtype])
    packed = ((codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)).to(torch.uint8)
    return packed, scale, codes.double() * scale.double().repeat_interleave(group, 1)


def check(got, x, w, dtype):
    x = x.double().reshape(-1, w.shape[1])
    ref, size = x @ w.T, x.abs() @ w.abs().T
    tol = HALF_ULP[dtype] * ref.abs() + w.shape[1] * 2.0 ** -24 * size + (2.0 ** -24 if dtype == "f16" else 0.0)
    err = (got.double().reshape(ref.shape) - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,group", [(16, 128, 32), (1, 32, 32), (37, 96, 32), (64, 320, 64), (130, 1024, 128),
                                       (250, 768, 256), (1000, 4096, 32), (33, 5632, 64)])
def test_against_sums(dtype, n, k, group):
    ck = pkg()
    packed, scale, w = weight(n, k, group, dtype, n + k)
    pw = ck.PackedWeight(packed, scale, group)
    g = torch.Generator(device="cuda").manual_seed(1)
    for m in (1, 2, 7, 8, 9, 16, 17, 32, 33, 64, 65, 130):
        x = torch.randn(m, k, device="cuda", generator=g).to(DT[dtype])
        y = pw.matvec(x)
        assert y.shape == (m, n) and y.dtype == x.dtype
        check(y, x, w, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_shapes_of_the_model_layers(dtype):
    ck = pkg()
    for n, k, group, m in ((4096, 4096, 32, 3), (2048, 5632, 64, 1), (5120, 13824, 64, 20), (14336, 4096, 128, 48)):
        packed, scale, w = weight(n, k, group, dtype, n)
        x = torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(DT[dtype])
        check(ck.PackedWeight(packed, scale, group).matvec(x), x, w, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_quantized_dense_weight(dtype):
    """from_dense = the package quantizer's codes and scales; dequantize and matmul agree with them."""
    ck = pkg()
    g = torch.Generator(device="cuda").manual_seed(4)
    dense = (torch.randn(72, 256, device="cuda", generator=g) / 16).to(DT[dtype])
    pw = ck.PackedWeight.from_dense(dense, group_size=64)
    codes, scale = ck.quantize(dense, ck.QuantConfig(bits=4, group_size=64))
    w = codes.double() * scale.double().repeat_interleave(64, 1)
    assert torch.equal(pw.dequantize(), (codes.float() * scale.float().repeat_interleave(64, 1)).to(DT[dtype]))
    x = torch.randn(5, 256, device="cuda", generator=g).to(DT[dtype])
    check(pw.matvec(x), x, w, dtype)
    assert torch.equal(pw.matmul(x), pw.matvec(x))
    big = torch.randn(200, 256, device="cuda", generator=g).to(DT[dtype])
    # above the row limit the weight itself is rounded to the dtype: its half ulp joins
    ref, size = big.double() @ w.T, big.double().abs() @ w.abs().T
    tol = HALF_ULP[dtype] * (ref.abs() + size) + 256 * 2.0 ** -24 * size
    assert bool(((pw.matmul(big).double() - ref).abs() <= tol).all())


def test_infinite_and_nan_activations_stay_in_their_row():
    ck = pkg()
    for dtype in DT:
        packed, scale, w = weight(40, 160, 32, dtype, 9)
        x = torch.randn(4, 160, device="cuda").to(DT[dtype])
        x[1, 5] = float("nan")
        x[2, 7] = float("inf")
        y = ck.PackedWeight(packed, scale, 32).matvec(x)
        assert bool(y[1].isnan().all())
        c = w[:, 7]
        assert bool(y[2][c > 0].eq(float("inf")).all()) and bool(y[2][c < 0].eq(float("-inf")).all())
        assert bool(y[2][c == 0].isnan().all())
        check(y[0::3], x[0::3], w, dtype)


def test_strides_streams_and_out():
    ck = pkg()
    packed, scale, w = weight(50, 256, 32, "f16", 11)
    pw = ck.PackedWeight(packed, scale, 32)
    wide = torch.randn(6, 512, device="cuda").half()
    for x in (wide[:, 256:], wide[:, :256], wide[::2, 3:259], wide[:, ::2], wide.view(2, 3, 512)[..., :256],
              wide[:1, :256].expand(3, 256), wide[0, :256]):
        y = pw.matvec(x)
        assert y.shape == (*x.shape[:-1], 50)
        check(y, x, w, "f16")
    assert pw.matvec(wide[:0, :256]).shape == (0, 50)
    out = torch.empty(6, 50, device="cuda", dtype=torch.float16)
    assert pw.matvec(wide[:, :256], out=out) is out
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = pw.matvec(wide[:, :256])
    s.synchronize()
    assert torch.equal(other, out)


def test_refusals():
    ck = pkg()
    packed, scale, _ = weight(16, 128, 32, "f16")
    pw = ck.PackedWeight(packed, scale, 32)
    with pytest.raises(ValueError, match="expected"):
        pw.matvec(torch.randn(2, 128, device="cuda"))
    with pytest.raises(ValueError, match="expected"):
        pw.matvec(torch.randn(2, 64, device="cuda").half())
    with pytest.raises(RuntimeError):
        pw.matvec(torch.randn(2, 128).half())
    with pytest.raises(ValueError, match="out"):
        pw.matvec(torch.randn(2, 128, device="cuda").half(), out=torch.empty(2, 17, device="cuda").half())
    with pytest.raises(ValueError, match="scale"):
        ck.PackedWeight(packed, scale[:, :3], 32)
    with pytest.raises(ValueError, match="byte"):
        ck.PackedWeight(packed.float(), scale, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ck.PackedWeight(packed.cpu(), scale, 32)
    p16, s16, _ = weight(16, 128, 16, "f16")
    with pytest.raises(ck._lib.CareKVError, match="unsupported"):
        ck.PackedWeight(p16, s16, 16)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,k,group,m", [(3001, 2912, 32, 33), (3001, 2912, 32, 64), (2999, 3008, 64, 41),
                                         (8209, 4128, 32, 17), (8200, 4224, 128, 20), (8193, 4352, 256, 32),
                                         (8209, 4128, 32, 100)])
def test_larger_weights_of_odd_sizes(dtype, n, k, group, m):
    """Weights above the size from which more rows go to the tensor cores: ragged rows, channels, groups, batches."""
    ck = pkg()
    packed, scale, w = weight(n, k, group, dtype, n + m)
    x = torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(m)).to(DT[dtype])
    check(ck.PackedWeight(packed, scale, group).matvec(x), x, w, dtype)


def test_result_must_not_overlap_its_rows():
    ck = pkg()
    packed, scale, w = weight(64, 64, 32, "bf16", 3)
    pw = ck.PackedWeight(packed, scale, 32)
    buf = torch.randn(2, 5, 64, device="cuda").to(torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        pw.matvec(buf[0], out=buf[0])
    x = buf[0].clone()
    check(pw.matvec(buf[0], out=buf[1]), x, w, "bf16")       # neighbours in one buffer are fine
    none = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    assert pw.matvec(none, out=torch.empty_like(none)).shape == (0, 64)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 64, 65])
def test_gradient_of_the_activations(dtype, rows):
    """dx = dy W, on both sides of the row limit of matmul.  Tolerance: the weight rounded to the dtype (half an ulp of
    each term), the library product's sums (n 2^-24, and half an ulp where a partial sum is kept in the dtype) and the
    result's own rounding."""
    ck = pkg()
    n, k = 96, 160
    packed, scale, w = weight(n, k, 32, dtype, 21)
    pw = ck.PackedWeight(packed, scale, 32)
    g = torch.Generator(device="cuda").manual_seed(rows)
    plain = torch.randn(rows, k, device="cuda", generator=g).to(DT[dtype])
    dy = torch.randn(rows, n, device="cuda", generator=g).to(DT[dtype])
    ref, size = dy.double() @ w, dy.double().abs() @ w.abs()
    tol = HALF_ULP[dtype] * (ref.abs() + 2 * size) + n * 2.0 ** -24 * size + (2.0 ** -24 if dtype == "f16" else 0.0)
    for fn in (pw.matvec, pw.matmul):
        x = plain.clone().requires_grad_()
        y = fn(x)
        assert y.requires_grad and torch.equal(y.detach(), fn(plain))
        y.backward(dy)
        assert x.grad.dtype == x.dtype and bool(((x.grad.double() - ref).abs() <= tol).all())
    x = plain.clone().requires_grad_()
    y = pw.matvec(x[None])
    y.backward(dy[None])
    assert bool(((x.grad.double() - ref).abs() <= tol).all())
    with pytest.raises(RuntimeError, match="autograd"):
        pw.matvec(x, out=torch.empty(rows, n, device="cuda", dtype=x.dtype))
    with torch.no_grad():
        assert not pw.matvec(x).requires_grad


def test_gradient_against_differences():
    """The map is linear: a central difference is the gradient up to rounding (fp32 sums of 64 products below 1)."""
    ck = pkg()
    packed, scale, w = weight(16, 64, 32, "f32", 22)
    pw = ck.PackedWeight(packed, scale, 32)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 64, device="cuda", generator=g, requires_grad=True)
    dy = torch.randn(2, 16, device="cuda", generator=g)
    pw.matvec(x).backward(dy)
    for j in (0, 31, 32, 63):
        e = torch.zeros_like(x)
        e[1, j] = 0.5
        with torch.no_grad():
            diff = float(((pw.matvec(x + e) - pw.matvec(x - e)).double() * dy.double()).sum())
        assert diff == pytest.approx(float(x.grad[1, j]), abs=1e-3)


def test_copies_and_checkpoints():
    """deepcopy, pickle, .to() and a state_dict keep the weight; a state of another weight is refused."""
    import copy
    import io
    ck = pkg()
    g = torch.Generator(device="cuda").manual_seed(30)
    packed, scale, w = weight(40, 96, 32, "f16", 30)
    pw = ck.PackedWeight(packed, scale, 32)
    x = torch.randn(3, 96, device="cuda", generator=g).half()
    want = pw.matvec(x)
    twin = copy.deepcopy(pw)
    assert twin.codes.data_ptr() != pw.codes.data_ptr() and torch.equal(twin.matvec(x), want)
    buf = io.BytesIO()
    torch.save(pw, buf)
    buf.seek(0)
    assert torch.equal(torch.load(buf, weights_only=False).matvec(x), want)
    state = {k: v.clone() if torch.is_tensor(v) else v for k, v in pw.state_dict().items()}
    for assign in (False, True):
        other = ck.PackedWeight(*weight(40, 96, 32, "f16", 31)[:2], 32)
        assert not torch.equal(other.matvec(x), want)
        other.load_state_dict({k: v.clone() if torch.is_tensor(v) else v for k, v in state.items()}, assign=assign)
        assert torch.equal(other.matvec(x), want)
    for bad in (ck.PackedWeight(*weight(40, 96, 32, "bf16", 31)[:2], 32),     # as many bytes, other values
                ck.PackedWeight(*weight(48, 96, 32, "f16", 31)[:2], 32)):
        with pytest.raises((RuntimeError, ValueError), match="PackedWeight"):
            bad.load_state_dict(state)
    away = copy.deepcopy(pw).cpu()
    with pytest.raises(RuntimeError, match="CUDA|expected a tensor on"):
        away.matvec(x)
    with pytest.raises(RuntimeError, match="CUDA|expected a tensor on"):
        away.matvec(x.cpu())
    with pytest.raises(RuntimeError, match="CUDA|expected a tensor on"):
        away.dequantize()
    assert torch.equal(away.cuda().matvec(x), want)
    assert torch.equal(copy.deepcopy(pw).bfloat16().matvec(x), want)      # codes and scales are bytes: no cast


def test_every_nan_of_fp32_stays_one():
    """fp32 NaN whose payload lies in the low half only; infinities stay infinities."""
    ck = pkg()
    packed, scale, w = weight(24, 64, 32, "f32", 42)
    x = torch.randn(4, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    bits = x.view(torch.int32)
    bits[1, 9], bits[2, 9] = 0x7F800001, -(1 << 23) + 1      # 0xFF800001
    y = ck.PackedWeight(packed, scale, 32).matvec(x)
    assert bool(y[1].isnan().all()) and bool(y[2].isnan().all())
    check(y[0::3], x[0::3], w, "f32")


@pytest.mark.parametrize("k,group", [(64, 32), (256, 128), (160, 32)])
def test_low_bits_of_fp32_activations(k, group):
    """Activations 1 and 1 + e 2^-23 under codes c and -c: what is left is c e 2^-23, held in the lowest of the three
    terms of an activation alone.  The codes' products of the upper terms cancel exactly (small integers, adjacent
    channels in one product), so the bound is that of the fp32 sum of what is left."""
    ck = pkg()
    g = torch.Generator(device="cuda").manual_seed(k)
    n, m = 40, 9
    codes = torch.randint(-7, 8, (n, k // 2, 1), device="cuda", generator=g) * torch.tensor([1, -1], device="cuda")
    codes = codes.view(n, k)
    packed = ((codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)).to(torch.uint8)
    scale = 0.5 + torch.rand(n, k // group, device="cuda", generator=g)
    e = torch.randint(0, 128, (m, k // 2), device="cuda", generator=g)
    x = torch.ones(m, k, device="cuda")
    x[:, 0::2] += e * 2.0 ** -23
    w = codes.double() * scale.double().repeat_interleave(group, 1)
    ref = x.double() @ w.T
    size = (x.double() - 1) @ w.abs().T
    err = (ck.PackedWeight(packed, scale, group).matvec(x).double() - ref).abs()
    assert bool((err <= k * 2.0 ** -24 * size).all()), float((err / size).max())


def test_one_row_of_any_stride():
    """A single row's distance to the next is never used: cut from rows of odd length it is one row like any other."""
    ck = pkg()
    for dtype in DT:
        packed, scale, w = weight(20, 64, 32, dtype, 40)
        pw = ck.PackedWeight(packed, scale, 32)
        wide = torch.randn(4, 67, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(DT[dtype])
        for x in (wide[:1, :64], wide[1:2, 3:], wide[None, 2:3, 1:65], wide.t()[:64].t()[3:]):
            check(pw.matvec(x), x, w, dtype)


@pytest.mark.parametrize("dtype,rows", [("f32", 8 * 65535 + 21), ("f16", 16 * 65535 + 37)])
def test_more_rows_than_one_launch_takes(dtype, rows):
    ck = pkg()
    packed, scale, w = weight(5, 32, 32, dtype, 41)
    x = torch.randn(rows, 32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(DT[dtype])
    check(ck.PackedWeight(packed, scale, 32).matvec(x), x, w, dtype)


def test_results_repeat_and_run_in_a_graph():
    ck = pkg()
    for n, k, m in ((250, 768, 3), (3001, 2912, 40), (8209, 4128, 20)):
        packed, scale, w = weight(n, k, 32, "bf16", 50)
        pw = ck.PackedWeight(packed, scale, 32)
        x = torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
        want = pw.matvec(x)
        for _ in range(20):
            assert torch.equal(pw.matvec(x), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pw.matvec(x)
        graph.replay()
        assert torch.equal(y, want)
