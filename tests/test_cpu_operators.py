"""Host side of the decode-step operators, no GPU: packed argument structures,
argument checks of the C entries, layout sizes, rotary frequencies."""

import ctypes
import math
import os
import re

import pytest
import torch

from conftest import ROOT, load_pkg


def lib():
    pkg = load_pkg()
    return pkg, pkg._lib.load()


def test_packed_structures_match_the_header():
    """The one-call packers write the bytes of the ctypes structures, whose fields follow the header."""
    pkg, _ = lib()
    L = pkg._lib
    r = L.Rotary()
    vals = dict(freq=3, positions=4, position_bytes=8, batch=2, tokens=5, head_dim=64, rotary_dim=32, interleaved=1,
                inverse=0, factor=1.5, dtype=2)
    for k, v in vals.items():
        setattr(r, k, v)
    r.position_stride[0], r.position_stride[1] = 7, 1
    rows = ((11, 12, 1, 2, 3, 4, 5, 6, 9), (21, 22, 10, 20, 30, 40, 50, 60, 8))
    for dst, x in zip((r.q, r.k), rows):
        dst.in_, dst.out, dst.heads = x[0], x[1], x[8]
        for i in range(3):
            dst.in_stride[i], dst.out_stride[i] = x[2 + i], x[5 + i]
    got = L.ROTARY_PACK(*rows[0], *rows[1], 3, 4, 7, 1, 8, 2, 5, 64, 32, True, False, 1.5, 2)
    assert got == bytes(r)
    p = L.Prefix()
    p.k, p.v, p.num_kv_heads, p.tokens, p.head_dim, p.dtype = 1, 2, 8, 100, 64, 1
    for i in range(2):
        p.k_stride[i], p.v_stride[i] = 10 + i, 20 + i
    assert L.PREFIX_PACK(1, 2, 10, 11, 20, 21, 8, 100, 64, 1) == bytes(p)
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "carekv_b200.h")).read(), flags=re.S)
    for name, cls in (("carekv_rows", L.Rows), ("carekv_rotary", L.Rotary), ("carekv_w4", L.W4),
                      ("carekv_prefix", L.Prefix)):
        body = src[src.index(f"typedef struct {name} {{") + len(f"typedef struct {name} {{"):src.index(f"}} {name}_t;")]
        fields = [re.sub(r"\[\d+\]|\*", "", f).strip() for line in body.split(";") if line.strip()
                  for f in re.sub(r"^\s*(const\s+)?\w+\s", "", line.strip()).split(",")]
        assert fields == [f.rstrip("_") for f, _ in cls._fields_], name


def test_rotary_refusals():
    pkg, l = lib()
    ok = dict(q=(16, 32, 0, 1, 1, 0, 1, 1, 1), k=(0,) * 9, freq=1, positions=1, pb=8, batch=0, tokens=0, D=64, rd=64,
              dt=0)

    def call(**kw):
        a = dict(ok, **kw)
        return l.carekv_rotary(pkg._lib.ROTARY_PACK(*a["q"], *a["k"], a["freq"], a["positions"], 0, 1, a["pb"],
                                                    a["batch"], a["tokens"], a["D"], a["rd"], 0, 0, 1.0, a["dt"]), None)
    assert call() == 0                       # no tokens: nothing to do
    assert call(rd=63) == 1 and call(rd=66) == 1 and call(rd=0) == 1
    assert call(D=512, rd=64) == 2
    assert call(pb=2) == 1 and call(dt=7) == 1 and call(freq=0) == 1
    assert call(batch=1, tokens=1, positions=0) == 1
    assert call(batch=1, tokens=1, q=(16, 16, 0, 1, 1, 0, 1, 1, 1)) == 1      # in place
    assert call(batch=1 << 20, tokens=1 << 20) == 2


def test_w4_layout_and_refusals():
    pkg, l = lib()
    w = pkg._lib.W4()
    sizes = (ctypes.c_size_t * 2)()

    def layout(n, k, g, dt=1):
        w.n, w.k, w.group_size, w.dtype = n, k, g, dt
        return l.carekv_w4_layout(ctypes.byref(w), sizes)
    assert layout(4096, 4096, 32) == 0 and list(sizes) == [4096 * 2048, 4096 * 128 * 2]
    # rows padded to 128, channels to 128
    assert layout(130, 96, 32) == 0 and list(sizes) == [256 * 64, 256 * 4 * 2]
    assert layout(16, 256, 256, 0) == 0 and list(sizes) == [128 * 128, 128 * 2 * 4]
    assert layout(16, 100, 32) == 1 and layout(0, 64, 32) == 1 and layout(16, 64, 16) == 2
    assert layout(16, 192, 96) == 2 and layout(16, 128, 32, 5) == 1
    layout(16, 128, 32)
    assert l.carekv_w4_matvec(ctypes.byref(w), 16, 128, 1, 16, None) == 1     # no buffers
    w.codes, w.scales = 1 << 16, (1 << 16) + 16
    assert l.carekv_w4_matvec(ctypes.byref(w), 16, 128, 1, 16, None) == 1     # misaligned scales
    w.scales = 1 << 17
    assert l.carekv_w4_matvec(ctypes.byref(w), 16, 128, 0, 16, None) == 0     # no rows
    assert l.carekv_w4_matvec(ctypes.byref(w), 16, 127, 1, 16, None) == 1     # rows overlap
    assert l.carekv_w4_matvec(ctypes.byref(w), 18, 128, 1, 16, None) == 1     # misaligned rows
    assert l.carekv_w4_matvec(ctypes.byref(w), None, 128, 1, 16, None) == 1


def test_prefix_refusals_and_workspace():
    pkg, l = lib()
    n = ctypes.c_size_t(0)

    def ws(hkv=2, tokens=100, d=64, dt=1, rows=4, heads=8):
        return l.carekv_prefix_workspace_bytes(pkg._lib.PREFIX_PACK(0, 0, 0, 0, 0, 0, hkv, tokens, d, dt), rows, heads,
                                               ctypes.byref(n))
    assert ws() == 0 and n.value > 0
    assert ws(tokens=0) == 0 and ws(rows=0) == 0
    assert ws(heads=7) == 1 and ws(hkv=0) == 1 and ws(tokens=-1) == 1 and ws(dt=9) == 1
    assert ws(d=300) == 2 and ws(rows=1 << 30, heads=8) == 2 and ws(tokens=(1 << 30) + 1) == 2

    def call(scale=1.0, q=16, out=16, tail=None, tl=None, ws_=256, nb=1 << 30, k=16):
        return l.carekv_prefix_attention(pkg._lib.PREFIX_PACK(k, k, 0, 64, 0, 64, 2, 100, 64, 1), q, 512, 64, 4, 8, scale,
                                         None, tail, tl, out, None, ws_, nb, None)
    assert call(scale=0.0) == 1 and call(scale=-1.0) == 1 and call(scale=float("nan")) == 1
    assert call(q=None) == 1 and call(out=None) == 1 and call(k=0) == 1
    assert call(tail=16) == 1 and call(tl=16) == 1 and call(ws_=None) == 1 and call(ws_=8) == 1
    assert call(nb=16) == 5
    assert l.carekv_prefix_attention(pkg._lib.PREFIX_PACK(16, 16, 0, 64, 0, 64, 2, 100, 64, 1), 16, 512, 64, 0, 8, 1.0,
                                     None, None, None, 16, None, None, 0, None) == 0      # no rows


@pytest.mark.parametrize("rd", [2, 64, 128, 6])
def test_frequencies(rd):
    pkg, _ = lib()
    f, a = pkg.rotary_frequencies(rd)
    want = 10000.0 ** (-2 * torch.arange(rd // 2, dtype=torch.float64) / rd) / (2 * math.pi)
    assert a == 1.0 and f.dtype == torch.int64
    assert float((f.double() / 2.0 ** 64 / want - 1).abs().max()) < 1e-15
    # a quarter turn of the fastest pair, exactly, at a far position
    assert (int(f[0]) * (1 << 40)) % (1 << 64) == ((int(f[0]) << 40) & ((1 << 64) - 1))


def test_prefix_object_without_a_gpu():
    pkg, _ = lib()
    sp = pkg.SharedPrefix(2)
    with pytest.raises(ValueError, match="must match"):
        sp.set(0, torch.zeros(2, 5, 8), torch.zeros(2, 6, 8))
    sp.set(0, torch.zeros(2, 5, 8), torch.zeros(2, 5, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        sp.attend(0, torch.zeros(1, 2, 8))


def test_overlap_of_strided_tensors():
    """overlap / interleaved / meets_itself against the sets of elements, on views of one small buffer."""
    import itertools
    import random
    pkg, _ = lib()
    T = pkg._tensors
    buf = torch.zeros(200, dtype=torch.float16)
    rng = random.Random(3)
    views = []
    for _ in range(150):
        shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 3))]
        stride = [rng.choice((0, 1, 2, 3, 4, 6, 8, 12, 16, 24)) for _ in shape]
        views.append(buf.as_strided(shape, stride, rng.randint(0, 60)))
    for base in (buf[:96].view(2, 6, 8), buf[:96].view(2, 3, 4, 4)):     # slices of fused buffers
        for d in range(1, base.dim()):
            for i in range(base.shape[d] + 1):
                views += [base.narrow(d, 0, i), base.narrow(d, i, base.shape[d] - i)]

    def elements(t):
        return [t.storage_offset() + sum(i * s for i, s in zip(x, t.stride()))
                for x in itertools.product(*(range(n) for n in t.shape))]
    sets = [set(elements(t)) for t in views]
    for a, sa in zip(views, sets):
        if a.numel() and not T.meets_itself(a):
            assert len(sa) == a.numel()
        for b, sb in zip(views, sets):
            if not sa.isdisjoint(sb):
                assert T.overlap(a, b) and not T.interleaved(a, b)
    fused = buf[:96].view(2, 6, 8)
    for d, i in ((1, 2), (2, 3)):
        a, b = fused.narrow(d, 0, i), fused.narrow(d, i, fused.shape[d] - i)
        assert T.overlap(a, b) and T.interleaved(a, b) and T.interleaved(b, a)
    assert not T.meets_itself(fused) and T.meets_itself(fused[:1].expand(3, 6, 8))
    assert not T.overlap(buf[:10], buf[10:20]) and not T.overlap(buf[:0], buf)


def test_prefix_layers_set_anew():
    pkg, _ = lib()
    sp = pkg.SharedPrefix(2)
    k = torch.ones(2, 5, 8)
    sp.set(1, k, k)
    sp.set(-1, k[:, :3], k[:, :3])          # the same layer, alone so far: another length
    assert sp.tokens == 3 and sp.layer(1)[0].is_contiguous()
    k.zero_()
    assert bool((sp.layer(1)[0] == 1).all())
    with pytest.raises(ValueError, match="the others 3"):
        sp.set(0, k, k)
    with pytest.raises(IndexError):
        sp.set(2, k[:, :3], k[:, :3])


def test_sizes_beyond_the_row_counters():
    """Sizes whose last tile would pass a 32-bit row counter are refused before any launch."""
    pkg, l = lib()
    most = 2 ** 31 - 1

    def rotary(tokens, heads):
        rows = (16, 32, 0, 1, 1, 0, 1, 1)
        return l.carekv_rotary(pkg._lib.ROTARY_PACK(*rows, heads, *rows, 1, 16, 16, 0, 1, 8, 1, tokens, 2, 2, 0, 0, 1.0,
                                                    1), None)
    assert rotary(most, 1) == 2 and rotary(most - 1000, 1) == 2
    assert rotary(1, most) == 2 and rotary(1, most - 1) == 2
    w, sizes = pkg._lib.W4(), (ctypes.c_size_t * 2)()
    for n, k in ((most, 32), (most - 1000, 32), (1, 2 ** 31 - 128)):
        w.n, w.k, w.group_size, w.dtype = n, k, 32, 1
        assert l.carekv_w4_layout(ctypes.byref(w), sizes) == 2
    need = ctypes.c_size_t(0)
    for rows, heads in ((most, 1), (1 << 30, 2), (most - 1000, 1)):
        assert l.carekv_prefix_workspace_bytes(pkg._lib.PREFIX_PACK(0, 0, 0, 0, 0, 0, 1, 100, 64, 1), rows, heads,
                                               ctypes.byref(need)) == 2
