"""The cache's decode attention with its log-sum-exp, merged with a shared
prefix, and a layer step that runs 4-bit projections, rotary positions and the
prefix together (GPU)."""

import math
import zlib

import numpy as np
import pytest
import torch

import oracle
from conftest import load_pkg
from helpers import PAPER_BEST_ENV, env, oracle_cache_for, oracle_selection, route_cfg_from

pytestmark = pytest.mark.gpu

TDT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# attention outputs: the decode path's own tolerances (test_gpu_decode.py)
TOL = {"fp32": (1e-3, 2e-3), "fp16": (3e-3, 3e-3), "bf16": (1e-2, 1e-2)}
# a log-sum-exp moves by at most the largest error of a logit; fp32 logits of
# D products of up to ~60 x 4 are off by D 2^-24 240 < 2e-3
LSE_TOL = 2e-3


@pytest.fixture(scope="module")
def pkg():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_pkg()


def build(pkg, D, bits, g, Hq, Hkv, dt, lens, seed, **kw):
    cfg = pkg.CacheConfig(num_layers=1, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, page_size=16,
                          max_pages=max(lens) // 16 + 3, base_bits=bits, group_size=g, scale_quant="int8",
                          packed_base=True, store_budget_mode="absolute", store_abs_k=2, store_abs_v=2,
                          route_policy="joint", store_sketch=False, **kw)
    cache = pkg.CAREKVCache(cfg, torch.device("cuda"), batch=len(lens))
    eng = pkg.DecodeEngine(cache)
    rng = np.random.default_rng(seed)
    seqs = []
    for b, T in enumerate(lens):
        oc = oracle_cache_for(cfg)
        if T:
            K = rng.standard_normal((Hkv, T, D)).astype(np.float32)
            K[:, :, :4] *= 20.0
            V = rng.standard_normal((Hkv, T, D)).astype(np.float32)
            K, V = oracle.round_to(K, dt), oracle.round_to(V, dt)
            eng.prefill_store(0, torch.from_numpy(K).cuda().to(TDT[dt])[None],
                              torch.from_numpy(V).cuda().to(TDT[dt])[None], seq_begin=b)
            for h in range(Hkv):
                oc.prefill_write(0, h, K[h], V[h], dt)
        seqs.append(oc)
    q = oracle.round_to(rng.standard_normal((len(lens), Hq, D)).astype(np.float32), dt)
    return cfg, cache, eng, seqs, q


CASES = [
    # name, D, bits, g, Hq, Hkv, dt, lengths, correction mode or None (no correction)
    ("base_mha", 128, 3, 32, 4, 4, "fp32", (90, 17, 0), None),
    ("exact_mha", 128, 3, 32, 4, 4, "fp32", (150, 33, 0), "exact"),
    ("exact_gqa4_int2", 128, 2, 32, 8, 2, "fp32", (64, 40), "exact"),
    ("exact_gqa8_d64", 64, 3, 32, 16, 2, "fp16", (77, 130), "exact"),
    ("linear_gqa2_int4", 64, 4, 64, 4, 2, "fp32", (50, 96), "linear"),
    ("exact_bf16", 128, 3, 32, 4, 4, "bf16", (100, 64), "exact"),
]


@pytest.mark.parametrize("case", CASES, ids=[c[0] for c in CASES])
def test_log_sum_exp_matches_oracle(pkg, case):
    """lse = log sum e^(logit), e^(logit + ds) under the exact correction; -inf for an empty sequence."""
    name, D, bits, g, Hq, Hkv, dt, lens, mode = case
    grp = Hq // Hkv
    with env(**dict(PAPER_BEST_ENV, CAREKV_K_CORRECTION_MODE=mode or "exact")):
        cfg, cache, eng, seqs, q = build(pkg, D, bits, g, Hq, Hkv, dt, lens, zlib.crc32(name.encode()),
                                         read_budget_mode="absolute", read_abs_k=2, read_abs_v=2)
        qt = torch.from_numpy(q).cuda().to(TDT[dt])
        plain = eng.attend(0, qt, correction=mode is not None)
        out, lse = eng.attend(0, qt, correction=mode is not None, return_lse=True)
        assert torch.equal(out, plain)       # asking for it changes nothing
        pages = max(eng._pages(b, 0) for b in range(len(lens)))
        sel = eng.last_selection(0, 0, len(lens), pages) if mode else None
        rc = route_cfg_from(cfg)
        lse = lse.double().cpu().numpy()
        checked = 0
        for b, oc in enumerate(seqs):
            for h in range(Hkv):
                rows = slice(h * grp, (h + 1) * grp)
                if lens[b] == 0:
                    assert np.all(np.isneginf(lse[b, rows]))
                    continue
                _, info = oracle.decode_attention_kvh(oc, 0, h, q[b, rows], rc, correction=mode is not None)
                S = info["S"].astype(np.float64)
                if mode == "exact":
                    want_sel = oracle_selection(info, grp)
                    for si, e in enumerate(info["k_index"]):
                        c0 = e["cg"] * cfg.k_channel_group
                        ds = q[b, rows][:, c0:c0 + cfg.k_channel_group].astype(np.float64) @ e["R"].T / math.sqrt(D)
                        S[:, e["pstart"]:e["pstart"] + e["nvalid"]] += info["sel_k"][:, si, None] * ds
                for i in range(grp):
                    if mode == "exact" and sorted(sel[(b, h, i)]) != want_sel[i]:
                        continue     # a tie within rounding: another, equally good set of slots
                    m = S[i].max()
                    want = m + math.log(np.exp(S[i] - m).sum())
                    assert abs(lse[b, h * grp + i] - want) <= LSE_TOL + 1e-5 * abs(want), (b, h, i)
                    checked += 1
        assert checked >= 0.9 * Hq * sum(1 for n in lens if n)
        cache.check_errors()


@pytest.mark.parametrize("dt,D,Hq,Hkv", [("fp32", 128, 8, 2), ("fp16", 64, 16, 2), ("bf16", 128, 4, 4)])
def test_prefix_and_cache_equal_one_softmax(pkg, dt, D, Hq, Hkv):
    """attend(prefix=...) = one softmax over the prefix's and the cache's (dequantized) tokens."""
    with env(**PAPER_BEST_ENV):
        lens = (70, 5, 0, 33)
        cfg, cache, eng, seqs, q = build(pkg, D, 3, 32, Hq, Hkv, dt, lens, 7, read_budget_mode="absolute",
                                         read_abs_k=0, read_abs_v=0)
        N, grp = 300, Hq // Hkv
        g = torch.Generator(device="cuda").manual_seed(1)
        kp = torch.randn(Hkv, N, D, device="cuda", generator=g).to(TDT[dt])
        vp = torch.randn(Hkv, N, D, device="cuda", generator=g).to(TDT[dt])
        sp = pkg.SharedPrefix(1)
        sp.set(0, kp, vp)
        qt = torch.from_numpy(q).cuda().to(TDT[dt])
        out, lse = eng.attend(0, qt, prefix=sp, return_lse=True)
        assert torch.equal(out, eng.attend(0, qt, prefix=sp))
        rt, at = TOL[dt]
        for b, oc in enumerate(seqs):
            for h in range(Hkv):
                K, V = kp[h].double().cpu().numpy(), vp[h].double().cpu().numpy()
                if lens[b]:
                    Kh, Vh, _ = oc.read_base_concat(0, h)
                    K, V = np.concatenate([K, Kh]), np.concatenate([V, Vh])
                S = q[b, h * grp:(h + 1) * grp].astype(np.float64) @ K.T / math.sqrt(D)
                m = S.max(1, keepdims=True)
                P = np.exp(S - m)
                O = P @ V / P.sum(1, keepdims=True)
                np.testing.assert_allclose(out[b, h * grp:(h + 1) * grp].double().cpu().numpy(), O, rtol=rt, atol=at)
                np.testing.assert_allclose(lse[b, h * grp:(h + 1) * grp].cpu().numpy(), m[:, 0] + np.log(P.sum(1)),
                                           rtol=1e-5, atol=LSE_TOL)


def test_prefix_on_a_kv_head_shard(pkg):
    """Two arenas with one kv head each give the rows of the unsharded call."""
    with env(**PAPER_BEST_ENV):
        D, Hq, Hkv, T = 64, 4, 2, 50
        kw = dict(num_layers=1, head_dim=D, max_pages=8, base_bits=3, group_size=32, scale_quant="int8",
                  packed_base=True, store_budget_mode="absolute", store_abs_k=1, store_abs_v=1,
                  read_budget_mode="absolute", read_abs_k=1, read_abs_v=1, route_policy="joint", store_sketch=False)
        g = torch.Generator(device="cuda").manual_seed(2)
        K, V = (torch.randn(1, Hkv, T, D, device="cuda", generator=g).half() for _ in range(2))
        kp, vp = (torch.randn(Hkv, 200, D, device="cuda", generator=g).half() for _ in range(2))
        q = torch.randn(1, Hq, D, device="cuda", generator=g).half()

        def run(h0, n, shard):
            cfg = pkg.CacheConfig(num_heads=n * Hq // Hkv, num_kv_heads=n, **kw)
            eng = pkg.DecodeEngine(pkg.CAREKVCache(cfg, torch.device("cuda"), batch=1), shard=shard)
            eng.prefill_store(0, K, V)
            sp = pkg.SharedPrefix(1)
            sp.set(0, kp[h0:h0 + n], vp[h0:h0 + n])
            return eng.attend(0, q, prefix=sp, return_lse=True)
        whole, wl = run(0, 2, None)
        for h in range(2):
            part, pl = run(h, 1, (h, 2))
            assert torch.equal(part[:, 2 * h:2 * h + 2], whole[:, 2 * h:2 * h + 2])
            assert torch.equal(pl[:, 2 * h:2 * h + 2], wl[:, 2 * h:2 * h + 2])


def rotated(x, positions, freq):
    """x [..., T, H, D] float64, half layout."""
    half = freq.numel()
    ang = positions.double().unsqueeze(-1) * (freq.double() * (2 * math.pi / 2.0 ** 64))
    c, s = torch.cos(ang).unsqueeze(-2), torch.sin(ang).unsqueeze(-2)
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * c - b * s, a * s + b * c, x[..., 2 * half:]), -1)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_layer_step_with_4bit_weights_rotary_and_prefix(pkg, dt):
    """Prefill and decode of a layer against the same mathematics in fp64 over the weights and the
    cache contents that the layer holds."""
    Hq, Hkv, D, dm, N, T, steps, B = 8, 2, 64, 96, 150, 21, 3, 3
    g = torch.Generator(device="cuda").manual_seed(3)

    def rand(*s):
        return torch.randn(*s, device="cuda", generator=g)
    with env(CAREKV_PREFILL_MODE="fp", **PAPER_BEST_ENV):
        cfg = pkg.CacheConfig(num_layers=1, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, max_pages=4, base_bits=4,
                              group_size=32, scale_quant="int8", packed_base=True, store_budget_mode="absolute",
                              store_abs_k=1, store_abs_v=1, read_budget_mode="absolute", read_abs_k=0, read_abs_v=0,
                              route_policy="joint", store_sketch=False)
        ws = [(rand(o, i) / math.sqrt(i)).to(TDT[dt]) for o, i in ((Hq * D, dm), (Hkv * D, dm), (Hkv * D, dm),
                                                                  (dm, Hq * D))]
        layer = pkg.CAREKVLayer(cfg, 0, *ws, torch.device("cuda")).quantize_weights(32)
        wq, wk, wv, wo = (layer._packed[n].dequantize().double() for n in ("W_Q", "W_K", "W_V", "W_O"))
        layer.rotary = pkg.RotaryEmbedding(D, device="cuda")
        sp = pkg.SharedPrefix(1)
        sp.set(0, rand(Hkv, N, D).to(TDT[dt]), rand(Hkv, N, D).to(TDT[dt]))
        kp, vp = (x.double().repeat_interleave(Hq // Hkv, 0) for x in sp.layer(0))
        cache = pkg.CAREKVCache(cfg, torch.device("cuda"), batch=B)
        hid = rand(B, T + steps, dm).to(TDT[dt])
        pos = N + torch.arange(T + steps, device="cuda")
        pre = layer.prefill_batch(cache, hid[:, :T], positions=pos[:T], prefix=sp)

        def qkv(x, p):
            x = x.double()
            r = [(x @ w.T).view(*x.shape[:-1], -1, D) for w in (wq, wk, wv)]
            return rotated(r[0], p, layer.rotary.freq), rotated(r[1], p, layer.rotary.freq), r[2]

        def attend(q, k, v, own_mask=None):      # q [Hq, n, D]; k, v [Hkv, m, D] of the own tokens
            k, v = (x.repeat_interleave(Hq // Hkv, 0) for x in (k, v))
            s = q @ torch.cat((kp, k), 1).transpose(1, 2) / math.sqrt(D)
            if own_mask is not None:
                s[..., N:] = s[..., N:].masked_fill(own_mask, -math.inf)
            return torch.softmax(s, -1) @ torch.cat((vp, v), 1)
        rt, at = {"fp32": (1e-3, 2e-3), "fp16": (1e-2, 1e-2)}[dt]
        causal = torch.triu(torch.ones(T, T, dtype=torch.bool, device="cuda"), 1)
        for b in range(B):
            q, k, v = (x.transpose(0, 1) for x in qkv(hid[b, :T], pos[:T]))
            want = attend(q, k, v, causal).transpose(0, 1).reshape(T, -1) @ wo.T
            np.testing.assert_allclose(pre[b].double().cpu(), want.cpu(), rtol=rt, atol=at)
        for j in range(T, T + steps):
            got = layer.decode_step_batch(cache, hid[:, j], positions=pos[j].expand(B), prefix=sp)
            for b in range(B):
                q, _, _ = qkv(hid[b, j:j + 1], pos[j:j + 1])
                kc, ks, vc, vs = [], [], [], []
                for h in range(Hkv):
                    a = cache.read_base_concat(0, h, seq=b)
                    kc.append(a[0].double() * a[1].double().repeat_interleave(32, 1))
                    vc.append(a[2].double() * a[3].double().repeat_interleave(32, 1))
                want = attend(q.transpose(0, 1), torch.stack(kc), torch.stack(vc)).reshape(1, -1) @ wo.T
                np.testing.assert_allclose(got[b:b + 1].double().cpu(), want.cpu(), rtol=rt, atol=at)
        cache.check_errors()


def test_layer_refusals(pkg):
    with env(CAREKV_PREFILL_MODE="carekv_stored", **PAPER_BEST_ENV):
        cfg = pkg.CacheConfig(num_layers=1, num_heads=2, num_kv_heads=2, head_dim=64, max_pages=4, base_bits=3,
                              group_size=32, scale_quant="int8", store_budget_mode="absolute", store_abs_k=1,
                              store_abs_v=1, read_budget_mode="absolute", read_abs_k=1, read_abs_v=1)
        W = torch.randn(128, 64, device="cuda")
        layer = pkg.CAREKVLayer(cfg, 0, W, W, W, W.T.contiguous(), torch.device("cuda"))
        cache = pkg.CAREKVCache(cfg, torch.device("cuda"), batch=1)
        sp = pkg.SharedPrefix(1)
        sp.set(0, torch.randn(2, 20, 64, device="cuda"), torch.randn(2, 20, 64, device="cuda"))
        hid = torch.randn(1, 5, 64, device="cuda")
        with pytest.raises(NotImplementedError, match="prefix"):
            layer.prefill_batch(cache, hid, prefix=sp)
        with pytest.raises(ValueError, match="rotary"):
            layer.prefill_batch(cache, hid, positions=torch.arange(5, device="cuda"))
        with pytest.raises(ValueError, match="has not been set"):
            pkg.SharedPrefix(1).attend(0, torch.randn(1, 2, 64, device="cuda"))


def test_decode_attention_carries_no_graph(pkg):
    """attend() answers alike whether its queries require a gradient, with and without a prefix."""
    with env(**PAPER_BEST_ENV):
        cfg, cache, eng, seqs, q = build(pkg, 64, 3, 32, 4, 2, "fp32", (20, 5), 3, read_budget_mode="absolute",
                                         read_abs_k=1, read_abs_v=1)
        sp = pkg.SharedPrefix(1)
        sp.set(0, torch.randn(2, 50, 64, device="cuda"), torch.randn(2, 50, 64, device="cuda"))
        qt = torch.from_numpy(q).cuda()
        for kw in ({}, dict(prefix=sp)):
            got = eng.attend(0, qt.clone().requires_grad_(), **kw)
            assert not got.requires_grad and torch.equal(got, eng.attend(0, qt, **kw))


def test_layer_calls_with_inputs_that_require_a_gradient(pkg):
    """Prefill by positions passes the gradient that prefill by tables passes; with a prefix, whose attention has no
    backward pass, it refuses.  Decode steps answer as without a gradient, as they do without positions or a prefix."""
    with env(CAREKV_PREFILL_MODE="fp", **PAPER_BEST_ENV):
        Hq, Hkv, D, dm, N, T = 4, 2, 64, 96, 40, 9
        cfg = pkg.CacheConfig(num_layers=1, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, max_pages=4, base_bits=4,
                              group_size=32, scale_quant="int8", packed_base=True, store_budget_mode="absolute",
                              store_abs_k=1, store_abs_v=1, read_budget_mode="absolute", read_abs_k=1, read_abs_v=1,
                              route_policy="joint", store_sketch=False)
        g = torch.Generator(device="cuda").manual_seed(3)
        ws = [torch.randn(o, i, device="cuda", generator=g) / math.sqrt(i)
              for o, i in ((Hq * D, dm), (Hkv * D, dm), (Hkv * D, dm), (dm, Hq * D))]
        layer = pkg.CAREKVLayer(cfg, 0, *ws, torch.device("cuda"))
        layer.rotary = pkg.RotaryEmbedding(D, device="cuda")
        sp = pkg.SharedPrefix(1)
        sp.set(0, *(torch.randn(Hkv, N, D, device="cuda", generator=g) for _ in range(2)))
        hid = torch.randn(1, T, dm, device="cuda", generator=g)
        pos = torch.arange(T, device="cuda")
        ang = pos.double().unsqueeze(-1) * (layer.rotary.freq.double() * (2 * math.pi / 2.0 ** 64))
        tables = tuple(torch.cat((f(ang), f(ang)), -1).float()[None] for f in (torch.cos, torch.sin))
        grads = []
        for kw in (dict(position_embeddings=tables), dict(positions=pos)):
            x = hid.clone().requires_grad_()
            cache = pkg.CAREKVCache(cfg, torch.device("cuda"), batch=1)
            layer.prefill_batch(cache, x, **kw).square().sum().backward()
            grads.append(x.grad)
        torch.testing.assert_close(grads[1], grads[0], rtol=1e-3, atol=1e-3 * float(grads[0].abs().max()))
        x = hid.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="backward"):
            layer.prefill_batch(pkg.CAREKVCache(cfg, torch.device("cuda"), batch=1), x, positions=N + pos, prefix=sp)
        outs = []
        for grad in (False, True):
            cache = pkg.CAREKVCache(cfg, torch.device("cuda"), batch=1)
            with torch.no_grad():
                layer.prefill_batch(cache, hid, positions=N + pos, prefix=sp)
            step = hid[:, 0].clone().requires_grad_(grad)
            outs.append(layer.decode_step_batch(cache, step, positions=N + pos[-1:] + 1, prefix=sp))
        assert torch.equal(outs[0], outs[1])


def test_quantized_layer_is_copied_saved_and_moved(pkg):
    """quantize_weights() loses nothing: a state_dict holds the 4-bit weights, copies and moves keep them, and a layer
    whose weights cannot all be quantized stays as it was."""
    import copy
    Hq, Hkv, D, dm = 4, 2, 64, 96
    cfg = pkg.CacheConfig(num_layers=1, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, max_pages=4, base_bits=4,
                          group_size=32, scale_quant="int8", packed_base=True, store_budget_mode="absolute",
                          store_abs_k=1, store_abs_v=1, read_budget_mode="absolute", read_abs_k=1, read_abs_v=1,
                          route_policy="joint", store_sketch=False)
    g = torch.Generator(device="cuda").manual_seed(4)

    def make(out=dm):
        ws = [torch.randn(o, i, device="cuda", generator=g) / math.sqrt(i)
              for o, i in ((Hq * D, dm), (Hkv * D, dm), (Hkv * D, dm), (out, Hq * D))]
        return pkg.CAREKVLayer(cfg, 0, *ws, torch.device("cuda"))
    layer = make().quantize_weights(32)
    layer.rotary = pkg.RotaryEmbedding(D, device="cuda")
    hid = torch.randn(1, 6, dm, device="cuda", generator=g)
    pos = torch.arange(6, device="cuda")

    def run(l):
        with env(CAREKV_PREFILL_MODE="fp", **PAPER_BEST_ENV):
            return l.prefill_batch(pkg.CAREKVCache(cfg, torch.device("cuda"), batch=1), hid, positions=pos)
    want = run(layer)
    assert torch.equal(run(copy.deepcopy(layer)), want)
    state = copy.deepcopy(layer.state_dict())
    other = make().quantize_weights(32)
    other.rotary = layer.rotary
    assert not torch.equal(run(other), want)
    other.load_state_dict(state)
    assert torch.equal(run(other), want)
    moved = copy.deepcopy(layer).cpu()
    assert moved.rotary.freq.device.type == "cpu"
    assert torch.equal(run(moved.cuda()), want)
    assert torch.equal(run(layer), want)
    odd = make()
    odd.W_O = torch.nn.Parameter(torch.randn(dm, Hq * D + 16, device="cuda"), requires_grad=False)
    with pytest.raises(Exception):
        odd.quantize_weights(32)
    assert all(getattr(odd, n) is not None for n in ("W_Q", "W_K", "W_V", "W_O"))
    dense = make()
    assert set(dense.state_dict()) == {"W_Q", "W_K", "W_V", "W_O"}


def test_prefix_that_does_not_fit_the_cache_is_refused(pkg):
    """A prefix of other kv heads, head size or type than the arena's is an error before anything is written."""
    with env(**PAPER_BEST_ENV):
        cfg, cache, eng, seqs, q = build(pkg, 64, 3, 32, 8, 4, "fp16", (20, 5), 3, read_budget_mode="absolute",
                                         read_abs_k=1, read_abs_v=1)
        qt = torch.from_numpy(q).cuda().half()
        out = torch.full_like(qt, 7.0)

        def prefix(h, d, dt):
            sp = pkg.SharedPrefix(1)
            sp.set(0, torch.randn(h, 50, d, device="cuda").to(dt), torch.randn(h, 50, d, device="cuda").to(dt))
            return sp
        for sp in (prefix(2, 64, torch.float16), prefix(8, 64, torch.float16), prefix(4, 128, torch.float16),
                   prefix(4, 64, torch.bfloat16), pkg.SharedPrefix(1)):
            with pytest.raises(ValueError, match="prefix|SharedPrefix"):
                eng.attend(0, qt, out=out, prefix=sp)
        assert bool((out == 7.0).all())
        eng.attend(0, qt, out=out, prefix=prefix(4, 64, torch.float16))


def test_layer_calls_refuse_a_prefix_before_the_cache_is_written(pkg):
    with env(CAREKV_PREFILL_MODE="fp", **PAPER_BEST_ENV):
        cfg = pkg.CacheConfig(num_layers=1, num_heads=4, num_kv_heads=4, head_dim=64, max_pages=4, base_bits=3,
                              group_size=32, scale_quant="int8", store_budget_mode="absolute", store_abs_k=1,
                              store_abs_v=1, read_budget_mode="absolute", read_abs_k=1, read_abs_v=1)
        W = torch.randn(256, 64, device="cuda")
        layer = pkg.CAREKVLayer(cfg, 0, W, W, W, W.T.contiguous(), torch.device("cuda"))
        cache = pkg.CAREKVCache(cfg, torch.device("cuda"), batch=1)
        sp = pkg.SharedPrefix(1)
        sp.set(0, torch.randn(2, 20, 64, device="cuda"), torch.randn(2, 20, 64, device="cuda"))
        hid = torch.randn(1, 5, 64, device="cuda")
        with pytest.raises(ValueError, match="SharedPrefix"):
            layer.prefill_batch(cache, hid, prefix=sp)
        with pytest.raises(ValueError, match="SharedPrefix"):
            layer.decode_step_batch(cache, hid[:, 0], prefix=sp)
        assert cache.total_valid_tokens(0, 0) == 0


@pytest.mark.parametrize("mode", ["exact", "linear"])
def test_log_sum_exp_of_the_cached_router(pkg, mode):
    """The router of the reference's decode step: base sum under the linear correction, shifted logits under the exact."""
    from oracle.legacy_router import legacy_correction
    from oracle import unpack_4bit
    D, Hq, Hkv, T = 64, 4, 2, 150
    grp = Hq // Hkv
    with env(**dict(PAPER_BEST_ENV, CAREKV_K_CORRECTION_MODE=mode, CAREKV_KSCORE_LIVE="0")):
        cfg = pkg.CacheConfig(num_layers=1, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, max_pages=T // 16 + 4,
                              base_bits=3, group_size=32, scale_quant="int8", store_budget_mode="absolute",
                              store_abs_k=2, store_abs_v=2, read_budget_mode="absolute", read_abs_k=2, read_abs_v=2,
                              route_policy="joint", sketch_dim=32, correction_impl="cached")
        cache = pkg.CAREKVCache(cfg, torch.device("cuda"), batch=1)
        eng = pkg.DecodeEngine(cache)
        rng = np.random.default_rng(17)
        K = rng.standard_normal((Hkv, T, D)).astype(np.float32)
        K[:, :, :4] *= 20.0
        V = rng.standard_normal((Hkv, T, D)).astype(np.float32)
        eng.prefill_store(0, torch.from_numpy(K).cuda()[None], torch.from_numpy(V).cuda()[None])
        oc = oracle_cache_for(cfg)
        for h in range(Hkv):
            oc.prefill_write(0, h, K[h], V[h], "fp32")
        rc = oracle.RouteConfig(head_dim=D, kind="both", route_policy="joint", score_normalize=True,
                                k_correction_mode=mode, read_budget_mode="absolute", read_abs_k=2, read_abs_v=2,
                                read_budget_ratio=0.0)
        q = rng.standard_normal((Hq, D)).astype(np.float32)
        qt = torch.from_numpy(q).cuda()[None]
        plain = eng.attend(0, qt, router="cached")
        out, lse = eng.attend(0, qt, router="cached", return_lse=True)
        assert torch.equal(out, plain)
        sel = eng.last_selection(0, 0, 1, eng._pages(0, 0))
        lse = lse[0].double().cpu().numpy()
        checked = 0
        for h in range(Hkv):
            K_hat, V_hat, _ = oc.read_base_concat(0, h)
            for i in range(grp):
                qi = q[h * grp + i]
                S, A, O = oracle.base_attention(K_hat, V_hat, qi[None], D)
                _, info = legacy_correction(oc, 0, h, qi, S[0], A[0], O[0], V_hat, rc, oc.sketch_P, kind="both",
                                            score_normalize=True, k_corr_scale=0.1, exact=mode == "exact",
                                            baseline="carekv", rel_thr=0.0, abs_thr=0.0, min_keep=0)
                want_sel = [("K", p, g) for p, g, _ in info["k_sel"]] + [("V", p, b) for p, b, _ in info["v_sel"]]
                if sorted(sel[(0, h, i)]) != sorted(want_sel):
                    continue     # a tie within rounding
                s = S[0].astype(np.float64)
                if mode == "exact":
                    for pid, cg, slot in info["k_sel"]:
                        p0 = pid * cfg.page_size
                        p1 = min(p0 + cfg.page_size, T)
                        packed, sc = oc.read_k_slot(slot)
                        R = unpack_4bit(packed, sc, cfg.page_size * cfg.k_channel_group)
                        R = R.reshape(cfg.page_size, cfg.k_channel_group)[:p1 - p0].astype(np.float64)
                        c0 = cg * cfg.k_channel_group
                        s[p0:p1] += R @ qi[c0:c0 + cfg.k_channel_group] / math.sqrt(D)
                m = s.max()
                want = m + math.log(np.exp(s - m).sum())
                assert abs(lse[h * grp + i] - want) <= LSE_TOL + 1e-5 * abs(want), (h, i)
                checked += 1
        assert checked >= Hq - 1
        cache.check_errors()
