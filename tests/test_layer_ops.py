"""The operators around the MoE FFN against their 64-bit restatement (oracle/layer_ref.py).

CPU: the restatement against torch, and every refusal.  GPU: the kernels, at
the sizes, strides and masks where they can go wrong.  Tolerances:

* expert ids equal, except where the 64-bit choice values of the two experts
  are within 2^-21 of each other (fp32 scores are within a few 2^-24); weights
  within 4e-6 relative (three fp32 operations and a sum of up to 32);
* norm and rotation: half a bf16 ulp (2^-8 of the value) plus 4e-6 of the
  row's largest value (fp32 sums, and the rotation's cancellation);
* cache codes and scale bytes, and what is read back: equal;
* attention: half a bf16 ulp plus the restatement's `slack`; lse within its
  `lse_slack` (2^-16 of the products' magnitudes) plus 4e-6 relative.
"""
import ctypes

import numpy as np
import pytest
import torch

from oracle import layer_ref as R
from warp_decode_b200 import capi

gpu = pytest.mark.gpu


def wd():
    from warp_decode_b200 import warp_decode

    return warp_decode


def np64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


# ---------------------------------------------------------------------------
# the restatement itself
# ---------------------------------------------------------------------------
def test_e4m3_table_and_rounding_match_torch():
    codes = torch.arange(256, dtype=torch.uint8)
    ref = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(R.TABLE, ref, equal_nan=True)
    x = torch.cat([torch.randn(4000) * 2.0 ** torch.randint(-12, 8, (4000,)), torch.linspace(-448, 448, 1793)])
    x = x.clamp(-448, 448)
    assert np.array_equal(R.e4m3_encode(x.double().numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert R.e4m3_encode(np.array([1e9, -1e9, np.nan])).tolist() == [0x7E, 0xFE, 0x7F]


def test_scale_exponent_is_the_least():
    for amax in [448.0, 448.5, 447.9, 1.0, 1.75, 1.7500001, 2.0 ** -100, 3e38]:
        e = R.scale_exponent(amax)
        assert amax <= 448 * 2.0 ** e and (e == -126 or amax > 448 * 2.0 ** (e - 1))


def test_attention_restatement_matches_torch():
    c = cache_case(2, 3, 4, 2, 32, 16, [21, 5], seed=1, device="cpu")
    out, lse, _, _ = R.attn(np64(c["q"]), *c["np"], 0.2, 0)
    for b, n in enumerate([21, 5]):
        k = R.kv_read(c["np"][0], c["np"][1], c["np"][4], [0, 0], n, [n, n])[b]
        v = R.kv_read(c["np"][2], c["np"][3], c["np"][4], [0, 0], n, [n, n])[b]
        for h in range(4):
            s = torch.tensor(np64(c["q"])[b, :, h] @ k[:, h // 2].T * 0.2)
            for i in range(3):
                s[i, n - 3 + i + 1:] = -torch.inf
            ref = torch.softmax(s, 1).numpy() @ v[:, h // 2]
            assert np.allclose(out[b, :, h], ref, atol=1e-12)
            assert np.allclose(lse[b, :, h], torch.logsumexp(s, 1).numpy())


# ---------------------------------------------------------------------------
# refusals: nothing is launched, the reason is told
# ---------------------------------------------------------------------------
def test_layer_library_exports_every_header_symbol():
    import subprocess

    from warp_decode_b200 import _build

    names = capi.header_symbols(capi.LAYER_HEADER)
    assert len(names) == 9, names
    out = subprocess.run(["nm", "-D", "--defined-only", str(_build.LAYER_LIB)], capture_output=True, text=True,
                         check=True).stdout
    assert {line.split()[-1] for line in out.splitlines() if " T " in line} == set(names)
    assert set(capi._LAYER_SIGS) == set(names)


A = 0x1000  # a well-aligned address that is never read


def router_call(**kw):
    a = dict(logits=A, fp32=1, bias=None, ids=A, w=A, T=4, E=64, K=8, scoring=1, n_group=8, pick=4, top=2, renorm=1)
    a.update(kw)
    return capi.layer_lib().wd_moe_router_scored_topk(
        a["logits"], a["fp32"], a["bias"], a["ids"], a["w"], a["T"], a["E"], a["K"], a["scoring"], a["n_group"],
        a["pick"], a["top"], a["renorm"], 1.0, None)


def qk_call(**kw):
    a = dict(q=A, k=A, qw=A, kw=A, pos=A, cs=A, max_pos=8, T=4, Hq=4, Hkv=2, D=64, rot=64)
    a.update(kw)
    return capi.layer_lib().wd_qk_norm_rope(
        a["q"], 256, 64, a["k"], 128, 64, a["qw"], a["kw"], 0, a["pos"], a["cs"], a["max_pos"], A, 256, 64, A, 128,
        64, a["T"], a["Hq"], a["Hkv"], a["D"], a["rot"], 0, 1e-6, None, None)


def write_call(**kw):
    a = dict(k=A, kc=A, ks=A, table=A, start=A, lens=None, B=2, S=3, H=2, D=64, page=16, pages=4)
    a.update(kw)
    return capi.layer_lib().wd_kv_cache_write_fp8(
        a["k"], 384, 128, 64, A, 384, 128, 64, a["kc"], a["ks"], A, A, a["table"], 4, a["start"], a["lens"], a["B"],
        a["S"], a["H"], a["D"], a["page"], a["pages"], None, None)


def read_call(**kw):
    a = dict(kc=A, table=A, start=A, lens=None, out=A, B=2, R=3, H=2, D=64, page=16, pages=4)
    a.update(kw)
    return capi.layer_lib().wd_kv_cache_read_fp8(a["kc"], A, A, A, a["table"], 4, a["start"], a["lens"], a["out"], A,
                                                 a["B"], a["R"], a["H"], a["D"], a["page"], a["pages"], None, None)


def attn_call(**kw):
    a = dict(q=A, kc=A, lens=A, out=A, lse=None, window=0, B=2, Sq=1, Hq=4, Hkv=2, D=64, page=16, pages=4, ws=A,
             ws_bytes=1 << 40)
    a.update(kw)
    return capi.layer_lib().wd_attn_decode_fp8(
        a["q"], 256, 256, 64, a["kc"], A, A, A, A, 4, a["lens"], a["out"], a["lse"], 1.0, a["window"], a["B"],
        a["Sq"], a["Hq"], a["Hkv"], a["D"], a["page"], a["pages"], a["ws"], a["ws_bytes"], None, None)


REFUSED = [
    (router_call, dict(T=-1), capi.WD_ERR_SHAPE, "T must"),
    (router_call, dict(E=0), capi.WD_ERR_SHAPE, "E (number"),
    (router_call, dict(E=1032), capi.WD_ERR_UNSUPPORTED, "1024"),
    (router_call, dict(K=0), capi.WD_ERR_SHAPE, "topk"),
    (router_call, dict(K=33), capi.WD_ERR_UNSUPPORTED, "32"),
    (router_call, dict(n_group=7), capi.WD_ERR_SHAPE, "divide"),
    (router_call, dict(n_group=64), capi.WD_ERR_UNSUPPORTED, "n_group"),
    (router_call, dict(pick=9), capi.WD_ERR_SHAPE, "topk_group"),
    (router_call, dict(top=3), capi.WD_ERR_SHAPE, "group_top"),
    (router_call, dict(pick=1, K=9), capi.WD_ERR_SHAPE, "exceeds"),
    (router_call, dict(scoring=2), capi.WD_ERR_SHAPE, "scoring"),
    (router_call, dict(logits=None), capi.WD_ERR_NULL_POINTER, "null"),
    (router_call, dict(logits=A + 2), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (router_call, dict(bias=A + 1), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (qk_call, dict(T=-1), capi.WD_ERR_SHAPE, "T must"),
    (qk_call, dict(D=63), capi.WD_ERR_SHAPE, "D must"),
    (qk_call, dict(D=258), capi.WD_ERR_UNSUPPORTED, "256"),
    (qk_call, dict(rot=66), capi.WD_ERR_SHAPE, "rot"),
    (qk_call, dict(rot=31), capi.WD_ERR_SHAPE, "rot"),
    (qk_call, dict(k=None), capi.WD_ERR_NULL_POINTER, "null"),
    (qk_call, dict(cs=None), capi.WD_ERR_NULL_POINTER, "null"),
    (qk_call, dict(q=A + 1), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (write_call, dict(B=-1), capi.WD_ERR_SHAPE, "B must"),
    (write_call, dict(S=-1), capi.WD_ERR_SHAPE, "S must"),
    (write_call, dict(H=0), capi.WD_ERR_SHAPE, "Hkv"),
    (write_call, dict(D=72), capi.WD_ERR_SHAPE, "multiple of 16"),
    (write_call, dict(D=272), capi.WD_ERR_UNSUPPORTED, "256"),
    (write_call, dict(page=48), capi.WD_ERR_UNSUPPORTED, "page"),
    (write_call, dict(pages=-1), capi.WD_ERR_SHAPE, "pages"),
    (write_call, dict(k=None), capi.WD_ERR_NULL_POINTER, "null"),
    (write_call, dict(table=None), capi.WD_ERR_NULL_POINTER, "null"),
    (write_call, dict(kc=A + 8), capi.WD_ERR_ALIGNMENT, "16-byte"),
    (write_call, dict(lens=A + 2), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (read_call, dict(R=-1), capi.WD_ERR_SHAPE, "R must"),
    (read_call, dict(start=None), capi.WD_ERR_NULL_POINTER, "null"),
    (read_call, dict(out=A + 8), capi.WD_ERR_ALIGNMENT, "16-byte"),
    (read_call, dict(page=0), capi.WD_ERR_UNSUPPORTED, "page"),
    (attn_call, dict(Sq=-1), capi.WD_ERR_SHAPE, "Sq"),
    (attn_call, dict(Hq=5), capi.WD_ERR_SHAPE, "multiple of Hkv"),
    (attn_call, dict(Hq=0), capi.WD_ERR_SHAPE, "multiple of Hkv"),
    (attn_call, dict(window=-1), capi.WD_ERR_SHAPE, "window"),
    (attn_call, dict(q=None), capi.WD_ERR_NULL_POINTER, "null"),
    (attn_call, dict(lens=None), capi.WD_ERR_NULL_POINTER, "null"),
    (attn_call, dict(out=A + 1), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (attn_call, dict(lse=A + 2), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (attn_call, dict(D=24), capi.WD_ERR_SHAPE, "multiple of 16"),
]


@pytest.mark.parametrize("call,kw,code,msg", REFUSED, ids=lambda v: str(v)[:40])
def test_refusals(call, kw, code, msg):
    L = capi.layer_lib()
    before = L.wd_layer_launch_count()
    assert call(**kw) == code
    assert msg in L.wd_layer_last_error_message().decode()
    assert L.wd_layer_launch_count() == before


def test_empty_calls_do_nothing():
    L = capi.layer_lib()
    before = L.wd_layer_launch_count()
    assert router_call(T=0, logits=None) == capi.WD_OK
    assert qk_call(T=0, q=None) == capi.WD_OK
    assert write_call(B=0, k=None) == capi.WD_OK
    assert write_call(S=0, k=None) == capi.WD_OK
    assert read_call(R=0, out=None) == capi.WD_OK
    assert attn_call(Sq=0, q=None) == capi.WD_OK
    assert attn_call(B=0, q=None) == capi.WD_OK
    assert L.wd_layer_launch_count() == before
    n = ctypes.c_size_t(0)
    assert L.wd_attn_decode_fp8_workspace(2, 1, 5, 2, 64, ctypes.byref(n)) == capi.WD_ERR_SHAPE
    assert L.wd_attn_decode_fp8_workspace(2, 1, 4, 2, 64, None) == capi.WD_ERR_NULL_POINTER


def test_torch_surface_rejects_cpu_tensors():
    z = torch.zeros
    with pytest.raises(RuntimeError, match="logits must be CUDA"):
        wd().moe_router_scored_topk(z(2, 8), 2)
    with pytest.raises(RuntimeError, match="q must be CUDA"):
        wd().qk_norm_rope(z(2, 2, 8).bfloat16(), z(2, 2, 8).bfloat16(), z(8), z(8), z(2).int(), z(4, 8))
    c = cache_case(1, 1, 2, 1, 16, 16, [3], seed=0, device="cpu")
    with pytest.raises(RuntimeError, match="contiguous CUDA uint8"):
        wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"])
    with pytest.raises(RuntimeError, match="contiguous CUDA uint8"):
        wd().kv_cache_write_fp8(c["q"], c["q"], *c["cache"], c["table"], c["lens"])
    with pytest.raises(RuntimeError, match="contiguous CUDA uint8"):
        wd().kv_cache_read_fp8(*c["cache"], c["table"], c["lens"], 1)


@gpu
def test_torch_surface_refusals_on_the_gpu():
    c = cache_case(2, 1, 4, 2, 64, 16, [3, 9], seed=0)
    with pytest.raises(RuntimeError, match="q must be bf16"):
        wd().attn_decode_fp8(c["q"].float(), *c["cache"], c["table"], c["lens"])
    with pytest.raises(RuntimeError, match="seq_lens must be"):
        wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"][:1])
    with pytest.raises(RuntimeError, match="contiguous in its last"):
        wd().attn_decode_fp8(c["q"].transpose(2, 3).contiguous().transpose(2, 3), *c["cache"], c["table"], c["lens"])
    with pytest.raises(RuntimeError, match="same shape"):
        k, ks, v, vs = c["cache"]
        wd().attn_decode_fp8(c["q"], k, ks, v[:1], vs, c["table"], c["lens"])
    with pytest.raises(RuntimeError, match="k and v must be"):
        wd().kv_cache_write_fp8(c["q"], c["q"], *c["cache"], c["table"], c["lens"])
    with pytest.raises(RuntimeError, match="n_group must divide"):
        wd().moe_router_scored_topk(torch.zeros(2, 8, device="cuda"), 2, n_group=3)
    with pytest.raises(RuntimeError, match="bias must be"):
        wd().moe_router_scored_topk(torch.zeros(2, 8, device="cuda"), 2, bias=torch.zeros(7, device="cuda"))
    with pytest.raises(RuntimeError, match="both be bf16 or both"):
        q = torch.zeros(2, 2, 8, device="cuda", dtype=torch.bfloat16)
        wd().qk_norm_rope(q, q, torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda").bfloat16(),
                          torch.zeros(2, device="cuda").int(), torch.zeros(4, 8, device="cuda"))


# ---------------------------------------------------------------------------
# expert choice
# ---------------------------------------------------------------------------
def check_router(lg, K, **kw):
    """Runs the kernel on logits `lg` (CPU) and holds it to the restatement."""
    bias = kw.get("bias")
    got = wd().moe_router_scored_topk(lg.cuda(), K, **{**kw, "bias": None if bias is None else bias.cuda()})
    ids, w = got[0].cpu().numpy(), np64(got[1])
    rid, rw, choice = R.router_scored(np64(lg), K, **{**kw, "bias": None if bias is None else np64(bias)})
    for t, k in zip(*np.nonzero(ids != rid)):
        a, b = choice[t, ids[t, k]], choice[t, rid[t, k]]
        assert abs(a - b) <= 2.0 ** -21 * max(1.0, abs(b)), (t, k, ids[t], rid[t])
    same = (ids == rid).all(1)
    assert same.mean() >= 0.99
    ok = np.abs(w - rw) <= 4e-6 * np.abs(rw) + 1e-30
    assert np.all(ok[same] | (np.isnan(w) & np.isnan(rw))[same])
    return ids, w


@gpu
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (3, 8, 8), (5, 33, 4), (64, 128, 8), (17, 256, 8), (2, 1000, 32),
                                   (4097, 160, 6)])
@pytest.mark.parametrize("kind", ["softmax", "softmax_all", "softmax_bias", "sigmoid", "sigmoid_bias"])
def test_router(T, E, K, kind):
    g = torch.Generator().manual_seed(E * 7 + K)
    lg = torch.randn(T, E, generator=g) * 2
    bias = torch.randn(E, generator=g) * 0.2 if kind.endswith("bias") else None
    if E > 64:
        lg = lg.bfloat16()  # and its many ties
    check_router(lg, K, scoring=kind.split("_")[0], bias=bias, renormalize=kind != "softmax_all",
                 scale=2.5 if E > 64 else 1.0)


@gpu
@pytest.mark.parametrize("E,n_group,pick,top,K", [(256, 8, 4, 2, 8), (64, 32, 3, 2, 6), (160, 8, 3, 1, 6),
                                                  (40, 5, 2, 2, 7), (96, 3, 1, 1, 32), (32, 32, 9, 2, 9),
                                                  (1024, 16, 16, 2, 8)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_router_groups(E, n_group, pick, top, K, scoring):
    g = torch.Generator().manual_seed(E + n_group)
    lg = torch.randn(33, E, generator=g) * 1.5
    bias = torch.randn(E, generator=g) * 0.1 if top == 2 else None
    check_router(lg, K, scoring=scoring, bias=bias, n_group=n_group, topk_group=pick, group_top=top)


@gpu
def test_router_ties_and_odd_logits():
    lg = torch.zeros(6, 64)
    lg[1, 60:] = 3.0
    lg[2] = float("nan")
    lg[3] = float("-inf")
    lg[4, ::2] = float("nan")
    lg[5] = -200.0  # every sigmoid underflows to 0: uniform weights
    for scoring in ("softmax", "sigmoid"):
        for n_group, pick in ((1, 1), (8, 4)):
            ids, w = check_router(lg, 8, scoring=scoring, n_group=n_group, topk_group=pick)
            assert ids[0].tolist() == list(range(8)) and np.allclose(w[0], 0.125)
            assert ids[2].tolist() == list(range(8)) and np.allclose(w[2], 0.125)
            assert ids[3].tolist() == list(range(8)) and np.allclose(w[3], 0.125)
            assert ids[1][:4].tolist() == [60, 61, 62, 63]
    neg = torch.tensor([[0.0, -0.0, 0.0, -0.0]])  # signed zeros tie
    assert check_router(neg, 4)[0].tolist() == [[0, 1, 2, 3]]


# ---------------------------------------------------------------------------
# norm and rotation
# ---------------------------------------------------------------------------
def check_rows_close(got, ref):
    ref = np.asarray(ref)
    big = np.abs(ref).max(-1, keepdims=True)
    err = np.abs(np64(got) - ref)
    assert np.all(err <= 2.0 ** -8 * np.abs(ref) + 4e-6 * big), float((err - 2.0 ** -8 * np.abs(ref)).max())


@gpu
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,inter", [
    (1, 1, 1, 128, 128, False), (64, 64, 4, 128, 128, False), (33, 8, 1, 64, 64, True), (7, 5, 3, 80, 32, False),
    (3, 2, 2, 256, 64, True), (5, 16, 2, 96, 96, False), (9, 3, 0, 64, 0, False), (4, 0, 2, 40, 16, True),
    (3, 2, 1, 2, 2, False), (6, 3, 1, 66, 6, True), (6, 3, 1, 250, 250, False), (11, 4, 4, 128, 24, False),
    (1000, 12, 2, 128, 64, False)])
@pytest.mark.parametrize("strided", [False, True])
def test_qk_norm_rope(T, Hq, Hkv, D, rot, inter, strided):
    g = torch.Generator(device="cuda").manual_seed(T * 100 + D)
    pad = 1 if strided and D % 16 else 0  # an odd offset: rows off the 16-byte grid
    buf = (torch.randn(T, (Hq + 2 * Hkv) * D + pad, generator=g, device="cuda") * 3).bfloat16()
    q, k = buf[:, pad:pad + Hq * D].unflatten(1, (Hq, D)), buf[:, pad + Hq * D:pad + (Hq + Hkv) * D].unflatten(1, (Hkv, D))
    if not strided:
        q, k = q.contiguous(), k.contiguous()
    wt = torch.float32 if T % 2 else torch.bfloat16
    qw = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(wt)
    kw = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(wt)
    pos = torch.randint(0, 97, (T,), generator=g, device="cuda", dtype=torch.int32)
    ang = torch.randn(97, max(rot // 2, 1), generator=g, device="cuda")[:, :rot // 2]
    cs = torch.cat([ang.cos(), ang.sin()], 1).contiguous()
    qo, ko = wd().qk_norm_rope(q, k, qw, kw, pos, cs, 1e-6, inter)
    rq = R.norm_rope(np64(q), np64(qw), pos.cpu(), cs.cpu().numpy(), 1e-6, inter)
    rk = R.norm_rope(np64(k), np64(kw), pos.cpu(), cs.cpu().numpy(), 1e-6, inter)
    if Hq:
        check_rows_close(qo, rq)
    if Hkv:
        check_rows_close(ko, rk)
    # in place: the same bits, and the values beside them untouched
    keep = buf[:, pad + (Hq + Hkv) * D:].clone()
    q2, k2 = wd().qk_norm_rope(q, k, qw, kw, pos, cs, 1e-6, inter, inplace=True)
    assert q2.data_ptr() == q.data_ptr()
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(buf[:, pad + (Hq + Hkv) * D:], keep)
    assert wd().status(True, 0) == 0


@gpu
def test_qk_norm_rope_zero_rows_and_bad_positions():
    q = torch.zeros(4, 2, 128, device="cuda", dtype=torch.bfloat16)
    q[1:] = 1.0
    w = torch.ones(128, device="cuda")
    pos = torch.tensor([0, -1, 4, 3], dtype=torch.int32, device="cuda")
    cs = torch.cat([torch.ones(4, 64), torch.zeros(4, 64)], 1).cuda()
    qo, ko = wd().qk_norm_rope(q, q, w, w, pos, cs)
    assert torch.equal(qo[:3], torch.zeros_like(qo[:3])) and torch.equal(qo, ko)
    assert torch.all((qo[3].float() - 1).abs() < 1e-2)
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_POSITION
    assert wd().status(True, 0) == 0


# ---------------------------------------------------------------------------
# FP8 paged cache
# ---------------------------------------------------------------------------
def cache_case(B, Sq, Hq, Hkv, D, page, lens, seed, device="cuda", spread=1.0):
    """A cache with sequences of the given lengths on shuffled pages, all codes past their ends NaN."""
    g = np.random.default_rng(seed)
    cols = max(1, max((n + page - 1) // page for n in lens))
    P = B * cols + 1
    table = (g.permutation(B * cols) + 1).reshape(B, cols).astype(np.int32)

    def one():
        codes = np.full((P, Hkv, page, D), 0x7F, np.uint8)
        scale = np.full((P, Hkv), 255, np.uint8)
        for b, n in enumerate(lens):
            if n <= 0:
                continue
            x = g.standard_normal((1, n, Hkv, D)) * np.exp(spread * g.standard_normal((1, n, Hkv, 1)))
            x = torch.tensor(x).bfloat16().double().numpy()
            R.kv_write(x, codes, scale, table[b:b + 1], [0], [n])
        return codes, scale

    (kc, ks), (vc, vs) = one(), one()
    q = torch.tensor(g.standard_normal((B, Sq, Hq, D))).bfloat16().to(device)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device)  # noqa: E731
    ln = np.asarray(lens, np.int32)
    return dict(q=q, cache=[t(kc), t(ks), t(vc), t(vs)], table=t(table), lens=t(ln), np=[kc, ks, vc, vs, table, ln])


@gpu
@pytest.mark.parametrize("B,S,H,D,page,starts", [
    (1, 1, 1, 128, 64, [0]), (3, 1, 2, 128, 64, [63, 64, 5]), (2, 5, 2, 64, 16, [14, 0]), (2, 100, 1, 80, 32, [31, 7]),
    (1, 300, 2, 256, 128, [127]), (4, 17, 3, 16, 16, [0, 1, 15, 33]), (65, 1, 4, 128, 16, None)])
@pytest.mark.parametrize("strided", [False, True])
def test_kv_write_and_read(B, S, H, D, page, starts, strided):
    g = np.random.default_rng(B * 1000 + S)
    starts = starts or g.integers(0, 90, B).tolist()
    lens = [S if b % 3 == 0 else int(g.integers(0, S + 1)) for b in range(B)]
    c = cache_case(B, 1, H, H, D, page, [max(n, 0) for n in starts], seed=S)
    cols = (max(starts) + S + page - 1) // page
    P = B * cols + 1
    # room for the new tokens: fresh pages appended to each table
    table = np.zeros((B, cols), np.int32)
    old_cols = c["np"][4].shape[1]
    fresh = iter(range(c["np"][0].shape[0], c["np"][0].shape[0] + P))
    for b in range(B):
        for j in range(cols):
            table[b, j] = c["np"][4][b, j] if j < min(old_cols, (starts[b] + page - 1) // page) else next(fresh)
    grow = lambda a: np.concatenate([a, np.full((P,) + a.shape[1:], 0x55, np.uint8)])  # noqa: E731
    kc, ks, vc, vs = (grow(a) for a in c["np"][:4])
    x = g.standard_normal((B, S, 2 * H * D)) * np.exp(1.5 * g.standard_normal((B, S, 1)))
    off = 1 if strided and D == 80 else 0
    buf = torch.zeros(B, S, 2 * H * D + off, dtype=torch.bfloat16)
    buf[..., off:] = torch.tensor(x).bfloat16()
    buf = buf.cuda()
    k, v = buf[..., off:off + H * D].unflatten(2, (H, D)), buf[..., off + H * D:].unflatten(2, (H, D))
    if not strided:
        k, v = k.contiguous(), v.contiguous()
    dev = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
    tab = torch.from_numpy(table).cuda()
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    wd().kv_cache_write_fp8(k, v, *dev, tab, i32(starts), i32(lens))
    R.kv_write(np64(k), kc, ks, table, starts, lens)
    R.kv_write(np64(v), vc, vs, table, starts, lens)
    for got, ref in zip(dev, (kc, ks, vc, vs)):
        assert np.array_equal(got.cpu().numpy(), ref)
    # read back: everything, and the tail
    ends = [s + n for s, n in zip(starts, lens)]
    for r0, n in (([0] * B, max(max(ends), 1)), ([max(e - 3, 0) for e in ends], 5)):
        want = [e - s for e, s in zip(ends, r0)]
        gk, gv = wd().kv_cache_read_fp8(*dev, tab, i32(r0), n, i32(want))
        assert np.array_equal(np64(gk), R.kv_read(kc, ks, table, r0, n, want))
        assert np.array_equal(np64(gv), R.kv_read(vc, vs, table, r0, n, want))
    assert wd().status(True, 0) == 0


@gpu
def test_kv_write_extremes():
    """Zeros, infinities, NaN, the smallest and largest bf16, and the exact border 448 * 2^e."""
    D, page = 32, 16
    rows = torch.zeros(8, 1, 1, D, dtype=torch.bfloat16)
    rows[1, ..., 0] = float("inf")
    rows[2, ..., :3] = torch.tensor([float("nan"), 5.0, -float("inf")]).bfloat16()
    rows[3, ..., 0] = torch.finfo(torch.bfloat16).max
    rows[4, ..., 0] = torch.finfo(torch.bfloat16).tiny / 128
    rows[5, ..., 0] = 448.0 * 8
    rows[6, ..., 0] = 450.0 * 8
    rows[7, ..., :] = -0.0
    P = 8
    kc, ks = np.full((P, 1, page, D), 0x33, np.uint8), np.full((P, 1), 9, np.uint8)
    table, zero, one = np.arange(P, dtype=np.int32)[:, None], [0] * P, [1] * P
    dev = [torch.from_numpy(a.copy()).cuda() for a in (kc, ks, kc, ks)]
    x = rows.cuda()
    wd().kv_cache_write_fp8(x, x, *dev, torch.from_numpy(table).cuda(), torch.tensor(zero, dtype=torch.int32).cuda())
    R.kv_write(np64(x), kc, ks, table, zero, one)
    assert np.array_equal(dev[0].cpu().numpy(), kc) and np.array_equal(dev[3].cpu().numpy(), ks)
    assert ks[5, 0] == 130 and ks[6, 0] == 131
    # a second token that raises every scale: the first one is rounded again
    big = torch.full((P, 1, 1, D), 3000.0, dtype=torch.bfloat16, device="cuda")
    wd().kv_cache_write_fp8(big, big, *dev, torch.from_numpy(table).cuda(), torch.tensor(one, dtype=torch.int32).cuda())
    R.kv_write(np64(big), kc, ks, table, one, one)
    assert np.array_equal(dev[2].cpu().numpy(), kc) and np.array_equal(dev[1].cpu().numpy(), ks)
    assert wd().status(True, 0) == 0


@gpu
def test_kv_bad_pages_and_positions():
    c = cache_case(3, 1, 2, 2, 64, 16, [20, 20, 20], seed=4)
    dev = [t.clone() for t in c["cache"]]
    table = c["table"].clone()
    table[0, 1] = -1
    table[1, 1] = 10 ** 6
    x = torch.ones(3, 1, 2, 64, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([20, 20, 32], dtype=torch.int32, device="cuda")  # the last one lies past its table
    wd().kv_cache_write_fp8(x, x, *dev, table, at)
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE
    assert all(torch.equal(a, b) for a, b in zip(dev, c["cache"]))
    k, v = wd().kv_cache_read_fp8(*dev, table, at, 1)
    assert not k.any() and not v.any()
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE
    wd().kv_cache_write_fp8(x, x, *dev, table, at - 40)
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_POSITION
    assert all(torch.equal(a, b) for a, b in zip(dev, c["cache"]))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def check_attn(c, window=0, scale=None, q=None, lens=None, workspace=None):
    q = c["q"] if q is None else q
    D = q.shape[3]
    s = 1 / D ** 0.5 if scale is None else scale
    out, lse = wd().attn_decode_fp8(q, *c["cache"], c["table"], c["lens"] if lens is None else lens, scale, window,
                                    workspace, True)
    kc, ks, vc, vs, table, ln = c["np"]
    ref, rlse, slack, lse_slack = R.attn(np64(q), kc, ks, vc, vs, table, ln if lens is None else lens.cpu().numpy(), s, window)
    got = np64(out)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    err = np.abs(got - ref)
    fine = ~np.isnan(ref)
    over = err[fine] - (2.0 ** -8 * np.abs(ref) + slack)[fine] - 1e-30
    assert over.max(initial=-1) <= 0, (float(over.max()), float(err[fine].max()))
    gl = lse.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isneginf(gl), np.isneginf(rlse)) and np.array_equal(np.isnan(gl), np.isnan(rlse))
    ok = np.isfinite(rlse)
    assert np.all(np.abs(gl - rlse)[ok] <= (lse_slack + 4e-6 * (1 + np.abs(rlse)))[ok])
    return out, lse


SHAPES = [  # B, Sq, Hq, Hkv, D, page, lens, window
    (1, 1, 1, 1, 128, 64, [1], 0),
    (1, 1, 8, 1, 128, 64, [1000], 0),
    (3, 1, 8, 2, 128, 16, [129, 0, 128], 0),
    (2, 1, 32, 4, 128, 128, [517, 40], 0),
    (2, 4, 32, 4, 128, 64, [300, 3], 0),
    (2, 1, 16, 1, 128, 32, [700, 65], 100),
    (1, 3, 10, 2, 128, 64, [260], 1),
    (1, 8, 16, 1, 128, 64, [390], 129),
    (2, 2, 5, 1, 128, 16, [257, 2], 7),
    (1, 1, 64, 64, 128, 64, [70], 0),
    (1, 1, 8, 1, 64, 64, [1000], 0),
    (3, 1, 14, 2, 64, 16, [129, 0, 1], 0),
    (2, 5, 16, 4, 64, 128, [300, 3], 33),
    (1, 8, 32, 2, 64, 32, [515], 0),
    (2, 1, 4, 2, 80, 16, [37, 200], 0),
    (1, 2, 3, 1, 256, 64, [131], 0),
    (1, 1, 6, 3, 16, 16, [45], 9),
    (2, 1, 2, 1, 192, 32, [64, 33], 0),
    (1, 1, 128, 1, 128, 64, [200], 0),
    (1, 40, 8, 2, 128, 64, [129], 0),
]


@gpu
@pytest.mark.parametrize("B,Sq,Hq,Hkv,D,page,lens,window", SHAPES)
def test_attention(B, Sq, Hq, Hkv, D, page, lens, window):
    c = cache_case(B, Sq, Hq, Hkv, D, page, lens, seed=Sq * 100 + D)
    out, lse = check_attn(c, window)
    again, lse2 = wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], None, window, None, True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("D", [64, 128, 48])
def test_attention_strided_queries_and_scale(D):
    c = cache_case(2, 3, 8, 2, D, 32, [200, 77], seed=8)
    big = torch.randn(2, 3, 8 * D + 2 * D + 1, device="cuda").bfloat16()
    q = big[..., 1:1 + 8 * D].unflatten(2, (8, D))  # off the 16-byte grid
    check_attn(c, q=q, scale=0.5)
    t = torch.randn(2, 8, 3, D, device="cuda").bfloat16().transpose(1, 2)  # heads outside tokens
    check_attn(c, q=t)
    check_attn(c, q=t * 1e-3)
    check_attn(c, scale=0.0)


@gpu
@pytest.mark.parametrize("D", [64, 128, 32])
def test_attention_growing_scores(D):
    """Each stretch of keys outweighs all before it by far, and shrinking ones: the running maximum's both ways."""
    c = cache_case(2, 2, 4, 1, D, 64, [900, 900], seed=5)
    kc, ks, vc, vs, table, ln = c["np"]
    for col in range(table.shape[1]):
        ks[table[0, col]] = 118 + col % 12
        ks[table[1, col]] = 130 - col % 12
        vs[table[0, col]] = 100 + 3 * ((col * 5) % 11)  # values of very different magnitude
    c["cache"] = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
    check_attn(c)


@gpu
@pytest.mark.parametrize("D", [64, 128, 32])
def test_attention_masked_nan_has_no_influence(D):
    """NaN codes and scales past the end, before the window and on other sequences' pages; a seen NaN is seen."""
    c = cache_case(2, 3, 8, 2, D, 16, [200, 90], seed=6)
    kc, ks, vc, vs, table, ln = c["np"]
    vc[table[0, 1], 0, 3] = 0x7F   # position 19 of sequence 0, head 0
    kc[table[0, 1], 1, 5] = 0xFF   # position 21, head 1
    vc[table[1, 5], 0, 9, 0] = 0x7F  # position 89 of sequence 1: the last token, seen by the last query only
    c["cache"] = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
    out, _ = check_attn(c, window=150)   # positions 19 and 21 lie before every window
    assert not out[0].isnan().any()
    assert out[1, 2, 0, 0].isnan() and not out[1, :2].isnan().any()
    out, _ = check_attn(c)
    assert out[0, 0, 0].isnan().all() and out[0, 0, 4].isnan().all()


@gpu
@pytest.mark.parametrize("D", [128, 64, 48])
def test_attention_bad_pages_are_masked(D):
    c = cache_case(2, 1, 4, 2, D, 16, [200, 64], seed=7)
    table = c["np"][4]
    table[0, 3] = -5
    table[0, 12] = 1 << 30
    table[1, :] = -1  # nothing left: zeros
    c["table"] = torch.from_numpy(table).cuda()
    out, lse = check_attn(c)
    assert not out[1].any() and torch.isneginf(lse[1]).all()
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE
    # a length past the table's columns: those tokens are masked too
    c = cache_case(1, 1, 4, 2, D, 16, [64], seed=9)
    check_attn(c, lens=torch.tensor([90], dtype=torch.int32, device="cuda"))
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE


@gpu
def test_attention_workspace_and_streams():
    """One workspace for calls of different sizes, in a row, on a stream of their own, and in a graph."""
    cases = [cache_case(1, 1, 16, 2, 128, 64, [3000], seed=1), cache_case(3, 2, 8, 1, 128, 32, [999, 5, 64], seed=2),
             cache_case(2, 1, 8, 8, 64, 16, [1500, 700], seed=3)]
    ws = torch.zeros(16 << 20, dtype=torch.uint8, device="cuda")
    plain = [check_attn(c)[0] for c in cases]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            for c, p in zip(cases, plain):
                got = wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], workspace=ws)
                assert torch.equal(got, p)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], workspace=ws) for c in cases]
    for _ in range(2):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, p) for o, p in zip(outs, plain))
    # the lengths are read by the kernel, not when the graph was made
    c = cases[0]
    c["lens"].fill_(130)
    graph.replay()
    torch.cuda.synchronize()
    ref, _, slack, _ = R.attn(np64(c["q"]), *c["np"][:5], [130], 128 ** -0.5, 0)
    assert np.all(np.abs(np64(outs[0]) - ref) <= 2.0 ** -8 * np.abs(ref) + slack)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("D,Hq,Hkv,page", [(128, 8, 1, 64), (64, 6, 2, 16), (128, 40, 1, 32)])
def test_attention_many_sequences(D, Hq, Hkv, page):
    """More sequences than a warp's lanes, empty ones among them: every CTA's share crosses several."""
    g = np.random.default_rng(D + page)
    lens = [0 if b % 9 == 4 else int(g.integers(1, 400)) for b in range(70)]
    c = cache_case(70, 1, Hq, Hkv, D, page, lens, seed=page)
    check_attn(c)
    check_attn(c, window=50)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("B,Sq,Hq,lens", [(1, 1, 4, [20011]), (2, 3, 16, [9000, 130]), (1, 5, 13, [12345])])
def test_attention_long_sequences(B, Sq, Hq, lens):
    """One key head whose tiles are split over dozens of CTAs, in every column width."""
    c = cache_case(B, Sq, Hq, 1, 128, 128, lens, seed=Hq)
    out, lse = check_attn(c)
    for _ in range(3):  # whichever CTA comes last
        again, lse2 = wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], return_lse=True)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert wd().status(True, 0) == 0


@gpu
def test_attention_workspace_refusals():
    c = cache_case(1, 1, 8, 1, 128, 64, [100], seed=3)
    call = lambda ws: wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], workspace=ws)  # noqa: E731
    with pytest.raises(RuntimeError, match="smaller than"):
        call(torch.zeros(1024, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        call(torch.zeros(16 << 20, dtype=torch.uint8, device="cuda")[8:])
    with pytest.raises(RuntimeError, match="workspace must be"):
        call(torch.zeros(16 << 20, dtype=torch.uint8))
    ws = wd().attn_decode_fp8_workspace(1, 1, 8, 1, 128)
    assert torch.equal(call(ws), call(None)) and ws.numel() <= 16 << 20
    assert wd().attn_decode_fp8_workspace(1, 1, 8, 1, 80).numel() == 0


@gpu
def test_attention_on_a_table_without_columns():
    c = cache_case(2, 1, 4, 2, 128, 16, [20, 3], seed=2)
    out, lse = wd().attn_decode_fp8(c["q"], *c["cache"], torch.zeros(2, 0, dtype=torch.int32, device="cuda"), c["lens"],
                                    return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE
    zero = torch.zeros_like(c["lens"])
    out, lse = wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], zero - 5, return_lse=True)  # negative: nothing seen
    assert not out.any() and torch.isneginf(lse).all()
    assert wd().status(True, 0) == 0


@gpu
def test_decoder_layer_example():
    """Prompt and single tokens through every operator together, against plain fp32 torch on the cache's values.

    The layer's outputs are bf16 (2^-9 of a value each, in norm 2^-9 of the row), its steps round to bf16 seven
    times in a row and differ from the plain ones in the order of fp32 sums before each: 1e-2 of a row's norm.
    """
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "decoder_layer_step.py"
    spec = importlib.util.spec_from_file_location("decoder_layer_step", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main() <= 1e-2


@gpu
def test_attention_on_two_streams_at_once():
    """Calls that overlap in time, each stream with a workspace of its own: the bits of calls in a row."""
    cases = [cache_case(2, 1, 16, 2, 128, 64, [2500, 900], seed=s) for s in (11, 12)]
    plain = [wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"]) for c in cases]
    spaces = [wd().attn_decode_fp8_workspace(2, 1, 16, 2, 128) for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                outs[i].append(wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], workspace=spaces[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, plain[i]) for i in range(2) for o in outs[i])
    assert wd().status(True, 0) == 0


@gpu
def test_operators_launch_once_a_call():
    c = cache_case(2, 1, 8, 2, 128, 16, [40, 3], seed=1)
    ws = wd().attn_decode_fp8_workspace(2, 1, 8, 2, 128)
    x = torch.zeros(2, 1, 2, 128, device="cuda", dtype=torch.bfloat16)
    dev = [t.clone() for t in c["cache"]]
    calls = [lambda: wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], workspace=ws),
             lambda: wd().kv_cache_write_fp8(x, x, *dev, c["table"], c["lens"] - 1),
             lambda: wd().kv_cache_read_fp8(*c["cache"], c["table"], c["lens"] - 1, 1),
             lambda: wd().qk_norm_rope(c["q"][0], x[0], torch.ones(128, device="cuda"), torch.ones(128, device="cuda"),
                                       torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(1, 128, device="cuda")),
             lambda: wd().moe_router_scored_topk(torch.zeros(3, 64, device="cuda"), 2)]
    for call in calls:
        before = wd().launch_count()
        call()
        assert wd().launch_count() == before + 1
    assert wd().status(True, 0) == 0
