"""The operators that complete a decoder layer's step against their 64-bit restatement
(oracle/block_ref.py, and oracle/layer_ref.py for attention).

CPU: the restatement against torch, the packing, and every refusal.  GPU: the kernels,
at the sizes, strides and masks where they can go wrong.  Tolerances: half a step of
the output's type (bf16 2^-8 of the value, fp32 2^-24) plus the restatement's slack;
attention's besides has 2^-18 of the query row's largest value times the key's
magnitudes in every score, which q's two terms may lose.
"""
import ctypes

import numpy as np
import pytest
import torch

from oracle import block_ref as B_
from oracle import layer_ref as R
from test_layer_ops import cache_case, np64, wd
from warp_decode_b200 import capi, w4

gpu = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


# ---------------------------------------------------------------------------
# the restatement and the packing
# ---------------------------------------------------------------------------
def test_block_norm_restatement_matches_torch():
    g = torch.Generator().manual_seed(0)
    y, r, w, p = (torch.randn(*s, generator=g, dtype=torch.float64) for s in [(5, 24), (5, 24), (24,), (24,)])
    gate = torch.randn(5, 1, generator=g, dtype=torch.float64)
    norm = lambda v, k: torch.nn.functional.rms_norm(v, (24,), k, 1e-6)  # noqa: E731
    x, out, *_ = B_.block_norm(y.numpy(), r.numpy(), w.numpy(), p.numpy(), gate.numpy(), 0.5)
    ref = 0.5 * r + gate * norm(y, p)
    assert np.allclose(out, ref.numpy(), atol=1e-13) and np.allclose(x, norm(ref, w).numpy(), atol=1e-13)
    x, out, *_ = B_.block_norm(y.numpy(), r.numpy(), w.numpy())
    assert np.allclose(x, norm(y + r, w).numpy(), atol=1e-13)


@pytest.mark.parametrize("N,K", [(1, 32), (3, 128), (5, 160), (2, 640)])
def test_w4_packing(N, K):
    codes = torch.randint(0, 16, (N, K), generator=torch.Generator().manual_seed(K), dtype=torch.uint8)
    packed = w4.pack_w4(codes)
    assert packed.shape == (N, -(-K // 128) * 64) and torch.equal(w4.unpack_w4(packed, K), codes)
    words = packed.numpy().view("<u4")
    for n in range(N):
        for k in range(K):  # the order that the C header gives
            b, s, t, i = k // 128, k % 128 // 32, k % 32 // 8, k % 8
            assert words[n, 16 * b + 4 * t + s] >> (4 * (i // 2) + 16 * (i % 2)) & 15 == codes[n, k]
    with pytest.raises(ValueError, match="0 to 15"):
        w4.pack_w4(codes + 16)


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype", [BF16, torch.float16, F32])
def test_w4_quantiser(zero_points, dtype):
    w = torch.randn(6, 256, generator=torch.Generator().manual_seed(3))
    w[2] = 0.0
    w[3] = w[3].abs() + 1
    packed, scale, zero = w4.quantize_w4(w, 64, zero_points, dtype)
    assert scale.dtype == dtype and scale.shape == (6, 4) and (zero is None) != zero_points
    back = w4.dequantize_w4(packed, scale, zero, 256)
    # half a step of the scale, which its rounding may leave up to eight steps short by 2^-8 each
    step = scale.float().repeat_interleave(64, 1)
    assert torch.all((back - w).abs() <= step * (0.5 + 15 * 2.0 ** -8) + 1e-7)
    assert not back[2].any()
    with pytest.raises(ValueError, match="multiple of group"):
        w4.quantize_w4(w, 48)


# ---------------------------------------------------------------------------
# refusals: nothing is launched, the reason is told
# ---------------------------------------------------------------------------
def test_block_library_exports_every_header_symbol():
    import subprocess

    from warp_decode_b200 import _build

    names = capi.header_symbols(capi.BLOCK_HEADER)
    assert len(names) == 7, names
    out = subprocess.run(["nm", "-D", "--defined-only", str(_build.BLOCK_LIB)], capture_output=True, text=True,
                         check=True).stdout
    assert {line.split()[-1] for line in out.splitlines() if " T " in line} == set(names)
    assert set(capi._BLOCK_SIGS) == set(names)


A = 0x1000  # a well-aligned address that is never read


def norm_call(**kw):
    a = dict(y=A, r=A, r32=0, nw=A, pw=None, w32=0, gate=None, gcs=1, g32=0, x=A, ro=A, T=4, H=64)
    a.update(kw)
    return capi.block_lib().wd_block_norm(a["y"], 64, a["r"], 64, a["r32"], a["nw"], a["pw"], a["w32"], a["gate"], 0,
                                          a["gcs"], a["g32"], 1.0, 1e-6, a["x"], 64, a["ro"], 64, a["T"], a["H"], None)


def linear_call(**kw):
    a = dict(x=A, w=A, s=A, st=0, z=None, out=A, T=4, N=64, K=256, group=64)
    a.update(kw)
    return capi.block_lib().wd_linear_w4(a["x"], 256, a["w"], a["s"], a["st"], a["z"], a["out"], 64, a["T"], a["N"],
                                         a["K"], a["group"], None)


def prefix_call(**kw):
    a = dict(q=A, kc=A, lens=A, pre=A, out=A, lse=None, window=0, B=2, Sq=1, Hq=4, Hkv=2, D=64, page=16, pages=4, ws=A,
             ws_bytes=1 << 40)
    a.update(kw)
    return capi.block_lib().wd_attn_decode_fp8_prefix(
        a["q"], 256, 256, 64, a["kc"], A, A, A, A, 4, a["lens"], a["pre"], a["out"], a["lse"], 1.0, a["window"], a["B"],
        a["Sq"], a["Hq"], a["Hkv"], a["D"], a["page"], a["pages"], a["ws"], a["ws_bytes"], None, None)


REFUSED = [
    (norm_call, dict(T=-1), capi.WD_ERR_SHAPE, "T must"),
    (norm_call, dict(H=0), capi.WD_ERR_SHAPE, "H must"),
    (norm_call, dict(H=16392), capi.WD_ERR_UNSUPPORTED, "16384"),
    (norm_call, dict(gate=A, gcs=2), capi.WD_ERR_SHAPE, "gate_channel_stride"),
    (norm_call, dict(y=None), capi.WD_ERR_NULL_POINTER, "null"),
    (norm_call, dict(nw=None), capi.WD_ERR_NULL_POINTER, "null"),
    (norm_call, dict(ro=None), capi.WD_ERR_NULL_POINTER, "null"),
    (norm_call, dict(y=A + 1), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (norm_call, dict(r=A + 2, r32=1), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (norm_call, dict(pw=A + 2, w32=1), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (norm_call, dict(gate=A + 1), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (linear_call, dict(T=-1), capi.WD_ERR_SHAPE, "T and N"),
    (linear_call, dict(N=-1), capi.WD_ERR_SHAPE, "T and N"),
    (linear_call, dict(group=16), capi.WD_ERR_UNSUPPORTED, "group"),
    (linear_call, dict(K=0), capi.WD_ERR_SHAPE, "K must"),
    (linear_call, dict(K=96), capi.WD_ERR_SHAPE, "multiple of group"),
    (linear_call, dict(K=(1 << 30) + 64), capi.WD_ERR_UNSUPPORTED, "2^30"),
    (linear_call, dict(st=3), capi.WD_ERR_SHAPE, "scale_type"),
    (linear_call, dict(x=None), capi.WD_ERR_NULL_POINTER, "null"),
    (linear_call, dict(s=None), capi.WD_ERR_NULL_POINTER, "null"),
    (linear_call, dict(w=A + 8), capi.WD_ERR_ALIGNMENT, "16 bytes"),
    (linear_call, dict(s=A + 2, st=2), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (linear_call, dict(N=1 << 20), capi.WD_ERR_UNSUPPORTED, "N must be at most"),
    (linear_call, dict(T=1 << 20), capi.WD_ERR_UNSUPPORTED, "T at most"),
    (prefix_call, dict(B=-1), capi.WD_ERR_SHAPE, "B must"),
    (prefix_call, dict(Sq=-1), capi.WD_ERR_SHAPE, "Sq"),
    (prefix_call, dict(Hq=5), capi.WD_ERR_SHAPE, "multiple of Hkv"),
    (prefix_call, dict(window=-1), capi.WD_ERR_SHAPE, "window"),
    (prefix_call, dict(page=8), capi.WD_ERR_UNSUPPORTED, "page"),
    (prefix_call, dict(D=24), capi.WD_ERR_SHAPE, "multiple of 16"),
    (prefix_call, dict(q=None), capi.WD_ERR_NULL_POINTER, "null"),
    (prefix_call, dict(pre=None), capi.WD_ERR_NULL_POINTER, "null"),
    (prefix_call, dict(lens=None), capi.WD_ERR_NULL_POINTER, "null"),
    (prefix_call, dict(pre=A + 2), capi.WD_ERR_ALIGNMENT, "misaligned"),
    (prefix_call, dict(out=A + 8), capi.WD_ERR_ALIGNMENT, "misaligned"),
]


@pytest.mark.parametrize("call,kw,code,msg", REFUSED, ids=lambda v: str(v)[:40])
def test_refusals(call, kw, code, msg):
    L = capi.block_lib()
    before = L.wd_block_launch_count()
    assert call(**kw) == code
    assert msg in L.wd_block_last_error_message().decode()
    assert L.wd_block_launch_count() == before


def test_empty_calls_do_nothing():
    L = capi.block_lib()
    before = L.wd_block_launch_count()
    assert norm_call(T=0, y=None) == capi.WD_OK
    assert linear_call(T=0, x=None) == capi.WD_OK
    assert linear_call(N=0, w=None) == capi.WD_OK
    assert prefix_call(B=0, q=None) == capi.WD_OK
    assert prefix_call(Sq=0, q=None) == capi.WD_OK
    assert L.wd_block_launch_count() == before
    n = ctypes.c_size_t(0)
    assert L.wd_attn_decode_fp8_prefix_workspace(2, 1, 5, 2, 64, ctypes.byref(n)) == capi.WD_ERR_SHAPE
    assert L.wd_attn_decode_fp8_prefix_workspace(2, 1, 4, 2, 64, None) == capi.WD_ERR_NULL_POINTER


def test_torch_surface_rejects_cpu_tensors():
    z = torch.zeros
    with pytest.raises(RuntimeError, match="y must be CUDA"):
        wd().block_norm(z(2, 8).bfloat16(), z(2, 8).bfloat16(), z(8))
    with pytest.raises(RuntimeError, match="x must be CUDA"):
        wd().linear_w4(z(2, 128).bfloat16(), z(4, 64, dtype=torch.uint8), z(4, 1))
    c = cache_case(1, 1, 2, 1, 64, 16, [3], seed=0, device="cpu")
    with pytest.raises(RuntimeError, match="contiguous CUDA uint8"):
        wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["lens"])


@gpu
def test_torch_surface_refusals_on_the_gpu():
    z = lambda *s, dtype=BF16: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    norm, lin = wd().block_norm, wd().linear_w4
    with pytest.raises(RuntimeError, match="residual must be"):
        norm(z(2, 8), z(3, 8), z(8))
    with pytest.raises(RuntimeError, match="must be \\[H\\]"):
        norm(z(2, 8), z(2, 8), z(9))
    with pytest.raises(RuntimeError, match="both be bf16 or both"):
        norm(z(2, 8), z(2, 8), z(8), z(8, dtype=F32))
    with pytest.raises(RuntimeError, match="gate must be"):
        norm(z(2, 8), z(2, 8), z(8), gate=z(3, 8))
    with pytest.raises(RuntimeError, match="contiguous in its last"):
        norm(z(2, 8), z(2, 8), z(8), gate=z(8, 2).t())
    with pytest.raises(RuntimeError, match="single memory location"):
        norm(z(2, 8), z(1, 8).expand(2, 8), z(8), inplace=True)
    with pytest.raises(RuntimeError, match="memory location"):
        r = z(5, 8)
        norm(r[1:], r[:4], z(8), inplace=True)
    with pytest.raises(RuntimeError, match="share memory"):
        norm(z(2, 8), z(40).as_strided((2, 8), (4, 1)), z(8), inplace=True)
    with pytest.raises(RuntimeError, match="ceil"):
        lin(z(2, 128), z(4, 128, dtype=torch.uint8), z(4, 1))
    with pytest.raises(RuntimeError, match="group"):
        lin(z(2, 128), z(4, 64, dtype=torch.uint8), z(4, 3))
    with pytest.raises(RuntimeError, match="group must be 32, 64 or 128"):
        lin(z(2, 256), z(4, 128, dtype=torch.uint8), z(4, 1))
    with pytest.raises(RuntimeError, match="w_zero"):
        lin(z(2, 128), z(4, 64, dtype=torch.uint8), z(4, 1), z(4, 2, dtype=torch.uint8))
    c = cache_case(2, 1, 4, 2, 64, 16, [3, 9], seed=0)
    with pytest.raises(RuntimeError, match="prefix_len must be"):
        wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["lens"])
    with pytest.raises(RuntimeError, match="prefix_len must be"):
        wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["lens"][:1].cpu())
    call = lambda ws: wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["lens"][:1],  # noqa: E731
                                                  workspace=ws)
    with pytest.raises(RuntimeError, match="smaller than"):
        call(z(1024, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        call(z(64 << 20, dtype=torch.uint8)[8:])
    assert wd().attn_decode_fp8_prefix_workspace(1, 1, 8, 1, 80).numel() == 0


# ---------------------------------------------------------------------------
# block norm
# ---------------------------------------------------------------------------
def check_norm(y, r, w, post=None, gate=None, scale=1.0, **kw):
    x, out = wd().block_norm(y, r, w, post, gate, scale, **kw)
    g = None if gate is None else np.broadcast_to(np64(gate), y.shape)
    rx, ro, xs, rs = B_.block_norm(np64(y), np64(r), np64(w), None if post is None else np64(post), g, scale)
    for got, ref, slack in ((x, rx, xs), (out, ro, rs)):
        err = np.abs(np64(got) - ref)
        assert np.all(err <= HALF[got.dtype] * np.abs(ref) + slack + 1e-37), float((err - slack).max())
    assert out.dtype == r.dtype and x.dtype == BF16
    return x, out


NORM_SIZES = [(1, 1), (3, 7), (5, 8), (1, 250), (2, 256), (9, 264), (300, 40), (301, 1000), (1, 1032), (700, 1024),
              (2, 2048), (310, 2056), (1, 7168), (299, 7168), (3, 8200), (400, 8192), (2, 16384), (330, 16376), (1, 16383)]


@gpu
@pytest.mark.parametrize("T,H", NORM_SIZES)
@pytest.mark.parametrize("kind", range(6))
def test_block_norm(T, H, kind):
    """Every size with every kind of gate, residual and weight, and rows on and off the 16-byte grid."""
    g = torch.Generator(device="cuda").manual_seed(T * 31 + H + kind)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    pad = kind % 2  # an odd offset
    y = (rand(T, H + 16)[:, pad:pad + H] * 2).to(BF16)
    big = (rand(T, H + 24) * 3).to(BF16 if kind < 3 else F32)
    r = big[:, pad:pad + H]
    wt = F32 if kind in (1, 4) else BF16
    w, post = (1 + 0.2 * rand(H)).to(wt), (1 + 0.2 * rand(H)).to(wt) if kind % 3 else None
    gate = [None, rand(H), rand(T, 1).to(BF16), rand(T, H + 8).to(BF16)[:, :H], rand(1, H).to(BF16).expand(T, H),
            rand(T, 1).expand(T, H)][kind]
    scale = 0.5 if kind == 2 else 1.0
    x, out = check_norm(y, r, w, post, gate, scale)
    # in place: the same bits, and the values beside the rows untouched
    keep = big.clone()
    x2, out2 = wd().block_norm(y, r, w, post, gate, scale, inplace=True)
    assert out2.data_ptr() == r.data_ptr() and torch.equal(x2, x) and torch.equal(r, out)
    keep[:, pad:pad + H] = out
    assert torch.equal(big, keep)


@gpu
def test_block_norm_odd_values():
    H = 320
    y = torch.randn(6, H, device="cuda").to(BF16)
    r = torch.randn(6, H, device="cuda").to(BF16)
    y[0], r[0] = 0, 0             # nothing at all: zeros
    y[1, 3] = float("nan")        # its row alone
    y[2, 5] = float("inf")
    y[3], r[3] = 1e-30, 0         # squares that underflow: eps stands
    y[4] *= 1e17                  # squares near 1e34
    x, out = wd().block_norm(y, r, torch.ones(H, device="cuda"), torch.ones(H, device="cuda"))
    assert not x[0].any() and not out[0].any()
    assert x[1].isnan().all() and out[1].isnan().all() and x[2].isnan().any()
    assert torch.isfinite(x[3:].float()).all() and torch.isfinite(out[3:].float()).all()
    keep = [0, 3, 4, 5]
    check_norm(y[keep], r[keep], torch.ones(H, device="cuda"), torch.ones(H, device="cuda"))
    gate = torch.full((6, 1), float("inf"), device="cuda")
    for width in (H, H - 3):  # an infinite gate of a token, on both paths
        x, out = wd().block_norm(y[5:, :width].contiguous(), r[5:, :width].contiguous(),
                                 torch.ones(width, device="cuda"), None, gate[5:])
        assert torch.isinf(out.float()).all()


# ---------------------------------------------------------------------------
# 4-bit projection
# ---------------------------------------------------------------------------
def linear_case(T, N, K, group, scales, zero, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T * 7 + N + K)
    x = torch.randn(T, K + 8, generator=g, device="cuda").to(BF16)[:, pad:pad + K]
    codes = torch.randint(0, 16, (N, K), generator=g, device="cuda", dtype=torch.uint8)
    scale = (0.02 * torch.exp(torch.randn(N, K // group, generator=g, device="cuda"))).to(scales)
    z = torch.randint(0, 16, (N, K // group), generator=g, device="cuda", dtype=torch.uint8) if zero else None
    packed = w4.pack_w4(codes)
    if K % 128:  # what lies behind the last code is not used
        used = w4.pack_w4(torch.full_like(codes, 15))
        packed |= ~used
    return x, codes, packed, scale, z


def check_linear(x, codes, packed, scale, z):
    out = wd().linear_w4(x, packed, scale, z)
    ref, slack = B_.linear_w4(np64(x), codes.cpu().numpy(), np64(scale), None if z is None else z.cpu().numpy())
    err = np.abs(np64(out) - ref)
    assert np.all(err <= 2.0 ** -8 * np.abs(ref) + slack), float((err - slack - 2.0 ** -8 * np.abs(ref)).max())
    return out


@gpu
@pytest.mark.parametrize("T,N,K", [(1, 1, 32), (1, 16, 128), (2, 5, 256), (8, 33, 1024), (9, 31, 384), (16, 100, 2048),
                                   (17, 64, 640), (31, 17, 4096), (33, 257, 128), (64, 128, 4096), (65, 40, 512),
                                   (130, 144, 1152), (1, 1200, 4096), (3, 2500, 160), (64, 2400, 64), (20, 4736, 96)])
@pytest.mark.parametrize("kind", range(4))
def test_linear_w4(T, N, K, kind):
    group = [128, 64, 32, 32][kind]
    group = group if K % group == 0 else 32
    scales, zero = [BF16, torch.float16, F32, BF16][kind], kind % 2 == 1
    case = linear_case(T, N, K, group, scales, zero, pad=[0, 1, 0, 8][kind])
    out = check_linear(*case)
    assert torch.equal(out, wd().linear_w4(case[0], *case[2:]))  # the same bits again
    # a token's result does not hang on the others'
    one = wd().linear_w4(case[0][T - 1:], *case[2:])
    ref = np64(out[T - 1:])
    assert np.all(np.abs(np64(one) - ref) <= 2.0 ** -7 * np.abs(ref) + 1e-3)


@gpu
def test_linear_w4_odd_values():
    x, codes, packed, scale, z = linear_case(5, 48, 256, 64, F32, True)
    clean = wd().linear_w4(x, packed, scale, z)
    x[1, 7] = float("nan")
    x[3, 200] = float("inf")
    out = wd().linear_w4(x, packed, scale, z)
    assert out[1].isnan().all() and not torch.isfinite(out[3].float()).any()
    assert torch.equal(out[[0, 2, 4]], clean[[0, 2, 4]])
    scale[10, 2] = float("nan")
    scale[11] = 0
    out = wd().linear_w4(x, packed, scale, z)
    assert out[:, 10].isnan().all() and not out[[0, 2, 4], 11].any()
    assert torch.equal(out[[0, 2, 4]][:, :10], clean[[0, 2, 4]][:, :10])
    z[:] = 255  # counts as 127
    a = wd().linear_w4(x[:1], packed, scale[:, :], z)
    z[:] = 127
    assert torch.equal(a.nan_to_num(7.0), wd().linear_w4(x[:1], packed, scale, z).nan_to_num(7.0))


@gpu
def test_linear_w4_of_quantised_weights():
    w = torch.randn(96, 512, device="cuda") * 0.05
    x = torch.randn(4, 512, device="cuda").to(BF16)
    for zero_points in (False, True):
        packed, scale, zero = w4.quantize_w4(w, 64, zero_points)
        check_linear(x, w4.unpack_w4(packed, 512), packed, scale, zero)


# ---------------------------------------------------------------------------
# attention behind a shared prefix
# ---------------------------------------------------------------------------
def prefix_case(B, Sq, Hq, Hkv, D, page, prefix, lens, seed, device="cuda", spread=1.0):
    """As cache_case, the first `prefix` tokens (whole pages of them) of all sequences on the longest one's pages;
    a sequence's own table shows pages of NaN there."""
    c = cache_case(B, Sq, Hq, Hkv, D, page, lens, seed, device, spread)
    kc, ks, vc, vs, table, ln = c["np"]
    lead, shared = int(np.argmax(ln)), prefix // page
    full = table.copy()
    full[:, :min(shared, table.shape[1])] = table[lead, :min(shared, table.shape[1])]
    c["np"][4] = full
    c["prefix"] = torch.tensor([prefix], dtype=torch.int32, device=device)
    own = table.copy()
    for b in range(B):
        if b != lead:
            own[b, :min(shared, table.shape[1])] = 0 if b % 2 else -7  # not read
    c["table"] = torch.from_numpy(own).to(device)
    return c


def check_prefix(c, window=0, scale=None, q=None, workspace=None):
    q = c["q"] if q is None else q
    D = q.shape[3]
    s = 1 / D ** 0.5 if scale is None else scale
    out, lse = wd().attn_decode_fp8_prefix(q, *c["cache"], c["table"], c["lens"], c["prefix"], scale, window, workspace,
                                           True)
    kc, ks, vc, vs, table, ln = c["np"]
    ref, rlse, slack, lse_slack = R.attn(np64(q), kc, ks, vc, vs, table, ln, s, window)
    kmax, vmax = (np.nan_to_num(np.abs(R.TABLE[cc] * R.scale_values(cs)[..., None, None])) for cc, cs in ((kc, ks), (vc, vs)))
    used = np.unique(table[(table >= 0) & (table < kc.shape[0])])
    far = 2.0 ** -18 * np.nan_to_num(np.abs(np64(q)), posinf=0).max(-1) * kmax[used].sum(-1).max(initial=0) * abs(s)
    got = np64(out)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    err, fine = np.abs(got - ref), ~np.isnan(ref)
    slack = slack + 2 * far[..., None] * vmax[used].max(initial=0)
    over = err[fine] - (2.0 ** -8 * np.abs(ref) + slack)[fine] - 1e-30
    assert over.max(initial=-1) <= 0, (float(over.max()), float(err[fine].max()))
    gl = lse.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isneginf(gl), np.isneginf(rlse)) and np.array_equal(np.isnan(gl), np.isnan(rlse))
    ok = np.isfinite(rlse)
    assert np.all(np.abs(gl - rlse)[ok] <= (lse_slack + far + 4e-6 * (1 + np.abs(rlse)))[ok])
    return out, lse


PREFIX = [  # B, Sq, Hq, Hkv, D, page, prefix, lens, window
    (1, 1, 1, 1, 128, 64, 64, [65], 0),
    (2, 1, 8, 1, 128, 64, 64, [64, 100], 0),
    (4, 1, 8, 2, 128, 16, 176, [177, 200, 300, 176], 0),
    (3, 1, 32, 4, 128, 128, 256, [257, 400, 300], 0),
    (5, 2, 16, 1, 128, 64, 640, [700, 641, 655, 642, 800], 0),
    (40, 1, 8, 1, 128, 32, 320, None, 0),
    (33, 1, 8, 1, 64, 64, 1000, None, 0),
    (17, 3, 24, 3, 128, 16, 500, None, 0),
    (70, 1, 10, 2, 64, 128, 390, None, 0),
    (9, 4, 16, 2, 64, 32, 1100, None, 300),
    (6, 1, 16, 2, 128, 64, 1300, None, 129),
    (6, 2, 4, 1, 128, 64, 512, None, 1),
    (3, 1, 4, 2, 48, 16, 64, [70, 100, 65], 0),
    (2, 1, 2, 1, 192, 32, 64, [65, 90], 0),
    (2, 1, 64, 64, 128, 64, 128, [130, 140], 0),
    (2, 40, 8, 1, 128, 64, 128, [200, 300], 0),      # more than 128 rows a sequence
    (2, 30, 12, 2, 64, 16, 96, [150, 333], 0),
    (3, 1, 8, 1, 128, 64, 64, [3000, 70, 2500], 0),  # own tokens over many blocks
    (40, 1, 8, 1, 128, 128, 5000, None, 0),          # several tiles a block
    (3, 2, 16, 1, 64, 32, 9000, None, 0),
]


def own_lens(B, Sq, prefix, seed):
    g = np.random.default_rng(seed)
    return [prefix + Sq + int(g.integers(0, 150)) for _ in range(B)]


@gpu
@pytest.mark.parametrize("B,Sq,Hq,Hkv,D,page,prefix,lens,window", PREFIX)
def test_prefix(B, Sq, Hq, Hkv, D, page, prefix, lens, window):
    lens = own_lens(B, Sq, prefix, B) if lens is None else lens
    c = prefix_case(B, Sq, Hq, Hkv, D, page, prefix, lens, seed=Sq * 100 + D)
    if D not in (64, 128):
        c["table"] = torch.from_numpy(c["np"][4]).cuda()  # each sequence by itself
    out, lse = check_prefix(c, window)
    again, lse2 = wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["prefix"], None, window, None,
                                              True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix,lens", [
    (0, [40, 300]), (-5, [40, 300]), (7, [40, 300]), (64, [40, 300]), (256, [300, 40, 0, 256, 257, 10]),
    (250, [700, 120, 0, -3, 64, 63]), (10 ** 6, [300, 200]), (2 ** 31 - 1, [64, 64]), (128, [0, 0]), (128, [0, 200])])
def test_prefix_lengths(D, prefix, lens):
    """No prefix, parts of a page, sequences that end within it or are empty, a prefix past everything."""
    for Sq in (1, 3):
        c = prefix_case(len(lens), Sq, 8, 2, D, 32, min(max(prefix, 0), 1 << 20), lens, seed=Sq + len(lens))
        c["prefix"].fill_(prefix)
        check_prefix(c)
        check_prefix(c, window=50)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("D,Hq,B", [(64, 8, 3), (128, 8, 3), (128, 24, 20)])
def test_prefix_strided_queries_and_scale(D, Hq, B):
    c = prefix_case(B, 3, Hq, 2, D, 32, 200, own_lens(B, 3, 200, D), seed=8)
    big = torch.randn(B, 3, Hq * D + 2 * D + 1, device="cuda").bfloat16()
    check_prefix(c, q=big[..., 1:1 + Hq * D].unflatten(2, (Hq, D)), scale=0.5)  # off the 16-byte grid
    t = torch.randn(B, Hq, 3, D, device="cuda").bfloat16().transpose(1, 2)  # heads outside tokens
    check_prefix(c, q=t)
    check_prefix(c, q=t * 1e-3)
    check_prefix(c, scale=0.0)
    check_prefix(c, scale=-0.1)


@gpu
@pytest.mark.parametrize("D,B", [(64, 2), (128, 2), (128, 40)])
def test_prefix_growing_scores(D, B):
    """Each stretch of keys outweighs all before it by far, or less and less: the references' both ways."""
    for up in (True, False):
        c = prefix_case(B, 1, 4, 1, D, 64, 1280, own_lens(B, 1, 1280, 3), seed=5)
        kc, ks, vc, vs, table, ln = c["np"]
        for col in range(table.shape[1]):
            ks[table[:, col], 0] = 118 + col % 12 if up else 130 - col % 12
            vs[table[:, col], 0] = 100 + 3 * ((col * 5) % 11)  # values of very different magnitude
        c["cache"] = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
        check_prefix(c)


@gpu
@pytest.mark.parametrize("D,B", [(64, 3), (128, 3), (128, 30)])
def test_prefix_masked_nan_has_no_influence(D, B):
    """NaN codes and scales before the window and past a short sequence's end; a seen NaN is seen."""
    lens = [300] * B
    lens[1] = 90  # ends within the prefix
    c = prefix_case(B, 1, 8, 2, D, 16, 256, lens, seed=6)
    kc, ks, vc, vs, table, ln = c["np"]
    vc[table[0, 6], 0, 3, 5] = 0x7F   # position 99, value 5, key head 0: not seen by sequence 1
    vs[table[0, 7], 0] = 255          # positions 112 to 127
    kc[table[0, 1], 1, 5] = 0xFF      # position 21, key head 1
    c["cache"] = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
    out, _ = check_prefix(c)
    assert out[0, 0, :4].isnan().all() and out[2, 0, 4:].isnan().all() and not out[1, 0, :4].isnan().any()
    out, _ = check_prefix(c, window=150)   # of 300, position 151 on
    assert not out[0].isnan().any() and not out[2].isnan().any()
    vs[table[0, 7], 0] = 120
    c["cache"] = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
    out, _ = check_prefix(c)
    assert out[0, 0, 0, 5].isnan() and out[0, 0, 0].isnan().sum() == 1
    q = c["q"].clone()
    q[2, 0, 1, 7] = float("inf")  # makes its row NaN, and no other
    out, _ = wd().attn_decode_fp8_prefix(q, *c["cache"], c["table"], c["lens"], c["prefix"], return_lse=True)
    assert out[2, 0, 1].isnan().all() and out[1, 0, :4].isfinite().all() and out[2, 0, 2].isnan().sum() == 1


@gpu
@pytest.mark.parametrize("D,B", [(128, 2), (64, 2), (128, 35)])
def test_prefix_bad_pages_are_masked(D, B):
    c = prefix_case(B, 1, 8, 2, D, 16, 128, [200] * B, seed=7)
    full, own = c["np"][4], c["table"].cpu().numpy()
    full[:, 3], own[0, 3] = -5, -5
    full[:, 5], own[0, 5] = 1 << 30, 1 << 30
    full[1, 9], own[1, 9] = -1, -1
    c["table"] = torch.from_numpy(own).cuda()
    check_prefix(c)
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE
    full[:, :8], own[:, :8] = -1, -1  # nothing left of the prefix
    c["table"] = torch.from_numpy(own).cuda()
    check_prefix(c)
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE


@gpu
def test_prefix_equals_attention_on_full_tables():
    c = prefix_case(8, 2, 16, 2, 128, 64, 600, own_lens(8, 2, 600, 1), seed=3)
    full = torch.from_numpy(c["np"][4]).cuda()
    a = wd().attn_decode_fp8(c["q"], *c["cache"], full, c["lens"])
    b = wd().attn_decode_fp8_prefix(c["q"], *c["cache"], full, c["lens"], c["prefix"])
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -7 * a.float().abs().max()
    for cols in (0,):  # no table at all
        out, lse = wd().attn_decode_fp8_prefix(c["q"], *c["cache"], full[:, :cols].contiguous(), c["lens"], c["prefix"],
                                               return_lse=True)
        assert not out.any() and torch.isneginf(lse).all()
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE


@gpu
def test_prefix_workspace_streams_and_graphs():
    """One workspace for calls of different sizes, in a row, on a stream of their own, and in a graph."""
    cases = [prefix_case(3, 1, 16, 2, 128, 64, 1000, [1001, 1100, 1050], seed=1),
             prefix_case(30, 2, 8, 1, 128, 32, 320, own_lens(30, 2, 320, 2), seed=2),
             prefix_case(2, 1, 8, 8, 64, 16, 64, [700, 70], seed=3)]
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    call = lambda c: wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["prefix"],  # noqa: E731
                                                 workspace=ws)
    plain = [check_prefix(c)[0] for c in cases]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            for c, p in zip(cases, plain):
                assert torch.equal(call(c), p)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [call(c) for c in cases]
    for _ in range(2):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, p) for o, p in zip(outs, plain))
    # the prefix is read by the kernels, not when the graph was made
    c = cases[2]
    c["table"].copy_(torch.from_numpy(c["np"][4]))
    for n in (0, 16, 48):
        c["prefix"].fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        ref, _, slack, _ = R.attn(np64(c["q"]), *c["np"][:5], c["np"][5], 64 ** -0.5, 0)
        assert np.all(np.abs(np64(outs[2]) - ref) <= 2.0 ** -8 * np.abs(ref) + 2 * slack)
    assert wd().status(True, 0) == 0


@gpu
def test_prefix_on_two_streams_at_once():
    cases = [prefix_case(20, 1, 16, 2, 128, 64, 900, own_lens(20, 1, 900, s), seed=s) for s in (11, 12)]
    call = lambda c, ws=None: wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["prefix"],  # noqa: E731
                                                          workspace=ws)
    plain = [call(c) for c in cases]
    spaces = [wd().attn_decode_fp8_prefix_workspace(20, 1, 16, 2, 128) for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                outs[i].append(call(c, spaces[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, plain[i]) for i in range(2) for o in outs[i])
    assert wd().status(True, 0) == 0


@gpu
def test_shared_prefix_example():
    """Every operator of a layer's step together, against plain fp32 torch on the cache's values.

    The steps round to bf16 eight times in a row, 2^-9 of a row's norm each, and an expert whose choice value ties
    within that may differ; the seed's values have no such tie. 1e-2 of a row's norm.
    """
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "shared_prefix_step.py"
    spec = importlib.util.spec_from_file_location("shared_prefix_step", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main() <= 1e-2


@gpu
def test_operators_on_another_stream_and_captured():
    """Norm and projections on a stream of their own and replayed from a graph: the bits of plain calls."""
    y, r = torch.randn(40, 1024, device="cuda").to(BF16), torch.randn(40, 1024, device="cuda").to(BF16)
    w = torch.ones(1024, device="cuda")
    x, codes, packed, scale, z = linear_case(20, 300, 1024, 64, BF16, True)
    big_y, big_r = torch.randn(1200, 2048, device="cuda").to(BF16), torch.randn(1200, 2048, device="cuda").to(BF16)
    big_w = torch.ones(2048, device="cuda", dtype=BF16)
    call = lambda: (*wd().block_norm(y, r, w, w), *wd().block_norm(big_y, big_r, big_w, big_w, big_w),  # noqa: E731
                    wd().linear_w4(x, packed, scale, z), wd().linear_w4(x[:2], packed, scale, z))
    plain = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(call(), plain))
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for _ in range(2):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, plain))
    # inputs are read when the graph runs
    y.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wd().block_norm(y, r, w, w)[0])
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("T,H", [(700, 1024), (600, 1032), (601, 4096), (592, 7168), (900, 16384), (1185, 2056)])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("residual", [BF16, F32])
def test_block_norm_of_many_rows(T, H, gate, residual):
    """Blocks that take several rows each, with both types of weights and every gate."""
    g = torch.Generator(device="cuda").manual_seed(T + H)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    y, r = rand(T, H).to(BF16), (rand(T, H) * 2).to(residual)
    shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[gate]
    for wt in (BF16, F32):
        w, post = (1 + 0.2 * rand(H)).to(wt), (1 + 0.2 * rand(H)).to(wt)
        ga = None if shape is None else rand(*shape).to(F32 if wt == BF16 else BF16)
        check_norm(y, r, w, post if gate != "token" else None, ga, 0.5)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("T,H", [(7200, 1024), (7300, 1000), (3601, 2056), (1801, 4096)])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
def test_block_norm_of_more_rows(T, H, gate):
    """Rows enough that blocks take several each at narrower widths too, and as many of a width that does not."""
    for residual in (BF16, F32):
        test_block_norm_of_many_rows(T, H, gate, residual)
