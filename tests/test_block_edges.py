"""The operators that complete a decoder layer's step where they can go wrong: values, sizes
and calls beside those of test_block_ops.py, against the same 64-bit restatements.

Tolerances: half a step of the output's type plus the restatement's bound.
"""
import re

import numpy as np
import pytest
import torch

from oracle import layer_ref as R
from test_block_ops import check_linear, check_norm, check_prefix, linear_case, own_lens, prefix_case
from test_layer_ops import np64, wd
from warp_decode_b200 import _build, w4

gpu = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
BF16_MAX = float(torch.finfo(BF16).max)


# ---------------------------------------------------------------------------
# attention behind a shared prefix
# ---------------------------------------------------------------------------
def prefix_spread(c, window=0, weight=2.0 ** -11, quantum=2.0 ** -31):
    """The operator on the case against the restatement with errors that add up as independent ones do.

    A weight is rounded to fp16: half a step, 2^-11 of itself, or 2^-25 where it is less than 2^-14,
    when the row's largest is 2^6 at least.
    """
    out, lse = wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["prefix"], None, window, None,
                                           True)
    D = c["q"].shape[3]
    ref, spread = R.attn_spread(np64(c["q"]), *c["np"], D ** -0.5, window, weight=weight, quantum=quantum)
    _, rlse, _, lse_slack = R.attn(np64(c["q"]), *c["np"], D ** -0.5, window)
    got, tol = np64(out), 2.0 ** -8 * np.abs(ref) + spread + 2.0 ** -133  # the least bf16 value above 0
    over = np.abs(ref) - tol > BF16_MAX  # what bf16 does not hold is infinite
    assert np.array_equal(got[over], np.sign(ref[over]) * np.inf)
    held = np.abs(ref) + tol <= BF16_MAX
    err = np.abs(got - ref)[held] - tol[held]
    assert not np.isnan(got).any() and err.max(initial=-1) <= 0, float((err / tol[held]).max())
    gl = lse.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isneginf(gl), np.isneginf(rlse))
    ok = np.isfinite(rlse)
    assert np.all(np.abs(gl - rlse)[ok] <= (lse_slack + 4e-6 * (1 + np.abs(rlse)))[ok])
    return out


def on_the_gpu(c, *arrays):
    c["cache"] = [torch.from_numpy(a).cuda() for a in arrays]


@gpu
@pytest.mark.parametrize("D,B", [(64, 3), (128, 3), (128, 40)])
@pytest.mark.parametrize("kind", ["largest", "masked", "mixed", "least"])
def test_prefix_value_scales(D, B, kind):
    """Every scale of V that the cache can hold: weights above 1 of values next to fp32's largest, values past
    bf16's in pages that a row does not see, scales of all magnitudes together, and the least ones."""
    lens = [500] * B
    lens[1] = 90  # ends within the prefix
    c = prefix_case(B, 1, 8, 2, D, 16, 320, lens, seed=9)
    kc, ks, vc, vs, table, ln = c["np"]
    g = np.random.default_rng(D + B)
    if kind == "largest":
        vs[:] = 246                 # up to 448 * 2^119
        for col in range(table.shape[1]):
            ks[table[:, col]] += min(col // 6, 3)  # later scores are larger, but references need not move
    elif kind == "masked":
        vs[table[0, 6:]] = 254      # tokens from 96 on
    elif kind == "mixed":
        vs[:] = g.integers(0, 255, vs.shape)
        ks[:] = 120 + g.integers(-2, 3, ks.shape)
    else:
        vs[:] = g.integers(0, 9, vs.shape)
    on_the_gpu(c, kc, ks, vc, vs)
    out = prefix_spread(c)
    if kind == "masked":
        assert out[1].isfinite().all() and out[1].abs().max() > 0
    prefix_spread(c, window=77)
    assert wd().status(True, 0) == 0


def joined_case(B, Sq, Hq, Hkv, D, page, prefix, own, seed, spread=0.3):
    """A case whose keys spread so little that thousands of them share the weight."""
    return prefix_case(B, Sq, Hq, Hkv, D, page, prefix, [prefix + n for n in own], seed=seed, spread=spread)


@gpu
@pytest.mark.parametrize("B,Sq,Hq,Hkv,D,page,prefix", [(3, 1, 8, 1, 128, 64, 1000), (40, 1, 8, 2, 64, 16, 700),
                                                       (5, 3, 16, 1, 128, 32, 900), (2, 1, 8, 1, 128, 128, 20000),
                                                       (150, 1, 8, 1, 128, 64, 256)])
def test_prefix_is_as_exact_as_its_output(B, Sq, Hq, Hkv, D, page, prefix):
    """Weights of eleven bits: the distance from 64 bits is the output's own rounding.

    Errors of weights are an eighth of the output's, random over the keys, and those of scores
    (2^-18 of q's largest value) less: together they add 1 % to its root mean square, 5 % are allowed.
    """
    c = joined_case(B, Sq, Hq, Hkv, D, page, prefix, [Sq + i % 90 for i in range(B)], seed=B + D)
    got = np64(prefix_spread(c))
    ref, _ = R.attn_spread(np64(c["q"]), *c["np"], D ** -0.5, 0)
    half = np64(torch.from_numpy(ref).to(BF16)) - ref
    assert np.sqrt(np.square(got - ref).mean()) <= 1.05 * np.sqrt(np.square(half).mean())


@gpu
@pytest.mark.parametrize("B,D", [(2, 128), (40, 128), (3, 64)])
@pytest.mark.parametrize("n,score", [(8192, 12.0), (65536, 14.0), (65536, 17.0)])
def test_prefix_strong_key_over_a_long_tail(B, D, n, score):
    """Weights down to 2^-24 of the row's largest, whose own values are 0: the tail is the output."""
    g = np.random.default_rng(n + D + int(10 * score))
    page, own = 128, 5
    k, v = 0.2 * g.standard_normal((1, n + own, 1, D)), 1 + 0.3 * g.standard_normal((1, n + own, 1, D))
    k[..., 0], k[0, 0, 0, 0] = 0.3 * g.standard_normal((1, n + own, 1)), score
    v[0, 0] = 0.0
    P = -(-(n + own) // page)
    kc, vc = (np.zeros((P, 1, page, D), np.uint8) for _ in range(2))
    ks, vs = (np.zeros((P, 1), np.uint8) for _ in range(2))
    one = np.arange(P, dtype=np.int32)[None]
    R.kv_write(k, kc, ks, one, [0], [n + own])
    R.kv_write(v, vc, vs, one, [0], [n + own])
    q = np.zeros((1, 1, 8, D))
    q[..., 0] = 1.0
    ref, spread = R.attn_spread(q[:, :, :1], kc, ks, vc, vs, one, [n + own], 1.0, 0, weight=2.0 ** -11, quantum=2.0 ** -31)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    lens = torch.full((B,), n + own, dtype=torch.int32, device="cuda")
    out = wd().attn_decode_fp8_prefix(up(q).bfloat16().expand(B, -1, -1, -1), up(kc), up(ks), up(vc), up(vs),
                                      up(one).repeat(B, 1), lens, lens[:1] - own, 1.0)
    assert torch.equal(out, out[:1, :, :1].expand_as(out))
    assert np.median(spread / ref) < 0.1  # the bound tells a lost tail from one that is there
    got = np64(out[:1, :, :1])
    assert np.all(np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + spread), (got.mean(), ref.mean(), spread.mean())


def random_codes(g, B, Sq, Hq, Hkv, D, page, prefix, lens):
    """As prefix_case, with codes drawn as such: every value but NaN alike, three scales."""
    shared, most = prefix // page, -(-max(lens) // page)
    P = shared + B * (most - shared)
    pool = g.permutation(P).astype(np.int32)
    own = pool[shared:].reshape(B, most - shared)
    table = np.concatenate([np.broadcast_to(pool[:shared], (B, shared)), own], 1)
    kc, vc = (g.integers(0, 256, (P, Hkv, page, D), np.uint8) for _ in range(2))
    for a in (kc, vc):
        a[(a & 0x7F) == 0x7F] = 0x38  # 1
    ks, vs = (g.integers(116, 119, (P, Hkv)).astype(np.uint8) for _ in range(2))
    ln = np.asarray(lens, np.int32)
    q = torch.from_numpy(g.standard_normal((B, Sq, Hq, D)).astype(np.float32)).cuda().to(BF16)
    mine = table.copy()
    mine[np.arange(B) != int(np.argmax(ln)), :shared] = -7  # not read
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return dict(q=q, cache=[up(a) for a in (kc, ks, vc, vs)], table=up(mine), lens=up(ln), np=[kc, ks, vc, vs, table, ln],
                prefix=torch.tensor([prefix], dtype=torch.int32, device="cuda"))


@gpu
@pytest.mark.parametrize("B,Sq,Hq,Hkv,D,page,prefix,own,window", [
    (128, 1, 32, 4, 128, 128, 16384, 256, 0), (64, 4, 32, 4, 64, 16, 12001, 700, 0), (16, 4, 32, 4, 128, 16, 12001, 1000, 5000),
    (300, 1, 8, 8, 64, 32, 300, 40, 0), (256, 1, 16, 1, 128, 64, 4096, 300, 4200), (2, 1, 8, 2, 128, 128, 131072, 2000, 0),
    (700, 1, 8, 1, 64, 64, 2000, 20, 100)])
def test_prefix_of_large_sizes(B, Sq, Hq, Hkv, D, page, prefix, own, window):
    """Batches, prefixes and windows of the sizes in use: some sequences of each against 64 bits, every one the same again."""
    g = np.random.default_rng(B + prefix)
    lens = [prefix + int(n) for n in g.integers(Sq, own + 1, B)]
    lens[B // 2] = max(1, prefix // 3)  # ends within the prefix
    c = random_codes(g, B, Sq, Hq, Hkv, D, page, prefix, lens)
    call = lambda: wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["prefix"], None, window)  # noqa: E731
    out = call()
    kc, ks, vc, vs, table, ln = c["np"]
    for b in sorted({0, B // 2, B - 1, int(np.argmax(ln)), int(g.integers(B))}):
        ref, spread = R.attn_spread(np64(c["q"][b:b + 1]), kc, ks, vc, vs, table[b:b + 1], ln[b:b + 1], D ** -0.5, window,
                                    weight=2.0 ** -11, quantum=2.0 ** -31)
        err = np.abs(np64(out[b:b + 1]) - ref)
        assert np.all(err <= 2.0 ** -8 * np.abs(ref) + spread), (b, float((err / (2.0 ** -8 * np.abs(ref) + spread)).max()))
    assert torch.equal(out, call())
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("D,B", [(64, 3), (128, 3), (128, 40)])
def test_prefix_queries_of_all_magnitudes(D, B):
    """Query rows of zeros, of bf16's least numbers, of one large value, and of values next to the largest."""
    c = prefix_case(B, 2, 8, 1, D, 32, 200, own_lens(B, 2, 200, D), seed=12)
    q = c["q"]
    q[0] = 0.0
    q[1, 0, 0] = 2.0 ** -133
    q[1, 0, 1] *= 2.0 ** -126
    q[1, 0, 2] = 0.0
    q[1, 0, 2, 5] = 3.0
    q[1, 1, :4, 7] *= 2.0 ** 12  # the others' eight bits are twelve octaves below
    q[2] *= 2.0 ** 100
    kc, ks, vc, vs, table, ln = c["np"]
    for col in range(200 // 32, table.shape[1]):  # so that sequence 2's own scores are small again
        ks[table[2, col]] = np.maximum(ks[table[2, col]].astype(int) - 100, 0)
    on_the_gpu(c, kc, ks, vc, vs)
    check_prefix(c)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_prefix_shares_a_workspace_with_attention(D):
    """Calls of both operators in turn, over sequences that several blocks share, leave it ready for each other."""
    c = prefix_case(3, 1, 16, 2, D, 64, 4096, [4100, 9000, 20000], seed=4)
    full = torch.from_numpy(c["np"][4]).cuda()
    ws = torch.zeros(32 << 20, dtype=torch.uint8, device="cuda")
    decode = lambda w: wd().attn_decode_fp8(c["q"], *c["cache"], full, c["lens"], workspace=w)  # noqa: E731
    prefix = lambda w: wd().attn_decode_fp8_prefix(c["q"], *c["cache"], c["table"], c["lens"], c["prefix"],  # noqa: E731
                                                   workspace=w)
    a, b = decode(None), prefix(None)
    for _ in range(3):
        assert torch.equal(prefix(ws), b)
        assert not ws[:2048].any()  # the counters of attn_decode_fp8
        assert torch.equal(decode(ws), a)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("D,Hq,Hkv", [(48, 4, 2), (80, 8, 1), (192, 2, 1), (256, 16, 4)])
@pytest.mark.parametrize("prefix,lens", [(64, [70, 100, 65]), (100, [200, 120, 200, 90]), (10 ** 6, [77, 300, 10, 0]),
                                         (-3, [40, 20]), (0, [40, 20]), (128, [0, 0, 0]), (64, [-2, 3, 130])])
def test_prefix_of_other_head_sizes(D, Hq, Hkv, prefix, lens):
    """The shared pages come from the longest sequence's table, whatever the others' show there."""
    for Sq, window in ((1, 0), (3, 50)):
        c = prefix_case(len(lens), Sq, Hq, Hkv, D, 16, min(max(prefix, 0), 1 << 20), lens, seed=D + Sq)
        c["prefix"].fill_(prefix)
        check_prefix(c, window)
    assert wd().status(True, 0) == 0


# ---------------------------------------------------------------------------
# block norm
# ---------------------------------------------------------------------------
@gpu
def test_block_norm_in_place_overlaps():
    """In place, rows that another input reads are refused however they lie, and rows between them are not."""
    H = 64
    norm = lambda y, r, w, **kw: wd().block_norm(y, r, w, inplace=True, **kw)  # noqa: E731
    w = torch.ones(H, device="cuda", dtype=BF16)
    big = torch.randn(9, 2 * H + 16, device="cuda").to(BF16)
    wide = torch.randn(9, H + 8, device="cuda").to(BF16)
    refused = [
        (wide[:-1, :H], wide[1:, :H], w, {}),                  # padded rows, one further
        (wide[:, 8:], wide[:, :H], w, {}),                     # columns that meet
        (big[:-1, H:2 * H], big[1:, 2 * H + 16 - H:], w, {}),  # columns that meet, one row further
        (big[:, 2 * H + 16 - H:], big[:, 17:17 + H], w, {}),    # by one value
        (big.as_strided((5, H), (2 * H, 1)), big[:5, :H], w, {}),             # of another stride
        (big.as_strided((5, H), (0, 1), 3 * (2 * H + 16)), big[:5, :H], w, {}),  # one row for all
        (wide[:4, :H].clone(), big[:4, :H], big[2, :H], {}),                  # the weights
        (wide[:4, :H].clone(), big[:4, :H], w, {"post_weight": big[1, H - 1:2 * H - 1]}),
        (wide[:4, :H].clone(), big[:4, :H], w, {"gate": big[:4, H - 1:H]}),
        (wide[:4, :H].clone(), big[:4, :H], w, {"gate": big[3, :H]}),
    ]
    for y, r, weight, kw in refused:
        before = big.clone(), wide.clone()
        with pytest.raises(RuntimeError, match="memory location"):
            norm(y, r, weight, **kw)
        assert torch.equal(big, before[0]) and torch.equal(wide, before[1])
    taken = [
        (big[:, H:2 * H], big[:, :H], w, {}),
        (big[1:, :H], big[:-1, H + 16:], w, {}),
        (big.as_strided((2, H), (8 * (2 * H + 16), 1), H), big[:2, :H], w, {}),  # of another stride, between
        (wide[:4, :H].clone(), big[:4, :H], big[6, :H].clone(), {"gate": big[:4, H:H + 1]}),
        (wide[:4, :H].clone(), big[:4, :H], big[2, H:2 * H], {"gate": big[5, :H]}),  # weights beside the rows
    ]
    for y, r, weight, kw in taken:
        x, out = wd().block_norm(y, r, weight, **kw)
        rest = big.clone()
        x2, out2 = norm(y, r, weight, **kw)
        assert torch.equal(x, x2) and torch.equal(out, out2) and out2.data_ptr() == r.data_ptr()
        at = (r.data_ptr() - big.data_ptr()) // 2
        rest.as_strided(r.shape, r.stride(), at).copy_(out)
        assert torch.equal(rest, big)


@gpu
def test_block_norm_of_the_most_rows():
    """2^31 - 1 rows of one value each: the rows' number is rounded up to whole blocks."""
    T = 2 ** 31 - 1
    one = lambda v, t: torch.full((1, 1), v, device="cuda", dtype=t).expand(T, 1)  # noqa: E731
    x, out = wd().block_norm(one(3.0, BF16), one(-1.0, BF16), torch.full((1,), 0.5, device="cuda", dtype=BF16))
    assert bool((out == 2.0).all()) and bool((x == 0.5).all())  # 2 rsqrt(4 + 1e-6) is within 2^-20 of 1


# Rows enough for the kernel whose blocks stay and copy rows ahead: 49152 values an SM from 1024 wide, four rows an SM
# from 4096.
STREAMED = [(7200, 1024), (4000, 2048), (1801, 4096), (3601, 2056), (900, 7168), (600, 16384)]


def streamed(T, H):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return H % 8 == 0 and (T >= 4 * sms if H > 4096 else H >= 1024 and T * H >= 49152 * sms)


@gpu
@pytest.mark.parametrize("T,H", STREAMED)
@pytest.mark.parametrize("kind", range(6))
def test_block_norm_streamed(T, H, kind):
    """Padded rows, every gate and type, in place too: the same bits, and the values beside the rows untouched."""
    assert streamed(T, H)
    g = torch.Generator(device="cuda").manual_seed(T + H + kind)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    pad = 8 * (kind % 2)
    y = (rand(T, H + 24)[:, pad:pad + H] * 2).to(BF16) if kind < 4 else (rand(T, H + 24) * 2).to(BF16)[:, 16 - pad:16 - pad + H]
    big = (rand(T, H + 40) * 3).to(BF16 if kind < 3 else F32)
    r = big[:, pad:pad + H]
    wt = F32 if kind in (1, 4) else BF16
    w, post = (1 + 0.2 * rand(H)).to(wt), (1 + 0.2 * rand(H)).to(wt) if kind % 3 else None
    gate = [None, rand(H), rand(T, 1).to(BF16), rand(T, H + 8).to(BF16)[:, :H], rand(1, H).to(BF16).expand(T, H),
            rand(T, 1).expand(T, H)][kind]
    scale = 0.5 if kind == 2 else 1.0
    x, out = check_norm(y, r, w, post, gate, scale)
    keep = big.clone()
    x2, out2 = wd().block_norm(y, r, w, post, gate, scale, inplace=True)
    assert out2.data_ptr() == r.data_ptr() and torch.equal(x2, x) and torch.equal(r, out)
    keep[:, pad:pad + H] = out
    assert torch.equal(big, keep)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("T,H", [(4000, 2048), (900, 7168)])
def test_block_norm_streamed_odd_values(T, H):
    """NaN and infinities stay in their rows, whatever row the block has next; infinite gates of a token."""
    assert streamed(T, H)
    y, r = torch.randn(T, H, device="cuda").to(BF16), torch.randn(T, H, device="cuda").to(BF16)
    w = torch.ones(H, device="cuda", dtype=BF16)
    clean = wd().block_norm(y, r, w, w)
    odd = torch.randperm(T, generator=torch.Generator().manual_seed(T))[:200].cuda()
    y2, r2 = y.clone(), r.clone()
    y2[odd[:50], 3] = float("nan")
    r2[odd[50:100], H - 1] = float("nan")
    y2[odd[100:150], 5] = float("inf")
    y2[odd[150:]], r2[odd[150:]] = 0, 0
    x, out = wd().block_norm(y2, r2, w, w)
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[odd] = False
    assert torch.equal(x[rest], clean[0][rest]) and torch.equal(out[rest], clean[1][rest])
    assert x[odd[:100]].isnan().all() and out[odd[:50]].isnan().all() and out[odd[50:100], H - 1].isnan().all()
    assert x[odd[100:150]].isnan().any(1).all() and not x[odd[150:]].any() and not out[odd[150:]].any()
    gate = torch.ones(T, 1, device="cuda")
    gate[odd] = float("inf")
    y[y == 0] = 1.0
    x, out = wd().block_norm(y, r, w, None, gate)
    plain = wd().block_norm(y, r, w)
    assert torch.isinf(out[odd]).all() and torch.equal(out[rest], plain[1][rest]) and torch.equal(x[rest], plain[0][rest])


@gpu
def test_block_norm_streamed_on_another_stream_and_captured():
    T, H = 3601, 2048
    assert streamed(T, H)
    y, r = torch.randn(T, H, device="cuda").to(BF16), torch.randn(T, H, device="cuda")
    w, gate = torch.randn(H, device="cuda").to(BF16), torch.randn(T, 1, device="cuda")
    call = lambda: wd().block_norm(y, r, w, w, gate, 0.5)  # noqa: E731
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
    y.mul_(2)  # inputs are read when the graph runs
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, call()))
    assert wd().status(True, 0) == 0


# ---------------------------------------------------------------------------
# 4-bit projection
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("N,K", [(0, 128), (3, 0), (0, 0), (0, 160)])
def test_w4_packing_of_nothing(N, K):
    packed = w4.pack_w4(torch.zeros(N, K, dtype=torch.uint8))
    assert packed.shape == (N, -(-K // 128) * 64) and w4.unpack_w4(packed, K).shape == (N, K)
    if K % 32 == 0 and K:
        packed, scale, zero = w4.quantize_w4(torch.zeros(N, K), 32, True)
        assert packed.shape[0] == 0 and scale.shape == zero.shape == (0, K // 32)
        assert w4.dequantize_w4(packed, scale, zero, K).shape == (0, K)


@pytest.mark.parametrize("dtype,value", [(torch.uint8, 16), (torch.int32, -1), (torch.int32, 271), (torch.int64, 1 << 40),
                                         (F32, 3.7), (F32, float("nan")), (F32, -1.0)])
def test_w4_packing_refuses_other_codes(dtype, value):
    """Codes that a byte would bring into range, too."""
    codes = torch.full((2, 40), 7, dtype=dtype)
    assert torch.equal(w4.unpack_w4(w4.pack_w4(codes), 40), codes.to(torch.uint8))
    codes[1, 39] = value
    with pytest.raises(ValueError, match="0 to 15"):
        w4.pack_w4(codes)


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype,value", [(BF16, float("nan")), (F32, float("inf")), (torch.float16, 1e6), (BF16, -float("inf"))])
def test_w4_quantiser_refuses_what_has_no_scale(zero_points, dtype, value):
    w = torch.randn(4, 64, generator=torch.Generator().manual_seed(1))
    w4.quantize_w4(w, 32, zero_points, dtype)
    w[2, 40] = value
    with pytest.raises(ValueError, match="finite"):
        w4.quantize_w4(w, 32, zero_points, dtype)


# ---------------------------------------------------------------------------
# the build
# ---------------------------------------------------------------------------
def test_every_included_file_makes_its_target_stale():
    for sources, deps in ((_build.LIB_SOURCES, _build.LIB_DEPS), (_build.LAYER_SOURCES, _build.LAYER_DEPS),
                          (_build.BLOCK_SOURCES, _build.BLOCK_DEPS), (_build.EXT_SOURCES, _build.EXT_DEPS)):
        todo, seen = list(sources), set()
        while todo:
            path = todo.pop()
            seen.add(path)
            for name in re.findall(r'^#include "([^"]+)"', path.read_text(), re.M):
                found = [d / name for d in (_build.CSRC, _build.INCLUDE) if (d / name).exists()]
                todo += [f for f in found if f not in seen]
        assert len(seen) > len(sources) and not seen - set(deps), seen - set(deps)


# At least two trips round the four stages of codes and of x, and so four of a converting
# group's two registers: a row of 128 k a step is shared by eight blocks at most.
LONG_ROWS = [(64, 40, 16384, 128), (16, 100, 8192, 64), (33, 130, 16384, 32), (20, 257, 16352, 32), (9, 17, 16320, 64),
             (64, 9216, 4096, 128), (16, 4096, 8192, 64), (130, 300, 9216, 128), (64, 19000, 2048, 128), (12, 64, 65536, 32)]


@gpu
@pytest.mark.parametrize("T,N,K,group", LONG_ROWS)
@pytest.mark.parametrize("scales,zero", [(BF16, False), (torch.float16, True), (F32, False)])
def test_linear_w4_of_long_rows(T, N, K, group, scales, zero):
    tiles = -(-N // 128) * -(-T // (16 if T <= 16 else 32 if T <= 32 else 64))
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert T > 8 and -(-K // 128) >= 8 * (8 if tiles * 8 <= sms else 4 if tiles * 4 <= sms else 2 if tiles * 2 <= sms else 1)
    case = linear_case(T, N, K, group, scales, zero, pad=8 * (T % 2))
    out = check_linear(*case)
    assert torch.equal(out, wd().linear_w4(case[0], *case[2:]))


@gpu
def test_linear_w4_of_a_prompt():
    """A prompt's token tiles, the last one ragged, together and each by itself.

    Both hold to the bound. Their bits may differ: a call's blocks share k by the number of its tiles, and sums of
    fp32 go in that order.
    """
    x, codes, packed, scale, z = linear_case(333, 260, 2048, 64, BF16, True)
    check_linear(x, codes, packed, scale, z)
    for t in range(0, 333, 64):
        check_linear(x[t:t + 64], codes, packed, scale, z)
