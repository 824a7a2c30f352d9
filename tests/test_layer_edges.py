"""Edges of the operators around the FFN that tests/test_layer_ops.py does not reach.

Its tolerances hold here too where a test names no other.
"""

import numpy as np
import pytest
import torch

from oracle import layer_ref as R
from test_layer_ops import SHAPES, cache_case, check_attn, check_rows_close, np64, read_call, wd, write_call
from warp_decode_b200 import capi

gpu = pytest.mark.gpu

LONG = [(1, 1, 4, 1, 128, 128, [20011], 0), (2, 3, 16, 1, 128, 128, [9000, 130], 0), (1, 5, 13, 1, 128, 128, [12345], 0),
        (1, 1, 6, 2, 64, 32, [15000], 0), (3, 2, 24, 2, 128, 64, [6000, 2500, 9], 4000)]

TILE, UNIT_COST, MIN_SHARE = 128, 2, 3  # keys of a tile, a unit's fixed cost and the least share in tiles


def split_pieces(lens, ctas):
    """Split pieces of each CTA's share when every sequence is one unit of whole tiles."""
    tiles = [max(1, -(-n // TILE)) for n in lens]
    total = sum(tiles) + UNIT_COST * len(lens)
    ctas = min(ctas, max(1, total // MIN_SHARE))
    first = [i * (total // ctas) + min(i, total % ctas) for i in range(ctas + 1)]
    split, at = [0] * ctas, 0
    for n in tiles:
        lo, hi = at + UNIT_COST, at + UNIT_COST + n
        for i in range(ctas):
            a, z = max(lo, first[i]), min(hi, first[i + 1])
            split[i] += a < z and (a > lo or z < hi)
        at = hi
    return split


def test_a_share_has_two_split_pieces_at_most():
    g = np.random.default_rng(0)
    for _ in range(200):
        lens = g.integers(0, 3000, int(g.integers(1, 200))).tolist()
        assert max(split_pieces(lens, 148)) <= 2


@gpu
@pytest.mark.parametrize("D,Hq", [(128, 8), (128, 32), (128, 64), (64, 8)])
def test_attention_shares_of_two_split_pieces(D, Hq):
    """Most shares end one unit and begin the next, with nothing between: both pieces go through the workspace."""
    lens = [16 * TILE] * 100
    assert sum(n == 2 for n in split_pieces(lens, 148)) > 50
    c = cache_case(100, 1, Hq, 1, D, 128, lens, seed=D + Hq)
    out, lse = check_attn(c)
    ws = wd().attn_decode_fp8_workspace(100, 1, Hq, 1, D)
    for _ in range(50):
        again, lse2 = wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], workspace=ws, return_lse=True)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert wd().status(True, 0) == 0


def fill_stages_with_nan(D):
    """A call whose K and V are NaN codes, on every CTA: what it leaves in shared memory must not matter to the next."""
    codes = torch.full((4, 1, 128, D), 0x7F, dtype=torch.uint8, device="cuda")
    scale = torch.full((4, 1), 127, dtype=torch.uint8, device="cuda")
    table = torch.arange(4, dtype=torch.int32, device="cuda").repeat(300, 4)
    q = torch.ones(300, 1, 8, D, dtype=torch.bfloat16, device="cuda")
    lens = torch.full((300,), 2048, dtype=torch.int32, device="cuda")
    wd().attn_decode_fp8(q, codes, scale, codes, scale, table, lens)


@gpu
@pytest.mark.parametrize("D", [64, 128, 48])
@pytest.mark.parametrize("lens,window,Sq", [([200], 0, 1), ([300], 0, 3), ([1000, 64], 0, 1), ([70, 190], 0, 2),
                                            ([1152], 128, 1), ([1153], 129, 1), ([1300, 100], 256, 4)])
def test_attention_lengths_past_the_table(D, lens, window, Sq):
    """Tokens past the table's last column are masked wherever its end lies in a tile of keys."""
    reach = 64
    c = cache_case(len(lens), Sq, 8, 2, D, 16, [reach] * len(lens), seed=sum(lens))
    fill_stages_with_nan(D)
    check_attn(c, window, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE


@gpu
@pytest.mark.parametrize("D", [64, 128, 48])
@pytest.mark.parametrize("length", [128, 300])
def test_attention_lengths_without_columns(D, length):
    c = cache_case(2, 1, 8, 2, D, 16, [20, 3], seed=length)
    fill_stages_with_nan(D)
    lens = torch.tensor([length, 0], dtype=torch.int32, device="cuda")
    out, lse = wd().attn_decode_fp8(c["q"], *c["cache"], torch.zeros(2, 0, dtype=torch.int32, device="cuda"), lens,
                                    return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()
    assert wd().status(True, 0) == capi.WD_STATUS_BAD_PAGE


@gpu
@pytest.mark.parametrize("D,Hq", [(128, 4), (128, 24), (128, 64), (64, 4), (64, 24), (64, 64), (48, 4)])
@pytest.mark.parametrize("length", [100, 1000, 20000])
def test_attention_nan_and_infinite_queries(D, Hq, length):
    """A row of q with a NaN or an infinity gives NaN however its sequence is split; the rows beside it are untouched."""
    c = cache_case(1, 1, Hq, 1, D, 128, [length], seed=length + Hq)
    c["q"][0, 0, 1, 5] = float("nan")
    c["q"][0, 0, 3, 0] = float("inf")
    out, lse = check_attn(c)
    bad = torch.zeros(Hq, dtype=torch.bool, device="cuda")
    bad[[1, 3]] = True
    assert torch.equal(out[0, 0].isnan().all(-1), bad) and torch.equal(lse[0, 0].isnan(), bad)
    assert wd().status(True, 0) == 0


@gpu
@pytest.mark.parametrize("D,Hq", [(128, 4), (128, 48), (128, 128), (64, 4), (64, 48), (48, 4)])
@pytest.mark.parametrize("length", [1000, 20000])
@pytest.mark.parametrize("column", [0, 2, 5, -1])
def test_attention_nan_key_scale_of_a_whole_tile(D, Hq, length, column):
    """A page of keys whose scale is NaN, all that a warpgroup has of its piece: NaN for its key head alone."""
    c = cache_case(1, 1, Hq, 2, D, 128, [length], seed=length + column)
    ks, table = c["np"][1], c["np"][4]
    ks[table[0, column], 0] = 255
    c["cache"][1] = torch.from_numpy(ks).cuda()
    out, lse = check_attn(c)
    assert out[0, 0, :Hq // 2].isnan().all() and lse[0, 0, :Hq // 2].isnan().all()
    assert not out[0, 0, Hq // 2:].isnan().any()


@gpu
@pytest.mark.parametrize("D,Hq", [(128, 4), (64, 16), (48, 4)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5])
def test_attention_window_of_the_largest_sizes(D, Hq, window):
    """A window that no sequence fills, on sequences shorter than their query tokens: as without one."""
    c = cache_case(4, 12, Hq, 2, D, 32, [1, 3, 9, 400], seed=D)
    out, lse = check_attn(c)
    again, lse2 = wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], None, window, None, True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def outside_spread(got, ref, spread):
    """Values further from `ref` than half a bf16 ulp and the random errors of weights and scores allow."""
    return np.abs(got - ref) > 2.0 ** -8 * np.abs(ref) + spread + 1e-30


@pytest.mark.parametrize("B,Sq,Hq,Hkv,D,page,lens,window", LONG)
def test_the_spread_tells_what_is_missing(B, Sq, Hq, Hkv, D, page, lens, window):
    """Zeros, or a page whose values are lost, are outside the bound in every long case."""
    c = cache_case(B, Sq, Hq, Hkv, D, page, lens, seed=Hq, device="cpu", spread=0.3)
    q, np_c = np64(c["q"])[:1, :1], list(c["np"])
    np_c[4], np_c[5] = np_c[4][:1], np_c[5][:1] - Sq + 1  # the first query token sees what a shorter sequence's last one does
    ref, spread = R.attn_spread(q, *np_c, D ** -0.5, window)
    assert outside_spread(np.zeros_like(ref), ref, spread).mean() > 0.9
    first = (np_c[5][0] - window if window else 0) // page + 1
    for col in np.linspace(first, (np_c[5][0] - 1) // page, 8).astype(int):
        lost = np_c[2].copy()
        lost[np_c[4][0, col]] = 0
        less, _ = R.attn_spread(q, *np_c[:2], lost, *np_c[3:], D ** -0.5, window)
        assert outside_spread(less, ref, spread).mean() > 0.1, col


@gpu
@pytest.mark.parametrize("B,Sq,Hq,Hkv,D,page,lens,window", SHAPES + LONG)
def test_attention_within_the_spread(B, Sq, Hq, Hkv, D, page, lens, window):
    c = cache_case(B, Sq, Hq, Hkv, D, page, lens, seed=Sq * 10 + D, spread=0.3)
    out = wd().attn_decode_fp8(c["q"], *c["cache"], c["table"], c["lens"], window=window)
    ref, spread = R.attn_spread(np64(c["q"]), *c["np"], D ** -0.5, window)
    far = outside_spread(np64(out), ref, spread)
    assert not far.any(), (int(far.sum()), far.size)


def strong_key_case(columns, D, n, score, outlier):
    """One unit for every SM over the same pages: key 0 weighs e^score times any other, whose values have a common mean."""
    g = np.random.default_rng(n + D + int(10 * score))
    page, units = 128, torch.cuda.get_device_properties(0).multi_processor_count
    P = -(-n // page)
    k, v = 0.2 * g.standard_normal((1, n, 1, D)), 1 + 0.3 * g.standard_normal((1, n, 1, D))
    k[..., 0], k[0, 0, 0, 0] = 0.3 * g.standard_normal((1, n, 1)), score
    v[0, 0] = 0.0
    v[0, 0, 0, 0] = outlier
    kc, vc = (np.zeros((P, 1, page, D), np.uint8) for _ in range(2))
    ks, vs = (np.zeros((P, 1), np.uint8) for _ in range(2))
    one = np.arange(P, dtype=np.int32)[None]
    R.kv_write(k, kc, ks, one, [0], [n])
    R.kv_write(v, vc, vs, one, [0], [n])
    q = np.zeros((1, 1, columns, D))
    q[..., 0] = 1.0
    ref, spread = R.attn_spread(q[:, :, :1], kc, ks, vc, vs, one, [n], 1.0, 0)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    out = wd().attn_decode_fp8(t(q).bfloat16().expand(units, -1, -1, -1), t(kc), t(ks), t(vc), t(vs),
                               t(one).repeat(units, 1), torch.full((units,), n, dtype=torch.int32, device="cuda"), 1.0)
    assert torch.equal(out, out[:1, :, :1].expand_as(out))
    return np64(out[:1, :, :1]), ref, spread


@gpu
@pytest.mark.parametrize("columns,D", [(1, 128), (24, 128), (64, 128), (1, 64), (64, 64), (2, 48)])
@pytest.mark.parametrize("n,score", [(8192, 11.0), (8192, 12.5), (20000, 13.0), (65536, 14.0)])
def test_attention_strong_key_over_a_long_tail(columns, D, n, score):
    """Weights too small for the two terms' quantum, one by one, have their share of the output all together."""
    got, ref, spread = strong_key_case(columns, D, n, score, 0.0)
    assert np.median(spread / ref) < 0.3  # the bound tells a lost tail from one that is there
    assert not outside_spread(got, ref, spread).any(), (got.mean(), ref.mean(), spread.mean())


@gpu
@pytest.mark.parametrize("columns,D", [(1, 128), (64, 128), (1, 64), (2, 48)])
def test_attention_one_page_of_large_values(columns, D):
    """A value that raises its page's scale by 2^12 takes the other pages' weights to the quantum, not their sum."""
    got, ref, spread = strong_key_case(columns, D, 8192, 0.5, 3000.0)
    assert np.median(spread / ref) < 0.1
    assert not outside_spread(got, ref, spread).any(), (got.mean(), ref.mean(), spread.mean())


@gpu
@pytest.mark.parametrize("E,kw", [(64, {}), (256, dict(renormalize=False)), (256, dict(bias=True)),
                                  (256, dict(bias=True, renormalize=False)),
                                  (64, dict(n_group=8, topk_group=3)), (160, dict(n_group=8, topk_group=3, group_top=2)),
                                  (33, {})])
def test_router_softmax_of_an_infinite_logit(E, kw):
    """+infinity leaves a softmax without scores: NaN weights, not even ones that hide it; valid experts all the same."""
    g = torch.Generator().manual_seed(E)
    lg = torch.randn(4, E, generator=g)
    lg[1, E // 2] = lg[3, 5] = lg[3, 9] = float("inf")
    kw = {**kw, "bias": torch.randn(E, generator=g) * 0.1 if kw.get("bias") else None}
    ids, w, _ = R.router_scored(np64(lg), 6, **{**kw, "bias": None if kw["bias"] is None else np64(kw["bias"])})
    got, gw = (t.cpu().numpy() for t in wd().moe_router_scored_topk(
        lg.cuda(), 6, **{**kw, "bias": None if kw["bias"] is None else kw["bias"].cuda()}))
    assert np.isnan(w[[1, 3]]).all() and np.isnan(gw[[1, 3]]).all()
    assert np.array_equal(got, ids) and np.allclose(gw[[0, 2]], w[[0, 2]], rtol=4e-6, atol=0)
    sig, sw = wd().moe_router_scored_topk(lg.cuda(), 6, "sigmoid")  # a score of 1
    assert sig[1, 0] == E // 2 and sig[3, :2].tolist() == [5, 9] and not sw.isnan().any()


@pytest.mark.parametrize("call", [write_call, read_call])
@pytest.mark.parametrize("page", [16, 128])
def test_cache_calls_of_too_many_tokens_are_refused(call, page):
    """The grid's limit is told, up to the largest count (no 32-bit overflow on the way)."""
    L, name = capi.layer_lib(), "S" if call is write_call else "R"
    for n in (65534 * page + 2, 2 ** 31 - 1):
        before = L.wd_layer_launch_count()
        assert call(page=page, **{name: n}) == capi.WD_ERR_UNSUPPORTED
        assert "65534 pages" in L.wd_layer_last_error_message().decode()
        assert L.wd_layer_launch_count() == before


@gpu
def test_kv_read_of_a_long_range_of_many_heads():
    """More tokens than the grid has spans of four: the same values as in two parts."""
    H, D, page, P, R_all = 256, 16, 64, 5, 300001
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = [torch.randint(0, 127, (P, H, page, D), generator=g, device="cuda", dtype=torch.uint8) if i % 2 == 0 else
             torch.randint(120, 130, (P, H), generator=g, device="cuda", dtype=torch.uint8) for i in range(4)]
    table = torch.randint(0, P, (1, R_all // page + 2), generator=g, device="cuda", dtype=torch.int32)
    at = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = wd().kv_cache_read_fp8(*cache, table, at(3), R_all, at(R_all - 1))
    assert not k[:, -1].any() and not v[:, -1].any()
    for r0, n in ((0, 150000), (150000, 150000)):
        k1, v1 = wd().kv_cache_read_fp8(*cache, table, at(3 + r0), n)
        assert torch.equal(k[:, r0:r0 + n], k1) and torch.equal(v[:, r0:r0 + n], v1)
    assert wd().status(True, 0) == 0


def test_workspace_goes_to_the_current_device():
    """Every rank has its own device current: none is meant unless it is named."""
    import inspect
    import re

    doc = inspect.getdoc(wd().attn_decode_fp8_workspace)
    assert re.search(r"device: [^,)]*= None", doc), doc


@gpu
def test_workspace_device():
    ws = wd().attn_decode_fp8_workspace(1, 1, 8, 1, 128)
    assert ws.device.index == torch.cuda.current_device() and not ws.any()
    assert wd().attn_decode_fp8_workspace(1, 1, 8, 1, 128, device=0).numel() == ws.numel()


@gpu
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,inter", [
    (1999, 16, 2, 64, 32, True), (1500, 7, 3, 128, 128, False), (1500, 9, 4, 128, 64, False), (4097, 6, 1, 128, 64, True),
    (8195, 1, 1, 128, 128, False), (1201, 5, 3, 256, 256, False)])
def test_qk_norm_rope_heads_a_group(T, Hq, Hkv, D, rot, inter):
    """Token counts that take one, two and four heads a lane group, with head counts that fill the groups unevenly."""
    g = torch.Generator(device="cuda").manual_seed(T + D)
    buf = (torch.randn(T, (Hq + Hkv) * D, generator=g, device="cuda") * 3).bfloat16()
    q, k = buf[:, :Hq * D].unflatten(1, (Hq, D)), buf[:, Hq * D:].unflatten(1, (Hkv, D))
    qw, kw = (1 + 0.2 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    pos = torch.randint(0, 97, (T,), generator=g, device="cuda", dtype=torch.int32)
    ang = torch.randn(97, rot // 2, generator=g, device="cuda")
    cs = torch.cat([ang.cos(), ang.sin()], 1).contiguous()
    qo, ko = wd().qk_norm_rope(q, k, qw, kw, pos, cs, 1e-6, inter)
    check_rows_close(qo, R.norm_rope(np64(q), np64(qw), pos.cpu(), cs.cpu().numpy(), 1e-6, inter))
    check_rows_close(ko, R.norm_rope(np64(k), np64(kw), pos.cpu(), cs.cpu().numpy(), 1e-6, inter))
    assert wd().status(True, 0) == 0


@gpu
def test_qk_norm_rope_in_place_refuses_rows_on_one_place():
    one = torch.randn(6, 1, 64, device="cuda").bfloat16()
    q, k = one.expand(6, 4, 64), torch.randn(6, 2, 64, device="cuda").bfloat16()
    w, pos, cs = torch.ones(64, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda"), torch.ones(1, 64, device="cuda")
    before = one.clone()
    for a, b in ((q, k), (k, q), (k, k)):
        with pytest.raises(RuntimeError, match="memory location"):
            wd().qk_norm_rope(a, b, w, w, pos, cs, inplace=True)
    assert torch.equal(one, before)
    qo, _ = wd().qk_norm_rope(q, k, w, w, pos, cs)  # read only: as many equal heads
    assert torch.equal(qo, qo[:, :1].expand_as(qo))


@gpu
@pytest.mark.parametrize("D", [128, 64, 48, 256])
def test_attention_infinite_query_against_keys_of_the_other_sign(D):
    """All scores -infinity are 0 / 0, not a row without keys."""
    c = cache_case(1, 1, 4, 2, D, 16, [40], seed=D)
    kc, table = c["np"][0], c["np"][4]
    kc[table[0]] |= 0x80  # every key below 0
    c["cache"][0] = torch.from_numpy(kc).cuda()
    c["q"][0, 0, 1, 2] = float("inf")
    for window in (0, 1):
        out, lse = check_attn(c, window)
        assert out[0, 0, 1].isnan().all() and lse[0, 0].isnan().tolist() == [False, True, False, False]
