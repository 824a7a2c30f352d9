"""The operators that complete a decoder layer's step where they can go wrong: values, sizes
and calls beside those of test_block_ops.py, against the same 64-bit restatements.

Tolerances: half a step of the output's type plus the restatement's bound.
"""
import numpy as np
import pytest
import torch

from oracle import layer_ref as R
from test_block_ops import own_lens, prefix_case
from test_layer_ops import np64, wd

gpu = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
BF16_MAX = float(torch.finfo(BF16).max)


# ---------------------------------------------------------------------------
# attention behind a shared prefix
# ---------------------------------------------------------------------------
def prefix_spread(c, window=0, weight=2.0 ** -9, quantum=2.0 ** -47):
    """The operator on the case against the restatement with errors that add up as independent ones do.

    A weight is rounded to bf16, within 2^-9 of itself; one whose page has a scale far below the
    others' may count with up to 2^-47 of the row's largest product.
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
