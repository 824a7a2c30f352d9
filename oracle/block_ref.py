"""The operators that complete a decoder layer's step, restated in numpy with 64-bit
floats from their definitions in ``include/warp_decode_block.h``, each with a bound of
what fp32 arithmetic may add before the output is rounded.

Attention behind a shared prefix is attention: ``layer_ref.attn`` on the whole tables.
"""
from __future__ import annotations

import numpy as np

# Operations on a value in fp32 and the sum of a row's squares (up to 32 in a thread,
# then a tree): 50 roundings of 2^-24 at most, halved by the root, and rsqrtf's two ulps.
NORM_REL = 4e-6


def block_norm(y, r, norm_weight, post_weight=None, gate=None, residual_scale=1.0, eps=1e-6):
    """(x, r', x_slack, r_slack) for y, r [T, H]; the slacks are without the outputs' own rounding."""
    y, r = np.asarray(y, np.float64), np.asarray(r, np.float64)

    def factor(v):
        return 1.0 / np.sqrt(np.square(v).mean(1, keepdims=True) + eps)

    z = y if post_weight is None else y * factor(y) * post_weight
    z = z if gate is None else z * gate
    out = residual_scale * r + z
    r_slack = NORM_REL * (np.abs(residual_scale * r) + np.abs(z))
    f = factor(out)
    x = out * f * norm_weight
    # f moves by the relative error of the row's squares: at most that of its largest parts together
    moved = (r_slack * np.abs(out)).sum(1, keepdims=True) / np.maximum(np.square(out).sum(1, keepdims=True), 1e-300)
    x_slack = (NORM_REL + moved) * np.abs(x) + r_slack * f * np.abs(norm_weight)
    return x, out, x_slack, r_slack


def linear_w4(x, codes, scale, zero=None):
    """(out, slack) for x [T, K], codes [N, K], scale [N, K / g].

    Products are exact in fp32.  A group is the sum of at most eight matrix
    instructions, each of which may drop 2^-22 of its operands' magnitudes: 2^-19.
    Groups are added one after the other, each a rounding of 2^-24 of what is
    there, up to all K / g of them where a block has the whole row; then up to
    sixteen sums of warps or blocks: (K / g + 16) 2^-24 of the sum of magnitudes.
    """
    x = np.asarray(x, np.float64)
    N, K = codes.shape
    g = K // scale.shape[1]
    z = 8.0 if zero is None else np.asarray(zero, np.float64).repeat(g, 1)
    w = (np.asarray(codes, np.float64) - z) * np.asarray(scale, np.float64).repeat(g, 1)
    return x @ w.T, (2.0 ** -19 + (K // g + 16) * 2.0 ** -24) * (np.abs(x) @ np.abs(w).T)
