"""The operators around the MoE FFN, restated in numpy with 64-bit floats.

Expert choice, per-head norm with the position rotation, the FP8 paged cache
and attention over it, each written from its definition in
``include/warp_decode_layer.h``.  The quantiser is exact: codes and scale
bytes are those the kernels have to produce, bit for bit.
"""
from __future__ import annotations

import math

import numpy as np

E4M3_MAX = 448.0


# ---------------------------------------------------------------------------
# expert choice
# ---------------------------------------------------------------------------
def _first_largest(values, n, allowed=None):
    """Indices of the n largest, ties to the lowest index."""
    order = sorted((i for i in range(len(values)) if allowed is None or allowed[i]),
                   key=lambda i: (-values[i], i))
    return order[:n]


def router_scored(logits, topk, scoring="softmax", bias=None, n_group=1, topk_group=1, group_top=1,
                  renormalize=True, scale=1.0):
    """(ids [T, topk], weights [T, topk], choice [T, E]) in 64 bits."""
    x = np.where(np.isnan(logits), -np.inf, np.asarray(logits, np.float64))
    T, E = x.shape
    if scoring == "softmax":
        top = np.where(np.isfinite(x.max(1)), x.max(1), 0.0)[:, None]
        e = np.exp(np.where(np.isposinf(x), 0.0, x) - top)
        den = e.sum(1, keepdims=True)
        score = np.divide(e, den, out=np.zeros_like(e), where=den > 0)
        score[np.isposinf(x).any(1)] = np.nan  # infinity over infinity
    else:
        with np.errstate(over="ignore"):
            score = 1.0 / (1.0 + np.exp(-x))
    choice = score + np.asarray(bias, np.float64) if bias is not None else score if group_top == 2 else x
    choice = np.where(np.isnan(choice), -np.inf, choice)
    ids = np.zeros((T, topk), np.int32)
    w = np.zeros((T, topk))
    size = E // n_group
    for t in range(T):
        allowed = None
        if n_group > 1:
            rank = [sum(sorted(choice[t, g * size:(g + 1) * size])[::-1][:group_top]) for g in range(n_group)]
            kept = set(_first_largest(rank, topk_group))
            allowed = [e // size in kept for e in range(E)]
        ids[t] = _first_largest(choice[t], topk, allowed)
        w[t] = score[t, ids[t]]
        if renormalize:
            if scoring == "softmax" and not np.isnan(w[t]).any():  # around the chosen logits' own maximum: no underflow
                l = x[t, ids[t]]
                m = l.max() if np.isfinite(l.max()) else 0.0
                w[t] = np.exp(l - m)
            s = w[t].sum()
            w[t] = w[t] / s if s != 0 else 1.0 / topk
    return ids, w * scale, choice


# ---------------------------------------------------------------------------
# norm and rotation
# ---------------------------------------------------------------------------
def norm_rope(x, weight, positions, cos_sin, eps, interleaved):
    """x [T, H, D] -> [T, H, D] in 64 bits; rows at positions outside the table are zeros."""
    x = np.asarray(x, np.float64)
    rot = cos_sin.shape[1]
    half = rot // 2
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    out = y.copy()
    for t, p in enumerate(np.asarray(positions)):
        if p < 0 or p >= cos_sin.shape[0]:
            out[t] = 0.0
            continue
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            c, s = float(cos_sin[p, i]), float(cos_sin[p, half + i])
            out[t, :, a] = y[t, :, a] * c - y[t, :, b] * s
            out[t, :, b] = y[t, :, b] * c + y[t, :, a] * s
    return out


# ---------------------------------------------------------------------------
# FP8 paged cache
# ---------------------------------------------------------------------------
def e4m3_table():
    """The 256 values of E4M3 (NaN at 0x7f and 0xff)."""
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        a = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = math.nan if c & 127 == 127 else -a if c & 128 else a
    return v


TABLE = e4m3_table()


def e4m3_encode(x):
    """Codes of the nearest E4M3 values (ties to even codes), saturating; NaN -> 0x7f."""
    x = np.asarray(x, np.float64)
    mags = TABLE[:127]  # ascending magnitudes 0 .. 448
    a = np.minimum(np.abs(x), E4M3_MAX)
    hi = np.clip(np.searchsorted(mags, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - mags[lo], mags[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(x), 0x7F, code)
    return (code | np.where(np.signbit(x) & ~np.isnan(x), 0x80, 0)).astype(np.uint8)


def scale_exponent(amax):
    """Least integer e with amax <= 448 * 2^e, within the scale byte's range."""
    if amax == 0:
        return -126
    m, x = math.frexp(amax)  # amax = m * 2^x, m in [0.5, 1)
    e = x - 9 if m <= 0.875 else x - 8
    return min(max(e, -126), 127)


def kv_write(x, cache, scale, table, start, lens):
    """x [B, S, H, D] into cache [P, H, page, D] codes and scale [P, H] bytes, in place."""
    P, H, page, D = cache.shape
    for b in range(x.shape[0]):
        n = min(max(int(lens[b]), 0), x.shape[1])
        end = int(start[b]) + n
        if start[b] < 0:
            continue
        for col in range(int(start[b]) // page, (end - 1) // page + 1 if n else 0):
            pid = int(table[b, col]) if col < table.shape[1] else -1
            if not 0 <= pid < P:
                continue
            lo, hi = max(int(start[b]), col * page), min(end, (col + 1) * page)
            old = lo - col * page
            for h in range(H):
                new = np.asarray(x[b, lo - start[b]:hi - start[b], h], np.float64)
                fin = np.abs(new[np.isfinite(new)])
                e = scale_exponent(float(fin.max(initial=0.0)))
                if old:
                    was = int(scale[pid, h]) - 127
                    if e > was:
                        cache[pid, h, :old] = e4m3_encode_signed_nan(TABLE[cache[pid, h, :old]] * 2.0 ** (was - e),
                                                                     cache[pid, h, :old])
                    e = max(e, was)
                cache[pid, h, old:hi - col * page] = e4m3_encode(new * 2.0 ** -e)
                scale[pid, h] = e + 127


def e4m3_encode_signed_nan(x, codes):
    """As e4m3_encode for values that came from `codes`: a NaN stays a NaN (either sign)."""
    return np.where(np.isnan(x), 0x7F, e4m3_encode(x)).astype(np.uint8)


def scale_values(scale):
    """What UE8M0 scale bytes stand for: 2^(byte - 127), 255 NaN."""
    return np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127))


def kv_values(cache, scale):
    return TABLE[cache] * scale_values(scale)[..., None, None]


def kv_read(cache, scale, table, start, length, lens):
    P, H, page, D = cache.shape
    out = np.zeros((table.shape[0], length, H, D))
    for b in range(table.shape[0]):
        for r in range(min(length, int(lens[b]))):
            t = int(start[b]) + r
            pid = int(table[b, t // page]) if t // page < table.shape[1] else -1
            if 0 <= pid < P:
                out[b, r] = TABLE[cache[pid, :, t % page]] * scale_values(scale[pid])[:, None]
    return out


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def attn(q, kc, ks, vc, vs, table, seq_lens, softmax_scale, window):
    """(out, lse, slack, lse_slack) in 64 bits for q [B, Sq, Hq, D].

    slack [B, Sq, Hq, D] bounds what an implementation that holds scores and
    sums in fp32 and each weight p as a sum of two E4M3 values may add before
    its rounding to bf16: two E4M3 terms are within 2^-9 of p, or within 2^-14
    of the largest p where p is small; a score is within 2^-16 of the sum of
    its products' magnitudes, which moves p by that factor (twice: numerator
    and denominator).
    """
    P, Hkv, page, D = kc.shape
    B, Sq, Hq, _ = q.shape
    G = Hq // Hkv
    out, slack = np.zeros(q.shape), np.zeros(q.shape)
    lse, lse_slack = np.full(q.shape[:3], -np.inf), np.zeros(q.shape[:3])
    for b in range(B):
        n = int(seq_lens[b])
        toks = np.arange(max(n, 0))
        pids = np.array([table[b, t // page] if t // page < table.shape[1] else -1 for t in toks], np.int64)
        good = (pids >= 0) & (pids < P)
        toks, pids = toks[good], pids[good]
        for hk in range(Hkv):
            k = TABLE[kc[pids, hk, toks % page]] * scale_values(ks[pids, hk])[:, None]
            v = TABLE[vc[pids, hk, toks % page]] * scale_values(vs[pids, hk])[:, None]
            for i in range(Sq):
                pos = n - Sq + i
                seen = (toks <= pos) & ((toks > pos - window) if window else True)
                if pos < 0 or not seen.any():
                    continue
                kk, vv = k[seen], v[seen]
                for g in range(G):
                    h = hk * G + g
                    qq = np.asarray(q[b, i, h], np.float64)
                    s = kk @ qq * softmax_scale
                    m = s.max()
                    if m == -np.inf:  # an infinite q against keys of the other sign alone: 0 / 0
                        out[b, i, h], lse[b, i, h] = np.nan, np.nan
                        continue
                    p = np.exp(s - m)
                    out[b, i, h] = p @ vv / p.sum()
                    lse[b, i, h] = m + math.log(p.sum()) if not math.isnan(m) else math.nan
                    ds = 2.0 ** -16 * (np.abs(kk) @ np.abs(qq)).max() * abs(softmax_scale)
                    lse_slack[b, i, h] = ds
                    slack[b, i, h] = ((2.0 ** -9 + 2 * ds) * (p @ np.abs(vv)) + 2.0 ** -14 * np.abs(vv).sum(0)) / p.sum()
    return out, lse, slack, lse_slack


def attn_spread(q, kc, ks, vc, vs, table, seq_lens, softmax_scale, window, sigmas=6.0):
    """(out, spread) in 64 bits: `spread` bounds the distance that rounding may make, key by key at random.

    `attn`'s slack adds the largest error of every key up, which over a long
    sequence passes the result itself.  Here the errors of n keys add up as
    independent ones do, by their squares, and are not larger than, for key j
    of weight w_j (of sum 1) and value v_j = code_j * 2^scale:

    * 2^-9 w_j v_j: a weight as two E4M3 terms of four significant bits;
    * 2^-17 lead code_j, lead the row's largest w * 2^scale: the two terms'
      quantum is 2^-16 of the largest, of which a rounding without bias takes
      half on average at most;
    * 2^-16 (1 + sum |q k| softmax_scale) w_j (v_j - out): the score in fp32, in
      numerator and denominator.

    Six of their standard deviations, each taken as large as its bound, leave
    less than one of 10^8 values outside.
    """
    P, Hkv, page, D = kc.shape
    B, Sq, Hq, _ = q.shape
    G = Hq // Hkv
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        toks = np.arange(max(int(seq_lens[b]), 0))
        cols = toks // page
        pids = np.where(cols < table.shape[1], table[b, np.minimum(cols, table.shape[1] - 1)], -1)
        good = (pids >= 0) & (pids < P)
        toks, pids = toks[good], pids[good]
        for hk in range(Hkv):
            k = TABLE[kc[pids, hk, toks % page]] * scale_values(ks[pids, hk])[:, None]
            code, unit = TABLE[vc[pids, hk, toks % page]], scale_values(vs[pids, hk])
            v = code * unit[:, None]
            for i in range(Sq):
                pos = int(seq_lens[b]) - Sq + i
                seen = (toks <= pos) & ((toks > pos - window) if window else True)
                if pos < 0 or not seen.any():
                    continue
                for h in range(hk * G, (hk + 1) * G):
                    qq = np.asarray(q[b, i, h], np.float64)
                    s = k[seen] @ qq * softmax_scale
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[b, i, h] = w @ v[seen]
                    ds = 2.0 ** -16 * (1 + np.abs(k[seen]) @ np.abs(qq) * abs(softmax_scale))
                    var = np.square(2.0 ** -9 * w) @ np.square(v[seen])
                    var += (2.0 ** -17 * (w * unit[seen]).max()) ** 2 * np.square(code[seen]).sum(0)
                    var += np.square(ds * w) @ np.square(v[seen] - out[b, i, h])
                    spread[b, i, h] = sigmas * np.sqrt(var)
    return out, spread
