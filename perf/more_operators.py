"""Cases of the operators that complete a decoder layer's step around the MoE FFN:

* ``norm``   -- a block's output, normed or not, gated onto the scaled residual
                stream, and the norm before the next block, in one pass;
* ``linear`` -- a projection of a few tokens with 4-bit weights, one scale (and
                zero point) per group of them;
* ``prefix`` -- attention over the FP8 paged cache of a batch whose sequences
                begin with the same tokens, kept in the same pages.

``run`` computes them either through the framework (``own``) or in a plain
form made of elementary torch operations in 32 bits.  ``exact`` restates each
operator in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-6
WORKSPACE_BYTES = 256 << 20  # what one stream's program keeps for attention


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One token between two blocks of a small model: the smallest call, all latency.
        dict(name="norm decode 1x2048", op="norm", T=1, H=2048, post=False, gate="none", scale=1.0, residual="bf16"),
        # A decode batch of a wide model that norms a block's output too, and scales it per channel.
        dict(name="norm decode 64x7168 sandwich", op="norm", T=64, H=7168, post=True, gate="channel", scale=1.0,
             residual="bf16"),
        # A prompt of odd length, gated token by token, on an fp32 residual stream.
        dict(name="norm prompt 1999x4096 gated", op="norm", T=1999, H=4096, post=False, gate="token", scale=0.5,
             residual="f32"),
        # A long prompt with both norms.
        dict(name="norm prompt 8192x4096 sandwich", op="norm", T=8192, H=4096, post=True, gate="channel", scale=1.0,
             residual="bf16"),
        # One token, the keys and values of one tensor-parallel shard: a projection that is all latency.
        dict(name="linear 1x4096 to 512", op="linear", T=1, N=512, K=4096, group=128, zero=False, scales="bf16"),
        # One token, queries, keys and values of a whole layer.
        dict(name="linear 1x4096 to 9216", op="linear", T=1, N=9216, K=4096, group=128, zero=False, scales="bf16"),
        # A small decode batch through the output projection, with zero points.
        dict(name="linear 16x8192 to 4096", op="linear", T=16, N=4096, K=8192, group=64, zero=True, scales="f16"),
        # A full decode batch, queries, keys and values.
        dict(name="linear 64x4096 to 9216", op="linear", T=64, N=9216, K=4096, group=128, zero=False, scales="bf16"),
        # Four short answers to one prompt, one tensor-parallel shard: the smallest attention call.
        dict(name="prefix 4x1 on 1000", op="prefix", B=4, Sq=1, Hq=8, Hkv=1, D=128, page=64, P=1000, own=100),
        # A full decode batch behind one long system prompt.
        dict(name="prefix 64x1 on 8192", op="prefix", B=64, Sq=1, Hq=32, Hkv=4, D=128, page=64, P=8192, own=512),
        # Four proposed tokens of each sequence verified at once, on small pages.
        dict(name="prefix 16x4 on 12001", op="prefix", B=16, Sq=4, Hq=32, Hkv=4, D=128, page=16, P=12001, own=1000),
        # A large batch of samples of one long document.
        dict(name="prefix 128x1 on 16384", op="prefix", B=128, Sq=1, Hq=32, Hkv=4, D=128, page=128, P=16384, own=256),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "prefix", "prefix"])
    if op == "norm":
        H = _log_int(rng, 64, 8192)
        if rng.random() < 0.85:
            H = (H + 63) // 64 * 64
        return dict(op=op, T=_log_int(rng, 1, min(16384, 8192 * 4096 // H)), H=H, post=rng.random() < 0.5,
                    gate=rng.choice(["none", "channel", "token", "full"]), scale=rng.choice([1.0, 1.0, 0.5]),
                    residual=rng.choice(["bf16", "bf16", "f32"]))
    if op == "linear":
        group = rng.choice([32, 64, 128, 128])
        K = group * _log_int(rng, 2, 16384 // group)
        N = _log_int(rng, 64, min(16384, 9216 * 4096 // K))
        if rng.random() < 0.8:
            N = (N + 15) // 16 * 16
        return dict(op=op, T=_log_int(rng, 1, 64), N=min(N, 9216 * 4096 // K), K=K, group=group,
                    zero=rng.random() < 0.4, scales=rng.choice(["bf16", "f16", "f32"]))
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 4, 5, 7, 8, 16])
    Sq = rng.choice([1, 1, 1, 1, 2, 3, 4])
    B = _log_int(rng, 1, 256)
    own_len = _log_int(rng, Sq, max(Sq, min(2048, 128 * 256 * 4 * 128 // (B * Hkv * D))))
    most = 128 * 32 * 128 * 16384 // (B * Sq * Hkv * G * D) - own_len
    return dict(op=op, B=B, Sq=Sq, Hq=Hkv * G, Hkv=Hkv, D=D, page=rng.choice([16, 32, 64, 128]),
                P=_log_int(rng, 1, max(1, min(65536, most))), own=own_len)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand_int(g, lo, hi, *shape):
    """int32 values of [lo, hi]."""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _pack(codes):
    """4-bit codes [N, K] as the framework keeps them: rows of whole blocks of 128 codes
    (64 bytes), in which 32-bit word 4 t + s holds the codes of k = 32 s + 8 t + 0..7, the
    even ones in its low half, the odd ones in its high half."""
    N, K = codes.shape
    c = torch.zeros(N, (K + 127) // 128 * 128, dtype=torch.int32, device=codes.device)
    c[:, :K] = codes
    c = c.view(N, -1, 4, 4, 4, 2).permute(0, 1, 3, 2, 5, 4)  # block, t, s, odd, pair
    b = c.reshape(N, -1, 2)
    return (b[..., 0] | b[..., 1] << 4).to(torch.uint8)


def _filled_cache(g, P, H, page, D):
    """Codes and scale bytes of a cache in use: every page normal values with a few strong channels."""
    strong = 1.0 + 3.0 * (torch.rand(H, 1, D, generator=g, device="cuda") < 0.03)
    codes = torch.empty(P, H, page, D, dtype=torch.uint8, device="cuda")
    step = max(1, (64 << 20) // (H * page * D))
    scale = torch.empty(P, H, dtype=torch.uint8, device="cuda")
    for p in range(0, P, step):
        x = _randn(g, min(step, P - p), H, page, D) * strong
        m, e = torch.frexp(x.abs().amax(dim=(2, 3)))
        e = e - 9 + (m > 0.875)
        scale[p:p + step] = (e + 127).to(torch.uint8)
        codes[p:p + step] = torch.ldexp(x, -e[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, scale


def prepare(case, seed):
    g, c, op = _gen(seed), case, case["op"]
    s = dict(case)
    if op == "norm":
        T, H = c["T"], c["H"]
        s["y"] = (_randn(g, T, H) * 0.7).to(torch.bfloat16)
        s["residual_in"] = (_randn(g, T, H) * 2.0).to(_TYPES[c["residual"]])
        s["norm_weight"] = (1.0 + 0.1 * _randn(g, H)).to(torch.bfloat16)
        s["post_weight"] = (1.0 + 0.1 * _randn(g, H)).to(torch.bfloat16) if c["post"] else None
        shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[c["gate"]]
        s["gate_in"] = (0.5 + 0.3 * _randn(g, *shape)).to(torch.bfloat16) if shape else None
    elif op == "linear":
        T, N, K, group = c["T"], c["N"], c["K"], c["group"]
        s["x"] = _randn(g, T, K).to(torch.bfloat16)
        codes = torch.clamp(torch.round(_randn(g, N, K) * 2.7 + 8.0), 0, 15).to(torch.int32)
        s["codes"] = codes.to(torch.uint8)  # what the plain form reads
        s["w"] = _pack(codes)
        s["w_scale"] = (torch.exp(0.3 * _randn(g, N, K // group)) * (0.37 / math.sqrt(K))).to(_TYPES[c["scales"]])
        s["w_zero"] = _rand_int(g, 5, 11, N, K // group).to(torch.uint8) if c["zero"] else None
    else:
        B, Sq, Hq, Hkv, D, page, P = c["B"], c["Sq"], c["Hq"], c["Hkv"], c["D"], c["page"], c["P"]
        own_lens = _rand_int(g, min(c["own"], max(Sq, c["own"] // 8)), c["own"], B)
        own_lens[0] = c["own"]
        s["seq_lens"] = P + own_lens
        shared = P // page  # whole pages that every sequence's table begins with
        each = (P + c["own"] + page - 1) // page - shared
        pool = torch.randperm(shared + B * each, generator=g, device="cuda").to(torch.int32) + 1
        s["block_table"] = torch.cat([pool[:shared].expand(B, shared), pool[shared:].view(B, each)], 1).contiguous()
        s["prefix_len"] = torch.full((1,), P, dtype=torch.int32, device="cuda")
        pages = shared + B * each + 1  # page 0 belongs to no sequence
        s["k_cache"], s["k_scale"] = _filled_cache(g, pages, Hkv, page, D)
        s["v_cache"], s["v_scale"] = _filled_cache(g, pages, Hkv, page, D)
        qkv = _randn(g, B, Sq, (Hq + 2 * Hkv) * D).to(torch.bfloat16)
        s["q"] = qkv[..., :Hq * D].unflatten(2, (Hq, D))
        s["workspace"] = torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    op = s["op"]
    if own:
        from warp_decode_b200 import warp_decode as wd

        if op == "norm":
            return wd.block_norm(s["y"], s["residual_in"], s["norm_weight"], s["post_weight"], s["gate_in"],
                                 s["scale"], EPS)
        if op == "linear":
            return wd.linear_w4(s["x"], s["w"], s["w_scale"], s["w_zero"])
        return wd.attn_decode_fp8_prefix(s["q"], s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"],
                                         s["block_table"], s["seq_lens"], s["prefix_len"], workspace=s["workspace"])
    if op == "norm":
        return _plain_norm(s)
    if op == "linear":
        return _plain_linear(s)
    return _plain_prefix(s)


def _rms(x, weight):
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.float()


def _plain_norm(s):
    z = s["y"].float()
    if s["post_weight"] is not None:
        z = _rms(z, s["post_weight"])
    if s["gate_in"] is not None:
        z = z * s["gate_in"].float()
    r = s["residual_in"].float() * s["scale"] + z
    return _rms(r, s["norm_weight"]).to(torch.bfloat16), r.to(s["residual_in"].dtype)


def _plain_linear(s):
    N, K, group = s["N"], s["K"], s["group"]
    w = s["codes"].view(N, K // group, group).float()
    w = w - (s["w_zero"].float()[..., None] if s["w_zero"] is not None else 8.0)
    w = (w * s["w_scale"].float()[..., None]).view(N, K)
    return torch.matmul(s["x"].float(), w.t()).to(torch.bfloat16)


def _values(codes, scale):
    """What codes [..., tokens, D] stand for, scale bytes [...]."""
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(), (scale.int() - 127)[..., None, None])


def _plain_prefix(s):
    B, Sq, Hq, Hkv, D, page = s["B"], s["Sq"], s["Hq"], s["Hkv"], s["D"], s["page"]
    G, shared = Hq // Hkv, s["P"] // page
    table = s["block_table"].long()
    first, rest = table[0, :shared], table[:, shared:]

    def head(cache, scale):  # [Hkv, shared * page, D]
        return _values(cache[first], scale[first]).permute(1, 0, 2, 3).reshape(Hkv, shared * page, D)

    def tail(cache, scale):  # [B, Hkv, own pages * page, D]
        return _values(cache[rest], scale[rest]).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)

    q = s["q"].float().view(B, Sq, Hkv, G, D).permute(2, 0, 1, 3, 4) * (1.0 / math.sqrt(D))  # [Hkv, B, Sq, G, D]
    x1 = torch.matmul(q.reshape(Hkv, B * Sq * G, D), head(s["k_cache"], s["k_scale"]).transpose(1, 2))
    x1 = x1.view(Hkv, B, Sq * G, shared * page)
    x2 = torch.matmul(q.reshape(Hkv, B, Sq * G, D), tail(s["k_cache"], s["k_scale"]).permute(1, 0, 3, 2))
    at = shared * page + torch.arange(x2.shape[-1], device=x2.device)
    pos = s["seq_lens"][:, None] - Sq + torch.arange(Sq, device=x2.device)  # [B, Sq]
    seen = (at <= pos[..., None])[:, :, None, :].expand(B, Sq, G, at.numel()).reshape(B, Sq * G, at.numel())
    x2 = torch.where(seen, x2, float("-inf"))
    seen1 = torch.arange(shared * page, device=x1.device) <= pos[..., None]
    seen1 = seen1[:, :, None, :].expand(B, Sq, G, shared * page).reshape(B, Sq * G, shared * page)
    x1 = torch.where(seen1, x1, float("-inf"))
    x = torch.cat([x1, x2], dim=-1)
    del x1, x2
    top = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - torch.where(top > float("-inf"), top, 0.0))
    den = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p[..., :shared * page].reshape(Hkv, B * Sq * G, shared * page), head(s["v_cache"], s["v_scale"]))
    o = o.view(Hkv, B, Sq * G, D)
    o = o + torch.matmul(p[..., shared * page:], tail(s["v_cache"], s["v_scale"]).permute(1, 0, 2, 3))
    o = torch.where(den > 0, o / den, 0.0)
    return o.view(Hkv, B, Sq, G, D).permute(1, 2, 0, 3, 4).reshape(B, Sq, Hq, D).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def work(case):
    c, op = case, case["op"]
    if op == "norm":
        n = c["T"] * c["H"]
        gate = {"none": 0, "channel": c["H"], "token": c["T"], "full": n}[c["gate"]]
        return {"bytes": n * (4 + 2 * _BYTES[c["residual"]]) + 2 * gate + c["H"] * (4 if c["post"] else 2),
                "flops": 8.0 * n}
    if op == "linear":
        T, N, K = c["T"], c["N"], c["K"]
        groups = N * K // c["group"]
        return {"bytes": N * K / 2 + groups * (_BYTES[c["scales"]] + (1 if c["zero"] else 0)) + 2 * T * (K + N),
                "flops": 2.0 * T * N * K}
    rows, mean = c["B"] * c["Sq"] * c["Hq"], 0.5625 * c["own"]  # own lengths are uneven
    return {"bytes": 2.0 * c["Hkv"] * c["D"] * (c["P"] + c["B"] * mean) + 4.0 * rows * c["D"],
            "flops": 4.0 * rows * c["D"] * (c["P"] + mean)}


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "norm":
        return _exact_norm(s)
    if op == "linear":
        return _exact_linear(s)
    return _exact_prefix(s)


def _exact_norm(s):
    def norm(x, weight):
        return x / torch.sqrt(x.square().sum(dim=1, keepdim=True) / x.shape[1] + EPS) * weight.double()

    z = s["y"].double()
    if s["post_weight"] is not None:
        z = norm(z, s["post_weight"])
    gate = 1.0 if s["gate_in"] is None else s["gate_in"].double()
    r = torch.add(gate * z, s["residual_in"].double(), alpha=s["scale"])
    return norm(r, s["norm_weight"]), r


def _exact_linear(s):
    out = torch.zeros(s["T"], s["N"], dtype=torch.float64, device=s["x"].device)
    x, group = s["x"].double(), s["group"]
    for j in range(s["K"] // group):  # one group's share of every output at a time
        part = slice(j * group, (j + 1) * group)
        zero = 8.0 if s["w_zero"] is None else s["w_zero"][:, j, None].double()
        out += x[:, part] @ (s["codes"][:, part].double() - zero).t() * s["w_scale"][:, j].double()
    return out


def _exact_prefix(s):
    B, Sq, Hq, Hkv, D, page = (s[k] for k in ("B", "Sq", "Hq", "Hkv", "D", "page"))
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64, device=s["q"].device)

    def tokens(which, pids):  # [Hkv, tokens, D]
        v = s[which + "_cache"][pids].view(torch.float8_e4m3fn).double()
        return (v * torch.exp2(s[which + "_scale"][pids].double() - 127.0)[:, :, None, None]).transpose(0, 1).flatten(1, 2)

    shared = s["P"] // page
    lead = s["block_table"][0, :shared].long()
    k0, v0 = tokens("k", lead), tokens("v", lead)
    for b, n in enumerate(s["seq_lens"].tolist()):
        pids = s["block_table"][b, shared:(n + page - 1) // page].long()
        k, v = torch.cat([k0, tokens("k", pids)], 1)[:, :n], torch.cat([v0, tokens("v", pids)], 1)[:, :n]
        for i in range(Sq):
            end = n - Sq + i + 1
            if end > 0:
                x = torch.bmm(s["q"][b, i].double().view(Hkv, Hq // Hkv, D), k[:, :end].transpose(1, 2))
                out[b, i] = torch.bmm(torch.softmax(x / math.sqrt(D), dim=-1), v[:, :end]).reshape(Hq, D)
    return out
