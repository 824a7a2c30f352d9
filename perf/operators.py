"""Cases of the operators that surround the MoE FFN in one decoder layer's step:

* ``router``    -- expert choice from router logits: softmax or sigmoid scores, a
                   balance bias, expert groups, top-k, renormalised weights;
* ``qk_norm``   -- RMS norm of every query and key head with the position
                   rotation in the same pass;
* ``kv``        -- new keys and values quantised (E4M3, one power-of-two scale per
                   page and head) as they are written into a paged cache, and a
                   range of tokens read back as bf16;
* ``attn``      -- attention of a few query tokens per sequence over that cache.

``run`` computes them either through the framework (``own``) or in a plain
form made of elementary torch operations in 32 bits.  ``exact`` restates each
operator in 64 bits.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
EPS = 1e-6
ROPE_BASE = 1e6
WORKSPACE_BYTES = 16 << 20  # what one stream's program keeps for attn


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One token of a 128-expert layer: the smallest call, all latency.
        dict(name="router decode 1x128", op="router", T=1, E=128, K=8, scoring="softmax", bias=False, groups=1,
             pick=1, top=1, renorm=True, scale=1.0, dtype="bf16"),
        # A decode batch of a 256-expert layer: sigmoid scores, bias, 4 of 8 groups.
        dict(name="router decode 64x256 grouped", op="router", T=64, E=256, K=8, scoring="sigmoid", bias=True,
             groups=8, pick=4, top=2, renorm=True, scale=2.5, dtype="f32"),
        # The same router over a long prompt.
        dict(name="router prompt 16384x256 grouped", op="router", T=16384, E=256, K=8, scoring="sigmoid", bias=True,
             groups=8, pick=4, top=2, renorm=True, scale=2.5, dtype="f32"),
        # A decode batch: one token of 64 sequences, 64 query and 4 key heads.
        dict(name="qk_norm decode 64", op="qk_norm", T=64, Hq=64, Hkv=4, D=128, rot=128, interleaved=False),
        # A prompt of odd length with small heads, half of each rotated in adjacent pairs.
        dict(name="qk_norm prompt 1999 partial", op="qk_norm", T=1999, Hq=16, Hkv=2, D=64, rot=32, interleaved=True),
        # A long prompt.
        dict(name="qk_norm prompt 8192", op="qk_norm", T=8192, Hq=32, Hkv=4, D=128, rot=128, interleaved=False),
        # One new token of each of 64 sequences, the page it lands on read back.
        dict(name="kv append 64x1", op="kv", B=64, S=1, past=1500, Hkv=4, D=128, page=64, read=64),
        # Prompt chunks of eight sequences, of uneven lengths and on top of a partly filled page, read back whole.
        dict(name="kv prompt 8x2048", op="kv", B=8, S=2048, past=40, Hkv=4, D=128, page=64, read=2048),
        # One sequence of one tensor-parallel shard: the smallest attention call.
        dict(name="attn 1x1 len 1000", op="attn", B=1, Sq=1, Hq=8, Hkv=1, D=128, page=64, L=1000, window=0, ragged=False),
        # A full decode batch with sequences of very different lengths.
        dict(name="attn 64x1 len 8192 ragged", op="attn", B=64, Sq=1, Hq=32, Hkv=4, D=128, page=64, L=8192, window=0,
             ragged=True),
        # One long sequence: the work of one row split over the whole GPU.
        dict(name="attn 1x1 len 131072", op="attn", B=1, Sq=1, Hq=64, Hkv=4, D=128, page=128, L=131072, window=0,
             ragged=False),
        # Four proposed tokens of each sequence verified at once, on small pages, within a sliding window.
        dict(name="attn 16x4 len 12001 window", op="attn", B=16, Sq=4, Hq=32, Hkv=4, D=128, page=16, L=12001,
             window=8000, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["router", "qk_norm", "kv", "attn", "attn"])
    if op == "router":
        E = rng.choice([8, 40, 64, 96, 128, 160, 256, 384, 512])
        grouped = rng.random() < 0.5 and E % 8 == 0 and E >= 64
        sigmoid = grouped or rng.random() < 0.5
        K = rng.randint(1, 8)
        return dict(op=op, T=_log_int(rng, 1, 16384 * 256 // max(256, E)), E=E, K=K,
                    scoring="sigmoid" if sigmoid else "softmax", bias=grouped or (sigmoid and rng.random() < 0.5),
                    groups=8 if grouped else 1, pick=rng.randint(1, 8) if grouped else 1, top=2 if grouped else 1,
                    renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["bf16", "f32"]))
    if op == "qk_norm":
        D = rng.choice([64, 128, 128])
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.choice([1, 2, 4, 5, 8, 16])
        most = 8192 * 36 * 128 // ((Hq + Hkv) * D)
        return dict(op=op, T=_log_int(rng, 1, min(16384, most)), Hq=Hq, Hkv=Hkv, D=D,
                    rot=rng.choice([D, D, D // 2, D // 4]), interleaved=rng.random() < 0.3)
    if op == "kv":
        D = rng.choice([64, 128, 128])
        Hkv = rng.choice([1, 2, 4, 8])
        S = rng.choice([1, 1, 1, 2, 5, _log_int(rng, 2, 2048), _log_int(rng, 2, 2048)])
        B = _log_int(rng, 1, max(1, min(256, 8 * 2048 * 4 * 128 // (S * Hkv * D))))
        page = rng.choice([16, 32, 64, 128])
        return dict(op=op, B=B, S=S, past=_log_int(rng, 1, 3000) - 1, Hkv=Hkv, D=D, page=page,
                    read=max(S, rng.choice([1, page])))
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 4, 5, 7, 8, 16])
    Sq = rng.choice([1, 1, 1, 1, 2, 3, 4, 8])
    B = _log_int(rng, 1, 128)
    most = 36 * 8192 * 4 * 128 // (B * Hkv * D * Sq)  # about the listed batch's keys, which are ragged
    L = _log_int(rng, 1, max(1, min(65536, most)))
    return dict(op=op, B=B, Sq=Sq, Hq=Hkv * G, Hkv=Hkv, D=D, page=rng.choice([16, 32, 64, 128]), L=L,
                window=rng.choice([0, 0, 0, _log_int(rng, 1, 16384)]), ragged=rng.random() < 0.7)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand_int(g, lo, hi, *shape):
    """int32 values of [lo, hi]."""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _tables(g, B, pages_each):
    """Block tables over a shuffled pool; page 0 belongs to no sequence."""
    pool = torch.randperm(B * pages_each, generator=g, device="cuda").to(torch.int32) + 1
    return pool.view(B, pages_each).contiguous(), B * pages_each + 1


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


def _cos_sin(positions, rot):
    inv = ROPE_BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float().contiguous()


def prepare(case, seed):
    g, c, op = _gen(seed), case, case["op"]
    s = dict(case)
    if op == "router":
        logits = _randn(g, c["T"], c["E"]) * 1.5
        s["logits"] = logits.to(torch.bfloat16) if c["dtype"] == "bf16" else logits
        s["bias"] = (_randn(g, c["E"]) * 0.1) if c["bias"] else None
    elif op == "qk_norm":
        T, Hq, Hkv, D = c["T"], c["Hq"], c["Hkv"], c["D"]
        # the rows of a fused projection: queries, keys and values of a token side by side
        qkv = (_randn(g, T, (Hq + 2 * Hkv) * D) * 2.0).to(torch.bfloat16)
        s["q"] = qkv[:, :Hq * D].unflatten(1, (Hq, D))
        s["k"] = qkv[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D))
        s["q_weight"] = (1.0 + 0.1 * _randn(g, D)).to(torch.bfloat16)
        s["k_weight"] = (1.0 + 0.1 * _randn(g, D)).to(torch.bfloat16)
        s["positions"] = _rand_int(g, 0, 16383, T)
        s["cos_sin"] = _cos_sin(16384, c["rot"])
    elif op == "kv":
        B, S, Hkv, D, page = c["B"], c["S"], c["Hkv"], c["D"], c["page"]
        start = _rand_int(g, c["past"] // 2, c["past"], B)
        lens = _rand_int(g, (S + 1) // 2, S, B)
        s["start"], s["lens"] = start, lens
        s["block_table"], P = _tables(g, B, (c["past"] + S - 1) // page + 2)
        s["k_cache"], s["k_scale"] = _filled_cache(g, P, Hkv, page, D)
        s["v_cache"], s["v_scale"] = _filled_cache(g, P, Hkv, page, D)
        kv = _randn(g, B, S, 2 * Hkv * D)
        kv *= torch.exp(0.5 * _randn(g, B, S, 1))  # tokens of uneven magnitude: some raise their page's scale
        kv = kv.to(torch.bfloat16)
        s["k"], s["v"] = kv[..., :Hkv * D].unflatten(2, (Hkv, D)), kv[..., Hkv * D:].unflatten(2, (Hkv, D))
        end = start + lens
        s["read_start"] = (end - c["read"]).clamp(min=0)
        s["read_lens"] = end - s["read_start"]
    else:
        B, Sq, Hq, Hkv, D, page, L = c["B"], c["Sq"], c["Hq"], c["Hkv"], c["D"], c["page"], c["L"]
        lens = _rand_int(g, max(1, L // 8), L, B) if c["ragged"] else torch.full((B,), L, dtype=torch.int32, device="cuda")
        lens[0] = L
        s["seq_lens"] = lens
        s["block_table"], P = _tables(g, B, (L + page - 1) // page)
        s["k_cache"], s["k_scale"] = _filled_cache(g, P, Hkv, page, D)
        s["v_cache"], s["v_scale"] = _filled_cache(g, P, Hkv, page, D)
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

        if op == "router":
            return wd.moe_router_scored_topk(s["logits"], s["K"], s["scoring"], s["bias"], s["groups"], s["pick"],
                                             s["top"], s["renorm"], s["scale"])
        if op == "qk_norm":
            return wd.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["cos_sin"], EPS,
                                   s["interleaved"])
        if op == "kv":
            wd.kv_cache_write_fp8(s["k"], s["v"], s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"],
                                  s["block_table"], s["start"], s["lens"])
            return wd.kv_cache_read_fp8(s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], s["block_table"],
                                        s["read_start"], s["read"], s["read_lens"])
        return wd.attn_decode_fp8(s["q"], s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], s["block_table"],
                                  s["seq_lens"], window=s["window"], workspace=s["workspace"])
    if op == "router":
        return _plain_router(s)
    if op == "qk_norm":
        return (_plain_norm_rope(s["q"], s["q_weight"], s), _plain_norm_rope(s["k"], s["k_weight"], s))
    if op == "kv":
        _plain_write(s, s["k"], s["k_cache"], s["k_scale"])
        _plain_write(s, s["v"], s["v_cache"], s["v_scale"])
        return _plain_read(s, s["k_cache"], s["k_scale"]), _plain_read(s, s["v_cache"], s["v_scale"])
    return _plain_attn(s)


def _plain_router(s):
    T, E, K = s["T"], s["E"], s["K"]
    x = s["logits"].float()
    if s["scoring"] == "softmax":
        e = torch.exp(x - x.amax(dim=1, keepdim=True))
        score = e / e.sum(dim=1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    # without a bias, and groups ranked by their best expert, the logits rank the experts as their scores do
    choice = score + s["bias"] if s["bias"] is not None else score if s["top"] == 2 else x
    if s["groups"] > 1:
        each = choice.view(T, s["groups"], E // s["groups"])
        rank = each.sort(dim=2, descending=True).values[..., :s["top"]].sum(dim=2)
        best = rank.sort(dim=1, descending=True, stable=True).indices[:, :s["pick"]]
        kept = torch.zeros(T, s["groups"], dtype=torch.bool, device=x.device).scatter_(1, best, True)
        choice = torch.where(kept[..., None], each, float("-inf")).view(T, E)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :K]
    w = score.gather(1, ids)
    if s["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return ids.to(torch.int32), w * s["scale"]


def _plain_norm_rope(x, weight, s):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.float()
    rot = s["rot"]
    cs = s["cos_sin"][s["positions"].long()][:, None, :]
    cos, sin = cs[..., :rot // 2], cs[..., rot // 2:]
    if s["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1).to(torch.bfloat16)


def _values(codes, scale):
    """What codes [..., tokens, D] stand for, scale bytes [...]."""
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(), (scale.int() - 127)[..., None, None])


def _plain_write(s, x, cache, scale):
    B, S, page = s["B"], s["S"], s["page"]
    H, D = x.shape[2], x.shape[3]
    N = (S - 1) // page + 2  # pages that a sequence's new tokens can touch
    first = s["start"] // page
    off, stop = (s["start"] % page)[:, None], (s["start"] % page + s["lens"])[:, None]
    slot = torch.arange(N * page, device=x.device)[None, :]
    is_new = (slot >= off) & (slot < stop)  # [B, N*page]
    is_old = slot < off
    at = first[:, None] + torch.arange(N, device=x.device)
    touched = at * page < (s["start"] + s["lens"])[:, None]
    pid = torch.where(touched, s["block_table"].gather(1, at.clamp(max=s["block_table"].shape[1] - 1).long()), 0).long()
    was = scale[pid]  # [B, N, H]
    old = _values(cache[pid], was).permute(0, 1, 3, 2, 4).reshape(B, N * page, H, D)
    new = x.float().gather(1, (slot - off).clamp(0, S - 1)[..., None, None].expand(B, N * page, H, D))
    new = torch.where(is_new[..., None, None], new, 0.0)
    m, e = torch.frexp(new.view(B, N, page, H, D).abs().amax(dim=(2, 4)))
    need = torch.where(m > 0, e - 9 + (m > 0.875) + 127, 1).clamp(1, 254)
    had = (is_old.view(B, N, page).any(dim=2))[..., None]
    now = torch.where(had, torch.maximum(need, was.int()), need)  # [B, N, H]
    v = torch.where(is_new[..., None, None], new, old).view(B, N, page, H, D).permute(0, 1, 3, 2, 4)
    codes = torch.ldexp(v, (127 - now)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    live = (is_new | is_old).view(B, N, 1, page, 1)
    cache[pid] = torch.where(live, codes, cache[pid])
    scale[pid] = now.to(torch.uint8)


def _plain_read(s, cache, scale):
    page, R = s["page"], s["read"]
    at = s["read_start"][:, None] + torch.arange(R, device=cache.device)  # [B, R]
    live = torch.arange(R, device=cache.device) < s["read_lens"][:, None]
    pid = s["block_table"].gather(1, (at // page).clamp(max=s["block_table"].shape[1] - 1).long()).long()
    v = _values(cache[pid, :, (at % page).long()].unsqueeze(3), scale[pid]).squeeze(3)  # [B, R, H, D]
    return torch.where(live[..., None, None], v, 0.0).to(torch.bfloat16)


def _plain_attn(s):
    B, Sq, Hq, Hkv, D, page = s["B"], s["Sq"], s["Hq"], s["Hkv"], s["D"], s["page"]
    G = Hq // Hkv
    table = s["block_table"].long()
    M = table.shape[1]
    k = _values(s["k_cache"][table], s["k_scale"][table]).permute(0, 2, 1, 3, 4).reshape(B, Hkv, M * page, D)
    v = _values(s["v_cache"][table], s["v_scale"][table]).permute(0, 2, 1, 3, 4).reshape(B, Hkv, M * page, D)
    q = s["q"].float().view(B, Sq, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Sq * G, D)
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    at = torch.arange(M * page, device=q.device)
    pos = (s["seq_lens"][:, None] - Sq + torch.arange(Sq, device=q.device))[..., None]  # [B, Sq, 1]
    seen = at <= pos
    if s["window"]:
        seen = seen & (at > pos - s["window"])
    seen = seen[:, None, :, None, :].expand(B, 1, Sq, G, M * page).reshape(B, 1, Sq * G, M * page)
    x = torch.where(seen, x, float("-inf"))
    top = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - torch.where(top > float("-inf"), top, 0.0))
    o = torch.matmul(p, v)
    den = p.sum(dim=-1, keepdim=True)
    o = torch.where(den > 0, o / den, 0.0)
    return o.view(B, Hkv, Sq, G, D).permute(0, 2, 1, 3, 4).reshape(B, Sq, Hq, D).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c, op = case, case["op"]
    if op == "router":
        per = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": c["T"] * (c["E"] * per + c["K"] * 8) + (4 * c["E"] if c["bias"] else 0),
                "flops": 4.0 * c["T"] * c["E"]}
    if op == "qk_norm":
        n = c["T"] * (c["Hq"] + c["Hkv"]) * c["D"]
        return {"bytes": 4 * n + c["T"] * (4 + 4 * c["rot"]) + 4 * c["D"], "flops": 8.0 * n}
    if op == "kv":
        one = 2 * c["Hkv"] * c["D"]  # values of a token; lengths are S * 3/4 on average
        new, back = 0.75 * c["B"] * c["S"], c["B"] * min(c["read"], 0.75 * (c["past"] + c["S"]))
        return {"bytes": one * (3 * new + back + 2 * c["B"] * c["read"]), "flops": 2.0 * one * (new + back)}
    mean = c["L"] if not c["ragged"] else (c["L"] + (c["B"] - 1) * 0.5625 * c["L"]) / c["B"]
    keys = min(mean, c["window"] + c["Sq"] - 1) if c["window"] else mean
    kv = 2.0 * c["B"] * keys * c["Hkv"] * c["D"]
    return {"bytes": kv + 4.0 * c["B"] * c["Sq"] * c["Hq"] * c["D"],
            "flops": 4.0 * c["B"] * c["Sq"] * c["Hq"] * c["D"] * keys}


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "router":
        return _exact_router(s)
    if op == "qk_norm":
        return _exact_norm_rope(s, s["q"], s["q_weight"]), _exact_norm_rope(s, s["k"], s["k_weight"])
    if op == "kv":
        return _exact_kv(s, s["k"], s["k_cache"], s["k_scale"]), _exact_kv(s, s["v"], s["v_cache"], s["v_scale"])
    return _exact_attn(s)


def _exact_router(s):
    x = s["logits"].double()
    score = torch.softmax(x, dim=1) if s["scoring"] == "softmax" else torch.sigmoid(x)
    choice = score if s["bias"] is None else score + s["bias"].double()
    if s["groups"] > 1:
        size = s["E"] // s["groups"]
        rank = torch.stack([choice[:, g * size:(g + 1) * size].topk(s["top"], dim=1).values.sum(dim=1)
                            for g in range(s["groups"])], dim=1)
        order = rank.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
        out = (order >= s["pick"]).repeat_interleave(size, dim=1)
        choice = choice.masked_fill(out, -1e300)
    ids = choice.argsort(dim=1, descending=True, stable=True)[:, :s["K"]]
    w = torch.take_along_dim(score, ids, dim=1)
    if s["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return None, w * s["scale"]


def _exact_norm_rope(s, x, weight):
    x, rot = x.double(), s["rot"]
    y = x / torch.sqrt(x.square().sum(dim=-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    half = rot // 2
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + half)
    cs = s["cos_sin"].double()[s["positions"].long()]
    turn = torch.complex(cs[:, None, :half], cs[:, None, half:])
    z = torch.complex(y[..., a], y[..., b]) * turn
    out = y.clone()
    out[..., a], out[..., b] = z.real, z.imag
    return out


def _round_e4m3(x):
    """Nearest E4M3 value, ties to even, of doubles within its range."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(x / step) * step


def _exact_kv(s, x, cache, scale):
    B, page, R = s["B"], s["page"], s["read"]
    out = torch.zeros(B, R, x.shape[2], x.shape[3], dtype=torch.float64, device=x.device)
    start, lens, rs, rl = (s[k].tolist() for k in ("start", "lens", "read_start", "read_lens"))
    table = s["block_table"].tolist()
    if sum(r // page + 2 for r in rl) > 20000:
        return None
    for b in range(B):
        end = start[b] + lens[b]
        for n in range(rs[b] // page, (rs[b] + rl[b] - 1) // page + 1):
            pid, t0 = table[b][n], n * page
            old = cache[pid, :, :max(0, min(page, start[b] - t0))].view(torch.float8_e4m3fn).double()
            exps = scale[pid].double() - 127.0
            lo, hi = max(start[b], t0), min(end, t0 + page)
            if lo < hi:
                new = x[b, lo - start[b]:hi - start[b]].double().transpose(0, 1)  # [H, n, D]
                most = new.abs().amax(dim=(1, 2)).clamp(min=1e-38)
                need = torch.ceil(torch.log2(most / E4M3_MAX))
                need = torch.where(torch.exp2(need - 1) * E4M3_MAX >= most, need - 1, need)
                need = torch.where(torch.exp2(need) * E4M3_MAX < most, need + 1, need)
                if old.shape[1]:
                    need = torch.maximum(need, exps)
                    old = _round_e4m3(old * torch.exp2(exps - need)[:, None, None])
                new = _round_e4m3(new * torch.exp2(-need)[:, None, None])
                vals = torch.cat([old, new], dim=1)
                exps = need
            else:
                vals = old
            vals = vals * torch.exp2(exps)[:, None, None]
            a, z = max(rs[b], t0), min(rs[b] + rl[b], t0 + page)
            out[b, a - rs[b]:z - rs[b]] = vals[:, a - t0:z - t0].transpose(0, 1)
    return out


def _exact_attn(s):
    B, Sq, Hq, Hkv, D, page, W = (s[k] for k in ("B", "Sq", "Hq", "Hkv", "D", "page", "window"))
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(s["seq_lens"].tolist()):
        pids = s["block_table"][b, :(n + page - 1) // page].long()
        k, v = ((s[c + "_cache"][pids].view(torch.float8_e4m3fn).double()
                 * torch.exp2(s[c + "_scale"][pids].double() - 127.0)[:, :, None, None])
                .transpose(0, 1).flatten(1, 2)[:, :n] for c in "kv")  # [Hkv, n, D]
        for i in range(Sq):
            pos = n - Sq + i
            if pos < 0:
                continue
            lo = max(0, pos - W + 1) if W else 0
            q = s["q"][b, i].double().view(Hkv, Hq // Hkv, D)
            p = torch.softmax(torch.bmm(q, k[:, lo:pos + 1].transpose(1, 2)) / math.sqrt(D), dim=-1)
            out[b, i] = torch.bmm(p, v[:, lo:pos + 1]).reshape(Hq, D)
    return out
