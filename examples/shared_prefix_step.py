"""Decoding steps of one decoder layer for a batch of answers to one prompt, with every
operator of the framework and no matrix product but the router's left to torch.

    python examples/shared_prefix_step.py

The prompt's keys and values are written once; every sequence's table begins with the
prompt's pages. A step is

    qkv = linear_w4(h)                               4-bit weights
    q, k = qk_norm_rope(q, k)
    kv_cache_write_fp8(k, v -> own pages)
    o = attn_decode_fp8_prefix(q, cache)             the prompt's pages read once for all
    h, r = block_norm(linear_w4(o), r)               residual and the next norm in one pass
    ids, weights = moe_router_scored_topk(h @ w_gate)
    h, r = block_norm(moe_ffn_3d_batched(h, ...), r, post_weight)

The script repeats every step in plain fp32 torch on the values that the cache holds
and prints how far apart the two residual streams are.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

HIDDEN, INTER, EXPERTS, TOPK = 1024, 128, 64, 4
HQ, HKV, D, PAGE, MAX_POS, GROUP = 16, 2, 128, 64, 4096, 64
GROUPS, PICK, EPS = 8, 4, 1e-6


class Layer:
    """The layer's weights, its cache and what its steps keep."""

    def __init__(self, batch: int, prompt: int, own: int, seed: int = 0, device: str = "cuda"):
        from warp_decode_b200 import w4
        from warp_decode_b200 import warp_decode as wd

        g = torch.Generator(device=device).manual_seed(seed)

        def rand(*shape, scale=1.0):
            return (torch.randn(*shape, generator=g, device=device) * scale).to(torch.bfloat16)

        self.w_qkv = rand((HQ + 2 * HKV) * D, HIDDEN, scale=HIDDEN ** -0.5)
        self.w_o = rand(HIDDEN, HQ * D, scale=(HQ * D) ** -0.5)
        self.qkv4, self.o4 = (w4.quantize_w4(w, GROUP, zero_points=True) for w in (self.w_qkv, self.w_o))
        # the plain steps multiply by what the packed weights stand for
        self.w_qkv = w4.dequantize_w4(*self.qkv4, HIDDEN)
        self.w_o = w4.dequantize_w4(*self.o4, HQ * D)
        self.w_gate = rand(HIDDEN, EXPERTS, scale=HIDDEN ** -0.5)
        self.gate_bias = torch.randn(EXPERTS, generator=g, device=device) * 0.1
        self.w_gate_up = rand(EXPERTS, 2 * INTER, HIDDEN, scale=HIDDEN ** -0.5)
        self.w_down = rand(EXPERTS, HIDDEN, INTER, scale=INTER ** -0.5)
        norm = lambda n: 1 + 0.1 * torch.randn(n, generator=g, device=device)  # noqa: E731
        self.q_norm, self.k_norm, self.attn_norm, self.ffn_norm, self.post_norm = (
            norm(n) for n in (D, D, HIDDEN, HIDDEN, HIDDEN))
        angle = torch.arange(MAX_POS, device=device)[:, None] * 1e4 ** (-torch.arange(0, D, 2, device=device) / D)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous()
        shared, each = prompt // PAGE, -(-own // PAGE)
        pages = shared + batch * each
        pool = torch.randperm(pages, generator=g, device=device).to(torch.int32)
        self.table = torch.cat([pool[:shared].expand(batch, shared), pool[shared:].view(batch, each)], 1).contiguous()
        self.cache = [torch.zeros(pages, HKV, PAGE, D, dtype=torch.uint8, device=device),
                      torch.zeros(pages, HKV, dtype=torch.uint8, device=device),
                      torch.zeros(pages, HKV, PAGE, D, dtype=torch.uint8, device=device),
                      torch.zeros(pages, HKV, dtype=torch.uint8, device=device)]
        self.prefix_len = torch.tensor([shared * PAGE], dtype=torch.int32, device=device)
        self.seq_lens = self.prefix_len.expand(batch).contiguous()
        self.workspace = wd.attn_decode_fp8_prefix_workspace(batch, 1, HQ, HKV, D)

    def project(self, h: torch.Tensor, pos: torch.Tensor):
        from warp_decode_b200 import warp_decode as wd

        q, k, v = wd.linear_w4(h, *self.qkv4).split([HQ * D, HKV * D, HKV * D], dim=-1)
        q, k = wd.qk_norm_rope(q.unflatten(1, (HQ, D)), k.unflatten(1, (HKV, D)), self.q_norm, self.k_norm, pos,
                               self.cos_sin, EPS)
        return q, k, v.unflatten(1, (HKV, D))

    def read_prompt(self, x: torch.Tensor) -> None:
        """Keys and values of the prompt x [prompt, hidden], written once, through the first table."""
        from warp_decode_b200 import warp_decode as wd

        h, _ = wd.block_norm(x, torch.zeros_like(x), self.attn_norm, eps=EPS)
        _, k, v = self.project(h, torch.arange(x.shape[0], dtype=torch.int32, device=x.device))
        zero = torch.zeros(1, dtype=torch.int32, device=x.device)
        wd.kv_cache_write_fp8(k[None], v[None], *self.cache, self.table[:1].contiguous(), zero)

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """x [batch, hidden]: one new token of each sequence; the residual stream after the layer, fp32."""
        from warp_decode_b200 import warp_decode as wd

        h, r = wd.block_norm(x, torch.zeros_like(x, dtype=torch.float32), self.attn_norm, eps=EPS)
        start = self.seq_lens
        q, k, v = self.project(h, start)
        wd.kv_cache_write_fp8(k[:, None], v[:, None], *self.cache, self.table, start)
        self.seq_lens = start + 1
        o = wd.attn_decode_fp8_prefix(q[:, None], *self.cache, self.table, self.seq_lens, self.prefix_len,
                                      workspace=self.workspace)
        h, r = wd.block_norm(wd.linear_w4(o.view(-1, HQ * D), *self.o4), r, self.ffn_norm, eps=EPS, inplace=True)
        ids, weights = wd.moe_router_scored_topk((h @ self.w_gate).float(), TOPK, "sigmoid", self.gate_bias, GROUPS,
                                                 PICK, 2)
        y = wd.moe_ffn_3d_batched(h, self.w_gate_up, self.w_down, ids, weights)
        return wd.block_norm(y, r, self.attn_norm, self.post_norm, residual_scale=0.5, eps=EPS, inplace=True)[1]

    def plain(self, x: torch.Tensor, start: torch.Tensor) -> torch.Tensor:
        """The step after `step` has written the cache, in fp32 torch on the cache's values."""
        from warp_decode_b200 import warp_decode as wd

        def norm(v, w):
            return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * w

        bf = lambda v: v.to(torch.bfloat16).float()  # noqa: E731
        r = x.float()
        qkv = bf(bf(norm(r, self.attn_norm)) @ self.w_qkv.t())
        q = norm(qkv[:, :HQ * D].unflatten(1, (HQ, D)), self.q_norm)
        c, s = self.cos_sin[start.long()].unsqueeze(1).chunk(2, dim=-1)
        a, b = q.chunk(2, dim=-1)
        q = bf(torch.cat([a * c - b * s, b * c + a * s], dim=-1))
        longest = int(start.max()) + 1
        k, v = (t.float() for t in wd.kv_cache_read_fp8(*self.cache, self.table, torch.zeros_like(start), longest,
                                                        start + 1))
        k, v = (t.repeat_interleave(HQ // HKV, dim=2) for t in (k, v))
        score = torch.einsum("bhd,bthd->bht", q, k) / math.sqrt(D)
        score = score.masked_fill(torch.arange(longest, device=x.device) > start[:, None, None], -torch.inf)
        o = bf(torch.einsum("bht,bthd->bhd", score.softmax(-1), v))
        r = r + bf(o.flatten(1) @ self.w_o.t())
        h = bf(norm(r, self.ffn_norm))
        gate = torch.sigmoid(bf(h @ self.w_gate.float()))
        choice = gate + self.gate_bias
        rank = choice.unflatten(-1, (GROUPS, -1)).topk(2, dim=-1).values.sum(-1)
        kept = torch.zeros_like(rank).scatter_(-1, rank.topk(PICK, dim=-1).indices, 1.0).bool()
        ids = choice.masked_fill(~kept.repeat_interleave(EXPERTS // GROUPS, dim=-1), -torch.inf).topk(TOPK, -1).indices
        w = gate.gather(-1, ids)
        w = w / w.sum(-1, keepdim=True)
        gu = torch.einsum("bh,bkih->bki", h, self.w_gate_up[ids].float())
        act = bf(torch.nn.functional.silu(gu[..., :INTER]) * gu[..., INTER:])
        y = bf((torch.einsum("bki,bkhi->bkh", act, self.w_down[ids].float()) * w[..., None]).sum(1))
        return 0.5 * r + norm(y, self.post_norm)


def main(batch: int = 12, prompt: int = 320, steps: int = 4) -> float:
    """Runs the prompt and `steps` tokens of each answer; the largest relative distance from the plain steps."""
    from warp_decode_b200 import warp_decode as wd

    layer = Layer(batch, prompt, steps)
    g = torch.Generator(device="cuda").manual_seed(1)
    layer.read_prompt(torch.randn(prompt, HIDDEN, generator=g, device="cuda").to(torch.bfloat16))
    worst = 0.0
    for step in range(steps):
        x = torch.randn(batch, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
        start = layer.seq_lens.clone()
        y, ref = layer.step(x), layer.plain(x, start)
        far = ((y - ref).norm(dim=-1) / ref.norm(dim=-1)).max().item()
        print(f"step {step}: {batch} sequences of {int(start[0]) + 1} tokens, relative distance {far:.2e}")
        worst = max(worst, far)
    status = wd.status(True, 0)
    assert status == 0, f"device status word {status:#x}"
    return worst


if __name__ == "__main__":
    main()
