"""One decoder layer's serving steps with every operator of the framework: a prompt
of uneven lengths, then single tokens.

    python examples/decoder_layer_step.py

A step of a layer is

    qkv = norm(x) @ w_qkv
    q, k = qk_norm_rope(q, k)                      per-head norm, position rotation
    kv_cache_write_fp8(k, v -> paged cache)        quantised as it is written
    o = attn_decode_fp8(q, cache)                  the step's tokens over all before
    x = x + o @ w_o
    ids, weights = moe_router_scored_topk(norm(x) @ w_gate)
    x = x + moe_ffn_3d_batched(norm(x), ..., ids, weights)

with the matrix products outside the framework's operators left to torch.  The
script repeats every step in plain fp32 torch on the values that the cache holds
and prints how far apart the two are.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

HIDDEN, INTER, EXPERTS, TOPK = 1024, 128, 64, 4
HQ, HKV, D, PAGE, MAX_POS = 16, 2, 128, 64, 4096
GROUPS, PICK, EPS = 8, 4, 1e-6


class Layer:
    """The layer's weights, its cache and what its steps keep."""

    def __init__(self, batch: int, max_len: int, seed: int = 0, device: str = "cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def rand(*shape, scale=1.0):
            return (torch.randn(*shape, generator=g, device=device) * scale).to(torch.bfloat16)

        self.w_qkv = rand(HIDDEN, (HQ + 2 * HKV) * D, scale=HIDDEN ** -0.5)
        self.w_o = rand(HQ * D, HIDDEN, scale=(HQ * D) ** -0.5)
        self.w_gate = rand(HIDDEN, EXPERTS, scale=HIDDEN ** -0.5)
        self.gate_bias = torch.randn(EXPERTS, generator=g, device=device) * 0.1
        self.w_gate_up = rand(EXPERTS, 2 * INTER, HIDDEN, scale=HIDDEN ** -0.5)
        self.w_down = rand(EXPERTS, HIDDEN, INTER, scale=INTER ** -0.5)
        self.q_norm = 1 + 0.1 * torch.randn(D, generator=g, device=device)
        self.k_norm = 1 + 0.1 * torch.randn(D, generator=g, device=device)
        angle = torch.arange(MAX_POS, device=device)[:, None] * 1e4 ** (-torch.arange(0, D, 2, device=device) / D)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous()
        columns = -(-max_len // PAGE)
        pages = batch * columns
        self.table = torch.randperm(pages, generator=g, device=device).to(torch.int32).view(batch, columns)
        self.cache = [torch.zeros(pages, HKV, PAGE, D, dtype=torch.uint8, device=device),
                      torch.zeros(pages, HKV, dtype=torch.uint8, device=device),
                      torch.zeros(pages, HKV, PAGE, D, dtype=torch.uint8, device=device),
                      torch.zeros(pages, HKV, dtype=torch.uint8, device=device)]
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.workspace = None

    @staticmethod
    def norm(x):
        return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + EPS)).to(torch.bfloat16)

    def step(self, x: torch.Tensor, lens: torch.Tensor) -> torch.Tensor:
        """x [B, S, hidden]: S new tokens of each sequence, of which the first lens[b] count."""
        from warp_decode_b200 import warp_decode as wd

        B, S, _ = x.shape
        qkv = self.norm(x) @ self.w_qkv
        q, k, v = qkv.split([HQ * D, HKV * D, HKV * D], dim=-1)
        v = v.unflatten(2, (HKV, D))
        start = self.seq_lens
        # a padding token's position does not matter: neither its key nor its output is used
        pos = (start[:, None] + torch.arange(S, device=x.device, dtype=torch.int32)).flatten()
        q, k = wd.qk_norm_rope(q.reshape(B * S, HQ, D), k.reshape(B * S, HKV, D), self.q_norm, self.k_norm, pos,
                               self.cos_sin, EPS)
        wd.kv_cache_write_fp8(k.view(B, S, HKV, D), v, *self.cache, self.table, start, lens)
        self.seq_lens = start + lens
        if self.workspace is None or S > 1:  # a step of more rows needs more of it
            self.workspace = wd.attn_decode_fp8_workspace(B, S, HQ, HKV, D, x.device.index)
        o = self.attend(q.view(B, S, HQ, D), lens)
        x = x + o.flatten(2) @ self.w_o
        h = self.norm(x).flatten(0, 1).contiguous()
        ids, weights = wd.moe_router_scored_topk((h @ self.w_gate).float(), TOPK, "sigmoid", self.gate_bias, GROUPS,
                                                 PICK, 2)
        return x + wd.moe_ffn_3d_batched(h, self.w_gate_up, self.w_down, ids, weights).view_as(x)

    def attend(self, q, lens):
        """Attention takes a sequence's last S tokens: rows past lens[b] go round to the front, where none is seen."""
        from warp_decode_b200 import warp_decode as wd

        S = q.shape[1]
        at = torch.arange(S, device=q.device)[None, :]
        turn = lambda t, by: t.gather(1, ((at + by[:, None]) % S)[..., None, None].expand_as(t))  # noqa: E731
        if S > 1:
            q = turn(q, lens - S)
        o = wd.attn_decode_fp8(q, *self.cache, self.table, self.seq_lens, workspace=self.workspace)
        return turn(o, S - lens) if S > 1 else o

    def plain(self, x: torch.Tensor, lens: torch.Tensor, start: torch.Tensor) -> torch.Tensor:
        """The step after `step` has written the cache, in fp32 torch on the cache's values."""
        from warp_decode_b200 import warp_decode as wd

        B, S, _ = x.shape
        qkv = (self.norm(x) @ self.w_qkv).float()
        q = qkv[..., :HQ * D].unflatten(2, (HQ, D))
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * self.q_norm
        pos = start[:, None] + torch.arange(S, device=x.device)
        c, s = self.cos_sin[pos].unsqueeze(2).chunk(2, dim=-1)
        a, b = q.chunk(2, dim=-1)
        q = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
        longest = int((start + lens).max())
        k, v = (t.float() for t in wd.kv_cache_read_fp8(*self.cache, self.table, torch.zeros_like(start), longest,
                                                        start + lens))
        k, v = (t.repeat_interleave(HQ // HKV, dim=2) for t in (k, v))
        score = torch.einsum("bshd,bthd->bhst", q, k) / math.sqrt(D)
        seen = torch.arange(longest, device=x.device) <= pos[..., None]
        score = score.masked_fill(~seen[:, None], -torch.inf)
        o = torch.einsum("bhst,bthd->bshd", score.softmax(-1), v).to(torch.bfloat16)
        x = x + o.flatten(2) @ self.w_o
        h = self.norm(x)
        gate = torch.sigmoid((h @ self.w_gate).float())
        choice = gate + self.gate_bias
        rank = choice.unflatten(-1, (GROUPS, -1)).topk(2, dim=-1).values.sum(-1)
        kept = torch.zeros_like(rank).scatter_(-1, rank.topk(PICK, dim=-1).indices, 1.0).bool()
        ids = choice.masked_fill(~kept.repeat_interleave(EXPERTS // GROUPS, dim=-1), -torch.inf).topk(TOPK, -1).indices
        w = gate.gather(-1, ids)
        w = w / w.sum(-1, keepdim=True)
        gu = torch.einsum("bsh,bskih->bski", h.float(), self.w_gate_up[ids].float())
        act = (torch.nn.functional.silu(gu[..., :INTER]) * gu[..., INTER:]).to(torch.bfloat16).float()
        y = torch.einsum("bski,bskhi->bskh", act, self.w_down[ids].float())
        return x + (y * w[..., None]).sum(2).to(torch.bfloat16)


def main(steps: int = 4) -> float:
    """Runs a prompt and `steps` single tokens; the largest relative distance from the plain steps."""
    from warp_decode_b200 import warp_decode as wd

    lens = torch.tensor([70, 9, 33], dtype=torch.int32, device="cuda")
    B, S = 3, int(lens.max())
    layer = Layer(B, S + steps)
    g = torch.Generator(device="cuda").manual_seed(1)
    worst = 0.0
    for step in range(steps + 1):
        n, tokens = (lens, S) if step == 0 else (torch.ones_like(lens), 1)
        x = torch.randn(B, tokens, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
        start = layer.seq_lens.clone()
        y, ref = layer.step(x, n), layer.plain(x, n, start)
        live = torch.arange(tokens, device="cuda") < n[:, None]
        far = ((y - ref).float()[live].norm(dim=-1) / ref.float()[live].norm(dim=-1)).max().item()
        print(f"step {step}: {int(n.sum())} tokens, lengths {layer.seq_lens.tolist()}, relative distance {far:.2e}")
        worst = max(worst, far)
    status = wd.status(True, 0)
    assert status == 0, f"device status word {status:#x}"
    return worst


if __name__ == "__main__":
    main()
