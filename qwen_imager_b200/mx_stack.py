"""A dual-stream DiT stack in MXFP4: the block operators as they are used together.

The block of dit_stack.py (image and text streams with their own weights, joint
attention) with four-bit activations and weights, normed and rotated q and k, and
norms on both sides of each sublayer:

  mods   = mod(silu(temb))                                     six vectors a stream, one token
  n      = mx(layer_norm(x) (1 + scale1) + shift1)             gated_residual_norm(quantize=True)
  qkv    = n . Wqkv^T                                          MxLinear on an MxTensor
  q, k   = rotate(rms(q) wq, rms(k) wk)                        qk_norm_rotary, in place
  a      = attention(q, k, v) over both streams' tokens        torch
  x, n   = x + gate1 rms(a . Wout^T) w1,  mx(layer_norm(x) ...)  gated_residual_norm
  h      = gelu(n . Wup^T)
  x, n   = x + gate2 rms(h . Wdown^T) w2, mx(layer_norm(x) ...)  with the next block's modulation

so between the linears there is one pass over the hidden state a sublayer, and
activations reach the linears as four-bit codes.  Run as a module it times one step:

  python -m qwen_imager_b200.mx_stack --blocks 4 --height 64 --width 64 --text 256
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch
import torch.nn.functional as F

from .gated_norm import gated_residual_norm
from .mxfp4 import MxLinear, MxTensor
from .rotary import RotaryAxes, qk_norm_rotary

EPS = 1e-6


@dataclass(frozen=True)
class MxStackConfig:
    """Shape of the stack; height x width image tokens (one frame), then text tokens."""

    height: int
    width: int
    text: int
    blocks: int = 60
    hidden: int = 3072
    heads: int = 24
    head_dim: int = 128
    ffn: int = 12288
    axes: Tuple[int, ...] = (8, 28, 28)  # pairs of a head turned by frame, row and column
    theta: float = 10000.0

    def __post_init__(self):
        if 2 * sum(self.axes) > self.head_dim or len(self.axes) != 3:
            raise ValueError(f"axes {self.axes} do not fit heads of {self.head_dim}")

    @property
    def image(self) -> int:
        return self.height * self.width

    @property
    def tokens(self) -> int:
        return self.image + self.text


def joint_positions(cfg: MxStackConfig, device="cuda") -> torch.Tensor:
    """int32 [tokens, 3]: (frame, row, column) of the image tokens, rows and columns
    counted from the middle; text tokens go on along every axis from the larger half."""
    row = torch.arange(cfg.height, dtype=torch.int32) - cfg.height // 2
    col = torch.arange(cfg.width, dtype=torch.int32) - cfg.width // 2
    grid = torch.stack([torch.zeros((cfg.height, cfg.width), dtype=torch.int32), row[:, None].expand(cfg.height, cfg.width),
                        col[None, :].expand(cfg.height, cfg.width)], -1).reshape(-1, 3)
    text = max(cfg.height, cfg.width) // 2 + torch.arange(cfg.text, dtype=torch.int32)
    return torch.cat([grid, text[:, None].expand(cfg.text, 3)]).contiguous().to(device)


@dataclass
class MxStream:
    """One stream's weights in one block."""

    mod: MxLinear              # hidden -> 6 hidden
    qkv: MxLinear              # hidden -> 3 heads head_dim
    out: MxLinear              # heads head_dim -> hidden
    up: MxLinear               # hidden -> ffn
    down: MxLinear             # ffn -> hidden
    q_norm: torch.Tensor       # [head_dim]
    k_norm: torch.Tensor
    post_attn: torch.Tensor    # [hidden], RMSNorm of the attention's output
    post_ffn: torch.Tensor     # [hidden], RMSNorm of the feed-forward's output

    @classmethod
    def random(cls, cfg: MxStackConfig, generator: torch.Generator, device) -> "MxStream":
        def lin(n, k):
            w = torch.randn((n, k), generator=generator, device=device) * k ** -0.5
            return MxLinear.from_dense(w, torch.randn((n,), generator=generator, device=device) * 0.01)

        def weight(n):
            return (1.0 + 0.1 * torch.randn((n,), generator=generator, device=device)).to(torch.bfloat16)

        d = cfg.heads * cfg.head_dim
        return cls(mod=lin(6 * cfg.hidden, cfg.hidden), qkv=lin(3 * d, cfg.hidden), out=lin(cfg.hidden, d), up=lin(cfg.ffn, cfg.hidden),
                   down=lin(cfg.hidden, cfg.ffn), q_norm=weight(cfg.head_dim), k_norm=weight(cfg.head_dim), post_attn=weight(cfg.hidden),
                   post_ffn=weight(cfg.hidden))


class MxStack:
    """The stack on one GPU."""

    def __init__(self, cfg: MxStackConfig, blocks: List[List[MxStream]]):
        self.cfg, self.blocks = cfg, blocks
        device = blocks[0][0].qkv.device
        self.positions = joint_positions(cfg, device)
        self.axes = RotaryAxes(cfg.axes, theta=cfg.theta, pairs="adjacent", device=device)

    @classmethod
    def random(cls, cfg: MxStackConfig, seed: int = 0, device="cuda") -> "MxStack":
        g = torch.Generator(device=device).manual_seed(seed)
        return cls(cfg, [[MxStream.random(cfg, g, device) for _ in range(2)] for _ in range(cfg.blocks)])

    def modulations(self, temb: torch.Tensor) -> torch.Tensor:
        """bf16 [blocks, 2, 6, hidden]: shift1, scale1, gate1, shift2, scale2, gate2 of every block and stream."""
        t = F.silu(temb.float()).to(torch.bfloat16).reshape(1, self.cfg.hidden)
        return torch.cat([s.mod.forward(t) for b in self.blocks for s in b]).view(len(self.blocks), 2, 6, self.cfg.hidden)

    def forward(self, x: torch.Tensor, temb: torch.Tensor) -> torch.Tensor:
        """x: bf16 [image + text tokens, hidden], image tokens first, updated in place; temb: bf16 [hidden]."""
        cfg = self.cfg
        if x.shape != (cfg.tokens, cfg.hidden):
            raise ValueError(f"hidden state {tuple(x.shape)} is not [{cfg.tokens}, {cfg.hidden}]")
        rows = (slice(0, cfg.image), slice(cfg.image, cfg.tokens))
        mods = self.modulations(temb)
        d = cfg.heads * cfg.head_dim
        qkv = torch.empty((cfg.tokens, 3, cfg.heads, cfg.head_dim), dtype=x.dtype, device=x.device)
        n: List[Optional[MxTensor]] = [gated_residual_norm(x[rows[s]], pre="layer", scale=mods[0, s, 1], shift=mods[0, s, 0], eps=EPS,
                                                           quantize=True)[1] for s in range(2)]
        for b, block in enumerate(self.blocks):
            m = mods[b]
            for s, w in enumerate(block):
                part = qkv[rows[s]]
                w.qkv.forward_fused(n[s], out=part.view(-1, 3 * d))
                qk_norm_rotary(part[:, 0], part[:, 1], self.positions[rows[s]], self.axes, q_weight=w.q_norm, k_weight=w.k_norm, eps=EPS,
                               q_out=part[:, 0], k_out=part[:, 1])
            q, k, v = (qkv[:, i].transpose(0, 1).unsqueeze(0) for i in range(3))
            attn = F.scaled_dot_product_attention(q, k, v).squeeze(0).transpose(0, 1).reshape(cfg.tokens, d)
            for s, w in enumerate(block):
                _, n[s] = gated_residual_norm(x[rows[s]], w.out.forward(attn[rows[s]]), post="rms", post_weight=w.post_attn, gate=m[s, 2],
                                              pre="layer", scale=m[s, 4], shift=m[s, 3], eps=EPS, x_out=x[rows[s]], quantize=True)
                branch = w.down.forward(w.up.forward_fused(n[s], activation="gelu_tanh"))
                last = b + 1 == len(self.blocks)
                after = {} if last else dict(pre="layer", scale=mods[b + 1, s, 1], shift=mods[b + 1, s, 0], quantize=True)
                _, n[s] = gated_residual_norm(x[rows[s]], branch, post="rms", post_weight=w.post_ffn, gate=m[s, 5], eps=EPS,
                                              x_out=x[rows[s]], **(after or dict(pre=None, n_out=branch)))
        return x


def main() -> None:
    import argparse

    ap = argparse.ArgumentParser(description="Times one step of a random MXFP4 stack on the current GPU.")
    ap.add_argument("--blocks", type=int, default=4)
    ap.add_argument("--height", type=int, default=64)
    ap.add_argument("--width", type=int, default=64)
    ap.add_argument("--text", type=int, default=256)
    ap.add_argument("--steps", type=int, default=10)
    a = ap.parse_args()
    cfg = MxStackConfig(a.height, a.width, a.text, blocks=a.blocks)
    stack = MxStack.random(cfg)
    x = torch.randn((cfg.tokens, cfg.hidden), device="cuda").to(torch.bfloat16)
    temb = torch.randn((cfg.hidden,), device="cuda").to(torch.bfloat16)
    for _ in range(3):
        stack.forward(x, temb)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(a.steps):
        stack.forward(x, temb)
    end.record()
    torch.cuda.synchronize()
    print(f"{cfg.blocks} blocks, {cfg.tokens} tokens: {start.elapsed_time(end) / a.steps:.3f} ms a step")


if __name__ == "__main__":
    main()
