"""Fine-tuning around frozen 8-bit linears: a small diffusion-transformer block over video tokens whose projections are
``Int8Linear`` (frozen, 8-bit weights), with the modulations, the norms of the queries and keys and a final head left
trainable.  It runs the 8-bit and training operators of ``convrot_mlx_b200`` together as a training step uses them:

  modulated_layer_norm -> int8 qkv -> layer_norm of q and k -> axial_rotary -> attention -> int8 projection
  modulated_layer_norm -> int8 -> gelu_tanh_saved8 -> int8

    python dit_finetune.py [--steps 20] [--width 768] [--frames 4 --rows 16 --cols 16] [--batch 2]

prints the loss of each step.  Inputs and targets are synthetic; the block learns a fixed random target.
"""

from __future__ import annotations

import argparse

import torch
import torch.nn.functional as F
from torch import nn

import convrot_mlx_b200 as cr
from convrot_mlx_b200.adapter import replace_int8_linears


class Norm(nn.Module):
    """Affine layer norm of each head's vector."""

    def __init__(self, width: int):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width))

    def forward(self, x):
        return cr.layer_norm(x, self.weight, self.bias)


class Block(nn.Module):
    """Attention and MLP of one token stream with adaptive norms; head dimension split over time, height and width."""

    def __init__(self, width: int, heads: int, axes=(16, 24, 24)):
        super().__init__()
        self.heads, self.axes = heads, axes
        self.modulation = nn.Linear(width, 6 * width)
        self.qkv = nn.Linear(width, 3 * width)
        self.q_norm, self.k_norm = Norm(width // heads), Norm(width // heads)
        self.proj = nn.Linear(width, width)
        self.up, self.down = nn.Linear(width, 4 * width), nn.Linear(4 * width, width)

    def forward(self, x, vec, positions):
        shift1, scale1, gate1, shift2, scale2, gate2 = self.modulation(F.silu(vec)).unsqueeze(1).chunk(6, dim=-1)
        qkv = self.qkv(cr.modulated_layer_norm(x, shift1, scale1))
        q, k, v = qkv.unflatten(-1, (3, self.heads, -1)).unbind(2)
        q, k = self.q_norm(q).transpose(1, 2), self.k_norm(k).transpose(1, 2)
        q, k = cr.axial_rotary(q, k, positions, self.axes)
        a = F.scaled_dot_product_attention(q, k, v.transpose(1, 2)).transpose(1, 2).flatten(2)
        x = x + gate1 * self.proj(a)
        h = cr.gelu_tanh_saved8(self.up(cr.modulated_layer_norm(x, shift2, scale2)))
        return x + gate2 * self.down(h)


FROZEN = ("qkv", "proj", "up", "down")


def build(width: int, heads: int, device, dtype=torch.bfloat16, seed: int = 0) -> Block:
    """A block with its projections frozen in 8 bits; the rest trainable."""

    torch.manual_seed(seed)
    block = Block(width, heads).to(device)
    keep = [name for name, m in block.named_modules() if isinstance(m, nn.Linear) and name not in FROZEN]
    replace_int8_linears(block, keep=keep)
    return block.to(dtype)


def grid_positions(frames: int, rows: int, cols: int, device) -> torch.Tensor:
    """(tokens, 3) positions along time, height and width."""

    return torch.cartesian_prod(*(torch.arange(n, device=device) for n in (frames, rows, cols))).float()


def train(steps: int, width: int, heads: int, batch: int, frames: int, rows: int, cols: int, device="cuda",
          lr: float = 2e-3, seed: int = 0) -> list[float]:
    """Adam steps on the trainable parameters; returns the losses."""

    block = build(width, heads, device, seed=seed)
    g = torch.Generator(device=device).manual_seed(seed + 1)
    positions = grid_positions(frames, rows, cols, device)
    shape = (batch, positions.shape[0], width)
    x = torch.randn(shape, generator=g, device=device).bfloat16()
    vec = torch.randn((batch, width), generator=g, device=device).bfloat16()
    target = x + 0.5 * torch.randn((batch, 1, width), generator=g, device=device).bfloat16()
    optimizer = torch.optim.Adam(block.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        loss = F.mse_loss(block(x, vec, positions).float(), target.float())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return [float(v) for v in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--width", type=int, default=768)
    ap.add_argument("--heads", type=int, default=12)
    ap.add_argument("--batch", type=int, default=2)
    ap.add_argument("--frames", type=int, default=4)
    ap.add_argument("--rows", type=int, default=16)
    ap.add_argument("--cols", type=int, default=16)
    a = ap.parse_args()
    for i, loss in enumerate(train(a.steps, a.width, a.heads, a.batch, a.frames, a.rows, a.cols)):
        print(f"step {i}: loss {loss:.5f}")


if __name__ == "__main__":
    main()
