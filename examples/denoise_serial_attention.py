"""Denoising point clouds with serialised attention: the operators of
``mps_pointops.attention`` together, in training and over cached keys.

A ragged batch of noisy spheres is ordered along the Z curve of its grid
coordinates; one attention block (norms and rotation of queries and keys,
sliding window along the curve, a few summary rows at the head of each cloud
that all points see, a learned table of relative grid positions) predicts
offsets, trained with the Chamfer distance to the clean clouds.  Then new points
of each cloud attend to the cached keys of the rest, one chunk and one point at
a time, and give the rows that the whole cloud gives under the same mask.

    python examples/denoise_serial_attention.py [--steps 30]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import Tensor, nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "mps-pointops_b200"))

from mps_pointops import attention, chamfer_distance  # noqa: E402


def z_order(grid: Tensor) -> Tensor:
    """Order of (N, 3) grid coordinates in [0, 1024) along the Z curve."""
    code = torch.zeros(len(grid), dtype=torch.int64, device=grid.device)
    for bit in range(10):
        for axis in range(3):
            code |= ((grid[:, axis] >> bit) & 1) << (3 * bit + axis)
    return code.argsort()


class SerialBlock(nn.Module):
    """Attention of rows (N, C) of a ragged batch along their order."""

    def __init__(self, channels: int, heads: int, reach: int, window: int, sinks: int):
        super().__init__()
        self.heads, self.dim = heads, channels // heads
        self.window, self.sinks = (window, window), sinks
        self.qkv = nn.Linear(channels, 3 * channels)
        self.out = nn.Linear(channels, channels)
        self.q_norm = nn.Parameter(torch.ones(self.dim))
        self.k_norm = nn.Parameter(torch.ones(self.dim))
        self.table = nn.Parameter(torch.zeros(3, 2 * reach + 1, heads))
        pairs = self.dim // 2
        freqs = torch.zeros(3, pairs)
        for p in range(pairs):  # the axes take turns, each with falling frequencies
            freqs[p % 3, p] = 100.0 ** (-(p // 3) / max(1, pairs // 3))
        self.register_buffer("freqs", freqs)

    def project(self, x: Tensor, grid: Tensor, dtype: torch.dtype):
        qkv = self.qkv(x).view(len(x), 3 * self.heads, self.dim).to(dtype)
        q, k, v = qkv.split(self.heads, dim=1)  # views of one projection
        q, k = attention.norm_rotate(q, k, grid, self.freqs, q_weight=self.q_norm,
                                     k_weight=self.k_norm)
        return q, k, v

    def forward(self, x: Tensor, grid: Tensor, segments: attention.Segments,
                dtype: torch.dtype = torch.bfloat16) -> Tensor:
        q, k, v = self.project(x, grid, dtype)
        y = attention.window_attention(q, k, v, segments, window=self.window, sinks=self.sinks,
                                       bias_table=self.table, position=grid)
        return x + self.out(y.reshape(len(x), -1).to(x.dtype))


def make_batch(sizes: list[int], device: torch.device, seed: int):
    """Clean and noisy points, grid coordinates and offsets, each cloud in curve order."""
    g = torch.Generator().manual_seed(seed)
    clean, noisy, grids = [], [], []
    for n in sizes:
        p = torch.randn(n, 3, generator=g)
        p = (p / p.norm(dim=1, keepdim=True)).to(device)
        q = p + 0.1 * torch.randn(n, 3, generator=g).to(device)
        grid = ((q + 2) * 32).clamp(0, 1023).to(torch.int32)
        order = z_order(grid.long())
        clean.append(p[order])
        noisy.append(q[order])
        grids.append(grid[order])
    offset = torch.tensor(sizes, device=device).cumsum(0)
    return clean, torch.cat(noisy), torch.cat(grids), offset


def train(steps: int, device: torch.device, sizes: list[int] = [700, 1024, 333]) -> list[float]:
    torch.manual_seed(0)
    clean, noisy, grid, offset = make_batch(sizes, device, 1)
    segments = attention.Segments(offset)  # once for the batch, whatever the layers
    embed, head = nn.Linear(3, 64).to(device), nn.Linear(64, 3).to(device)
    block = SerialBlock(64, heads=4, reach=15, window=64, sinks=2).to(device)
    params = [*embed.parameters(), *block.parameters(), *head.parameters()]
    optimizer = torch.optim.AdamW(params, lr=3e-3)
    losses = []
    longest = max(sizes)
    lengths = torch.tensor(sizes, device=device)
    target = torch.zeros(len(sizes), longest, 3, device=device)
    for b, p in enumerate(clean):
        target[b, :len(p)] = p
    for _ in range(steps):
        moved = noisy + head(block(embed(noisy), grid, segments))
        padded = torch.stack([nn.functional.pad(p, (0, 0, 0, longest - len(p)))
                              for p in moved.split(sizes)])
        loss, _ = chamfer_distance(padded, target, x_lengths=lengths, y_lengths=lengths)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


@torch.no_grad()
def cached_rows(device: torch.device, sizes: list[int] = [700, 1024, 333], chunk: int = 40) -> float:
    """Largest difference between the last rows of each cloud formed with the whole
    cloud (causal) and those formed over cached keys: a chunk, then a single row."""
    torch.manual_seed(0)
    _, noisy, grid, offset = make_batch(sizes, device, 2)
    block = SerialBlock(64, heads=4, reach=15, window=200, sinks=2).to(device)
    nn.init.normal_(block.table, std=0.5)
    q, k, v = block.project(nn.Linear(3, 64).to(device)(noisy), grid, torch.bfloat16)
    opts = dict(window=(200, 0), sinks=2, causal=True, bias_table=block.table)
    whole = attention.window_attention(q, k, v, attention.Segments(offset), position=grid, **opts)
    worst = 0.0
    ends = offset.tolist()
    for new in (chunk, 1):
        last = torch.cat([torch.arange(e - new, e) for e in ends]).to(device)
        rows = torch.arange(new, new * len(ends) + 1, new, device=device)
        part = attention.window_attention(
            q[last].contiguous(), k, v, attention.Segments(rows, offset), position=grid[last],
            key_position=grid, **opts)
        worst = max(worst, (part.float() - whole[last].float()).abs().max().item())
    return worst


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=30)
    args = parser.parse_args()
    cuda = torch.device("cuda")
    curve = train(args.steps, cuda)
    print(f"Chamfer distance: {curve[0]:.5f} -> {curve[-1]:.5f} in {args.steps} steps")
    print(f"cached rows against whole clouds: {cached_rows(cuda):.2e}")
