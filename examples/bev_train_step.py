"""A small bird's-eye-view training step that runs the library's operators together.

Camera features pass a deformable convolution and a group norm with SiLU; a
grid of queries, looked up with learned row and column positions, samples them
with deformable attention; a group norm with ReLU and a 1x1 convolution give a
map.  After the backward pass the gradients are clipped to a global norm and
the weights take a step.  Everything stays channels-last, and after the first
step nothing in a step waits for the device.

    python examples/bev_train_step.py [--steps 20] [--dtype bf16]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "bev-kernels_b200"))

from grad_clip import clip_grad_norm_                            # noqa: E402
from group_norm_act import GroupNormAct                          # noqa: E402
from modulated_deform_conv import ModulatedDeformConv2dPack      # noqa: E402
from ms_deform_attn import multi_scale_deformable_attn           # noqa: E402
from scaled_embedding import ScaledEmbedding                     # noqa: E402


class BevHead(nn.Module):
    """Image features [cameras, C, h, w] -> a map [classes, rows, cols]."""

    def __init__(self, channels: int, rows: int, cols: int, classes: int, heads: int = 8,
                 points: int = 4):
        super().__init__()
        self.rows, self.cols, self.heads, self.points = rows, cols, heads, points
        self.conv = ModulatedDeformConv2dPack(channels, channels, 3, padding=1)
        self.norm = GroupNormAct(32, channels, act="silu")
        self.row_pos = ScaledEmbedding(rows, channels // 2)
        self.col_pos = ScaledEmbedding(cols, channels // 2)
        self.offsets = nn.Linear(channels, heads * points * 2)
        self.weights = nn.Linear(channels, heads * points)
        self.out_norm = GroupNormAct(32, channels, act="relu")
        self.out = nn.Conv2d(channels, classes, 1)
        r, c = torch.meshgrid(torch.arange(rows), torch.arange(cols), indexing="ij")
        self.register_buffer("row_ids", r.reshape(-1))
        self.register_buffer("col_ids", c.reshape(-1))
        self._levels = {}  # (h, w, device): a copy from the host would wait in every step

    def levels(self, h: int, w: int, device):
        """The attention's shapes and level starts of one [h, w] level."""
        key = (h, w, device)
        if key not in self._levels:
            self._levels[key] = (torch.tensor([[h, w]], device=device),
                                 torch.zeros(1, dtype=torch.int64, device=device))
        return self._levels[key]

    def forward(self, feats: torch.Tensor) -> torch.Tensor:
        n, c, h, w = feats.shape
        x = self.norm(self.conv(feats))                                       # [n, C, h, w]
        value = x.permute(0, 2, 3, 1).reshape(n, h * w, self.heads, c // self.heads)
        query = torch.cat([self.row_pos(self.row_ids), self.col_pos(self.col_ids)], -1)
        q, k = query.shape[0], self.heads * self.points
        centre = torch.stack([(self.col_ids + 0.5) / self.cols, (self.row_ids + 0.5) / self.rows], -1)
        loc = centre.view(q, 1, 1, 1, 2).to(query.dtype) + 0.1 * torch.tanh(
            self.offsets(query)).view(q, self.heads, 1, self.points, 2)
        att = self.weights(query).view(q, self.heads, self.points).softmax(-1).view(
            q, self.heads, 1, self.points)
        shapes, start = self.levels(h, w, feats.device)
        seen = multi_scale_deformable_attn(
            value.contiguous(), shapes, start, loc.expand(n, q, self.heads, 1, self.points, 2).contiguous(),
            att.expand(n, q, self.heads, 1, self.points).contiguous(), 64)
        bev = (query + seen.mean(0)).view(1, self.rows, self.cols, c).permute(0, 3, 1, 2)
        return self.out(self.out_norm(bev))[0]


def train(steps: int, dtype: torch.dtype, cameras: int = 2, channels: int = 256, size=(29, 50),
          bev=(48, 40), classes: int = 4, max_norm: float = 1.0, lr: float = 0.05):
    """Fits a fixed random map; -> (losses, gradient norms) of the steps."""
    dev = torch.device("cuda")
    torch.manual_seed(0)
    model = BevHead(channels, *bev, classes).to(dev, dtype)
    # the norms' parameters stay fp32
    for m in (model.norm, model.out_norm):
        m.float()
    feats = torch.randn(cameras, channels, *size, device=dev).to(
        dtype, memory_format=torch.channels_last)
    target = torch.randint(0, classes, bev, device=dev)
    opt = torch.optim.SGD(model.parameters(), lr=lr, momentum=0.9)
    losses, norms = [], []
    for _ in range(steps):
        loss = nn.functional.cross_entropy(model(feats).float()[None], target[None])
        opt.zero_grad(set_to_none=True)
        loss.backward()
        norms.append(clip_grad_norm_(model.parameters(), max_norm))
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist(), torch.stack(norms).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--dtype", choices=("f32", "bf16", "f16"), default="bf16")
    a = ap.parse_args()
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[a.dtype]
    for i, (loss, norm) in enumerate(zip(*train(a.steps, dtype))):
        print(f"step {i:3d}  loss {loss:.4f}  gradient norm {norm:.3f}")


if __name__ == "__main__":
    main()
