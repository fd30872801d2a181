"""Trains a small network of morphological layers and channel mixers on synthetic images, and says what its
forward keeps for the backward.

    python examples/train_mixer.py [--steps 60] [--size 64] [--batch 4] [--channels 32] [--dtype bfloat16]
                                   [--attend 4]

The task: the morphological gradient (the range of each pixel's 3x3 neighbourhood) of an image, from the
image with bright specks and dark holes in it, which an opening and a closing remove. A dilation lifts the
image to `channels` maps; blocks of a per-channel opening or closing (kept by its input in 8 bits,
nn.Checkpoint8) and a gated channel mixer (nn.ChannelMixer: norm with the residual, two linear layers and the
gated activation, kept in 8 bits) follow; a linear layer reads the answer out. With --attend N each block also mixes
its pixels with those before them by N heads of linear attention (nn.TokenMixer). Needs a HIP device.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))  # the package in place, not installed

import morphocore_amd.functional as F
from morphocore_amd.nn import ChannelMixer, Checkpoint8, Closing, Dilation, Opening, RMSNorm, TokenMixer


class Net(nn.Module):
    def __init__(self, channels: int, blocks: int, dtype: torch.dtype, attend: int = 0):
        super().__init__()
        self.lift = Dilation(1, channels, 3, "sum", dtype=dtype)
        self.morph = nn.ModuleList(Checkpoint8((Opening, Closing)[i % 2](channels, channels, 3, dtype=dtype)) for i in range(blocks))
        self.mix = nn.ModuleList(ChannelMixer(channels, 2 * channels, dtype=dtype) for _ in range(blocks))
        self.attend = nn.ModuleList(TokenMixer(channels, attend, axes=2, dtype=dtype) for _ in range(blocks if attend else 0))
        self.norm = RMSNorm(channels, dtype=dtype)
        self.read = nn.Parameter(torch.zeros(1, channels, dtype=dtype))
        with torch.no_grad():
            for p in (self.lift.weight, *(w for m in self.morph for w in m.parameters())):
                p.add_(0.1 * torch.randn(p.shape, dtype=dtype))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = self.lift(x)
        out = None
        for i, (morph, mix) in enumerate(zip(self.morph, self.mix)):
            y = morph(h).permute(0, 2, 3, 1)  # channels last, as the mixer reads them
            out, last = mix(y, h.permute(0, 2, 3, 1))
            if self.attend:
                out, last = self.attend[i](out, last)
            h = (out + last).permute(0, 3, 1, 2).contiguous()
        y = self.norm(h.permute(0, 2, 3, 1))
        return F.linear8(y, self.read).permute(0, 3, 1, 2)


def images(batch: int, size: int, seed: int, device):
    """Smooth random images with one pixel in fifteen set to white or black, and the gradient of the clean ones."""
    g = torch.Generator().manual_seed(seed)
    clean = torch.nn.functional.interpolate(torch.rand(batch, 1, size // 8, size // 8, generator=g), size=(size, size), mode="bicubic").clamp(0, 1)
    speck = torch.rand(clean.shape, generator=g)
    noisy = torch.where(speck < 1 / 30, 0.0, torch.where(speck > 29 / 30, 1.0, clean))
    padded = torch.nn.functional.pad(clean, (1, 1, 1, 1), mode="replicate")
    pool = torch.nn.functional.max_pool2d
    return noisy.to(device), (pool(padded, 3, 1) + pool(-padded, 3, 1)).to(device)


def train(steps: int = 60, size: int = 64, batch: int = 4, channels: int = 32, blocks: int = 2, dtype: torch.dtype = torch.bfloat16,
          lr: float = 3e-3, seed: int = 0, attend: int = 0):
    """Returns the losses of the steps and the bytes that a forward keeps."""
    device = torch.device("cuda")
    torch.manual_seed(seed)
    net = Net(channels, blocks, dtype, attend).to(device)
    opt = torch.optim.Adam(net.parameters(), lr=lr, eps=1e-6)
    losses, kept = [], 0
    for step in range(steps):
        noisy, wanted = images(batch, size, seed + step, device)
        before = torch.cuda.memory_allocated(device)
        loss = (net(noisy.to(dtype)).float() - wanted).square().mean()
        kept = torch.cuda.memory_allocated(device) - before
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses, kept


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--size", type=int, default=64)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--channels", type=int, default=32)
    ap.add_argument("--dtype", choices=["float32", "float16", "bfloat16"], default="bfloat16")
    ap.add_argument("--attend", type=int, default=0)
    a = ap.parse_args()
    losses, kept = train(a.steps, a.size, a.batch, a.channels, dtype=getattr(torch, a.dtype), attend=a.attend)
    values = a.batch * a.channels * a.size * a.size
    for i in range(0, a.steps, max(1, a.steps // 6)):
        print(f"step {i:4d}  loss {losses[i]:.5f}")
    print(f"last loss {losses[-1]:.5f}; a forward keeps {kept / 1e6:.2f} MB, {kept / values:.1f} bytes a pixel and channel")


if __name__ == "__main__":
    main()
