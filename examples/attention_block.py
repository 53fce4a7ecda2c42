"""An image or clip transformer block on the package's block operators.

    python examples/attention_block.py [--frames 4] [--height 34] [--width 60] [--channels 512]

What a denoiser with global attention runs at the bottom of its U-Net, channels last:

    y = x + proj(attention(rotate(q), rotate(k), v)),  q, k, v = linear(group_norm(x))
    z = y + linear(group_norm(y) with SiLU)
    s = attention of one learned query over all cells of z       (a summary of the clip)

Queries and keys turn with their cell's frame, row and column; cells that only pad a frame to
the batch's size are hidden by the key mask. The linear maps are plain matrix products.
"""
import argparse
import importlib
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
scb = importlib.import_module("scunet-rs_b200")
ops = scb.ops


class AttentionBlock:
    """Seeded weights of one block: `c` channels, heads of `d` channels, three position axes."""

    def __init__(self, c, d=64, groups=32, theta=100.0, seed=0, dtype=torch.float16, device="cuda"):
        g = torch.Generator().manual_seed(seed)

        def weight(*shape):
            return (torch.randn(shape, generator=g) * shape[-1] ** -0.5).to(dtype).to(device)

        self.heads, self.d, self.groups = c // d, d, groups
        self.qkv, self.proj, self.linear = weight(3 * c, c), weight(c, c), weight(c, c)
        self.query = weight(self.heads, d)
        self.norms = [(1 + 0.1 * torch.randn(c, generator=g).to(device), 0.1 * torch.randn(c, generator=g).to(device))
                      for _ in range(2)]
        pairs = d // 2
        self.sections = (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)  # frame, row, column
        self.inv_freq = torch.cat([theta ** (-torch.arange(m) / m) for m in self.sections]).float().to(device)

    def positions(self, t, h, w):
        """[t h w, 3] cells of a clip: frame, row, column."""
        axes = [torch.arange(n, device=self.inv_freq.device, dtype=torch.int32) for n in (t, h, w)]
        return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).view(-1, 3)

    def __call__(self, x, key_mask=None):
        """x [clips, frames, height, width, c] -> (the same shape, summary [clips, c])."""
        n, t, h, w, c = x.shape
        cells = t * h * w
        y = ops.group_norm(x, self.groups, *self.norms[0])
        q, k, v = (y @ self.qkv.t()).view(n, cells, 3, self.heads, self.d).unbind(2)
        pos = self.positions(t, h, w)
        q, k = ops.rotate_axes(q, k, pos, self.inv_freq, self.sections, layout="axial")
        a = ops.attention(q, k, v, key_mask=key_mask)
        y = x + (a.view(n, cells, c) @ self.proj.t()).view(x.shape)
        z = y + ops.group_norm(y, self.groups, *self.norms[1], act="silu") @ self.linear.t()
        z_heads = z.view(n, cells, self.heads, self.d)
        one = self.query.expand(n, 1, self.heads, self.d)
        return z, ops.attention(one, z_heads, z_heads, key_mask=key_mask).view(n, c)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("clips", 1), ("frames", 4), ("height", 34), ("width", 60), ("channels", 512), ("steps", 20)):
        ap.add_argument(f"--{name}", type=int, default=default)
    a = ap.parse_args()
    block = AttentionBlock(a.channels)
    x = torch.randn((a.clips, a.frames, a.height, a.width, a.channels), device="cuda").half()
    # the last eighth of every row is padding
    seen = torch.ones((a.clips, a.frames, a.height, a.width), dtype=torch.bool, device="cuda")
    seen[..., a.width - a.width // 8:] = False
    seen = seen.view(a.clips, -1)
    for _ in range(3):
        z, s = block(x, seen)
    ops.status()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(a.steps):
        z, s = block(x, seen)
    end.record()
    ops.status()
    print(f"{tuple(x.shape)} {x.dtype}: {start.elapsed_time(end) / a.steps:.3f} ms a block, "
          f"|z| {z.float().abs().mean():.4f}, |s| {s.float().abs().mean():.4f}")


if __name__ == "__main__":
    main()
