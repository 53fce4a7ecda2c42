"""The example block (examples/attention_block.py) against the same block in 64 bits."""
import importlib.util

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def plain(torch, block, x, seen):
    """The block's formulas in 64 bits on the same weights."""
    x = x.double()
    n, t, h, w, c = x.shape
    cells = t * h * w

    def norm(v, wb):
        per = v.reshape(n, cells, block.groups, -1)
        mean = per.mean((1, 3), keepdim=True)
        var = (per - mean).square().mean((1, 3), keepdim=True)
        return ((per - mean) / torch.sqrt(var + 1e-5)).reshape(v.shape) * wb[0].double() + wb[1].double()

    def attend(q, k, v):
        s = torch.einsum("nqhd,nkhd->nhqk", q, k) * block.d ** -0.5
        s = s.masked_fill(~seen[:, None, None, :], -torch.inf)
        return torch.einsum("nhqk,nkhd->nqhd", torch.softmax(s, 3), v)

    qkv = norm(x, block.norms[0]) @ block.qkv.double().t()
    q, k, v = qkv.view(n, cells, 3, block.heads, block.d).unbind(2)
    pos, out, at = block.positions(t, h, w).double(), [], 0
    for a, m in enumerate(block.sections):
        out.append(pos[:, a, None] * block.inv_freq[at:at + m].double())
        at += m

    def turn(u):
        parts, first = [], 0
        for m, angle in zip(block.sections, out):
            lo, hi = u[..., first:first + m], u[..., first + m:first + 2 * m]
            cos, sin = angle.cos()[None, :, None], angle.sin()[None, :, None]
            parts += [lo * cos - hi * sin, lo * sin + hi * cos]
            first += 2 * m
        return torch.cat([*parts, u[..., first:]], -1)

    a = attend(turn(q), turn(k), v).reshape(n, cells, c)
    y = x + (a @ block.proj.double().t()).view(x.shape)
    u = norm(y, block.norms[1])
    z = y + (u * torch.sigmoid(u)) @ block.linear.double().t()
    zh = z.view(n, cells, block.heads, block.d)
    s = attend(block.query.double().expand(n, 1, block.heads, block.d), zh, zh)
    return z, s.reshape(n, c)


@pytest.mark.parametrize("n,t,h,w,c,d", [(1, 1, 8, 8, 128, 32), (2, 3, 7, 13, 256, 64), (1, 2, 17, 30, 512, 128)])
def test_block(n, t, h, w, c, d):
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location("attention_block", ROOT / "examples" / "attention_block.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    block = example.AttentionBlock(c, d=d, seed=c)
    g = torch.Generator(device="cuda").manual_seed(h * w)
    x = torch.randn((n, t, h, w, c), generator=g, device="cuda").half()
    seen = torch.rand((n, t * h * w), generator=g, device="cuda") < 0.8
    z, s = block(x, seen)
    example.ops.status()
    want_z, want_s = plain(torch, block, x, seen)
    # fp16 storage between the steps: about ten roundings of 2^-11 of values up to a few units,
    # through products of unit gain, sqrt(10) of them in quadrature with a margin of 3
    for got, want in ((z, want_z), (s, want_s)):
        rel = float((got.double() - want).norm() / want.norm())
        assert rel < 3 * 10 ** 0.5 * 2.0 ** -11, rel
