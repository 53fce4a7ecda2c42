"""Many keys of faint weight beside a few strong ones."""
import math

import pytest

from test_ops_gpu import attention64, ops, torch  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("lq,heads", [(1, 1), (200, 1), (130, 148), (1, 1200)])  # cut into pieces; whole units
@pytest.mark.parametrize("bits", [22, 26, 29])
def test_faint_tail(torch, ops, dtype, lq, heads, bits):  # noqa: F811
    """One key of weight 1 and value 0, a tail of weights about 2^-bits and values about 1, whose
    sum is the result. A weight is rounded to 16 bits, relatively (u) or, in fp16, to the nearest
    of its subnormal numbers, which lie no further than 2^-31 of the row's largest weight apart:
    u of the sum and 2^-32 a key, beside the rounding of the result and of float32 sums."""
    dt, lk, d = getattr(torch, dtype), 30000, 32
    g = torch.Generator(device="cuda").manual_seed(bits)
    q = torch.zeros((1, lq, heads, d), device="cuda").to(dt)
    k = torch.zeros((1, lk, 1, d), device="cuda").to(dt)
    q[..., 0] = q[..., 1] = 1.0
    k[..., 0] = -bits * math.log(2)
    k[..., 1] = 0.2 * torch.randn((1, lk, 1), generator=g, device="cuda").to(dt)
    v = (1 + 0.1 * torch.randn((1, lk, 1, d), generator=g, device="cuda")).to(dt)
    k[:, 7], v[:, 7] = 0.0, 0.0
    out = ops.attention(q, k.expand(-1, -1, heads, -1), v.expand(-1, -1, heads, -1), scale=1.0)
    want, size, _ = attention64(torch, q[:, :1, :1], k, v, 1.0, None)
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dt]
    # float32: scores of size `bits`, and chains of at most a few hundred sums
    bound = (3 * u + (4 * bits + 300) * 2.0 ** -24) * size + lk * 2.0 ** -32 * float(v.abs().max())
    bound = bound + (2.0 ** -25 if dt == torch.float16 else 0)  # the result's own subnormal rounding
    off = (out.double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
