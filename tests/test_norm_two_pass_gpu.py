"""Group norm of maps that do not fit in a cluster's shared memory: two launches in each
direction, the rows streamed through a ring, partial sums of many blocks joined.

Shapes (with 148 SMs; V elements an access, forward 16-bit / gradient 16-bit / float32):
groups across vectors (8 / 4 / 4), four channels a group (8 / 4 / 4), whole vectors of 8 in
the gradient, V = 2 (66 channels), V = 1 (35), one group of everything, groups that span the
chunks of a row of more than 512 V channels, several pictures."""
import pytest

import test_ops_gpu as plain
from test_ops_gpu import E, ACTS, dtype_of, gen, least, norm64, norm_bound, ops, roundoff, torch, within  # noqa: F401

pytestmark = pytest.mark.gpu

SHAPES = [((2, 40001, 320), 32), ((1, 200003, 64), 16), ((2, 30011, 512), 32), ((1, 60001, 66), 3), ((1, 100001, 35), 5),
          ((3, 157, 163, 96), 1), ((1, 9001, 4104), 27), ((1, 3001, 4608), 4), ((1, 12007, 2184), 7)]
# A thread adds up to 130 rows of terms before the joins: 170 operations where the one-launch
# form's tests count 40, 200 where the gradient's count 64.
LONGER = 170 / 40
GRAD = 200


def inputs(torch, shape, dt, seed):  # noqa: F811
    g, c = gen(torch, seed), shape[-1]
    x = (torch.randn(shape, generator=g, device="cuda") * 2 + torch.randn(c, generator=g, device="cuda")).to(dt)
    w, b = (torch.randn(c, generator=g, device="cuda") for _ in range(2))
    dy = torch.randn(shape, generator=g, device="cuda").to(dt)
    return x, w, b, dy


def check_forward(torch, x, groups, w, b, act, got, mean=None, rstd=None, what=""):  # noqa: F811
    want, m64, r64, z = norm64(torch, x.double(), groups, w.double(), b.double(), 1e-5, act)
    bound = norm_bound(torch, x.double(), groups, w.double(), m64, r64, z, want, x.dtype)
    exact_part = roundoff(torch, x.dtype) * want.abs() + least(torch, x.dtype)
    within(got, want, (bound - exact_part) * LONGER + exact_part, what)
    if mean is not None:
        big = x.double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups).abs().amax((1, 3))
        within(mean, m64, 170 * E * big, "mean " + what)
        within(rstd, r64, 170 * E * r64 * (1 + (big * r64).square().clamp_max(64)), "rstd " + what)
    return m64, r64, z


def check_backward(torch, dy, x, groups, w, b, act, m64, r64, got, what=""):  # noqa: F811
    shape, n = x.shape, x.shape[0]
    wx, ww, wb = plain.norm_grad64(torch, dy.double(), x.double(), groups, w.double(), b.double(), act)
    per, m, r = (n, -1, groups, shape[-1] // groups), m64.reshape(n, 1, groups, 1), r64.reshape(n, 1, groups, 1)
    xe = ((x.double().reshape(per).abs() + m.abs()) * r).reshape(shape) * (4 * E)
    hat = ((x.double().reshape(per) - m) * r).reshape(shape).abs()
    gz, dims = dy.double().abs() * 1.13, tuple(range(len(shape) - 1))
    ge = gz * (xe * w.double().abs() + 16 * E)
    dx, dw, db = got
    within(dw, ww, (ge * hat + gz * xe + GRAD * E * gz * hat).sum(dims), "dweight " + what)
    within(db, wb, (ge + GRAD * E * gz).sum(dims), "dbias " + what)
    h, he = gz * w.double().abs(), ge * w.double().abs()
    m1 = (he + GRAD * E * h).reshape(per).mean((1, 3), keepdim=True)
    m2 = (he * hat + h * xe + GRAD * E * h * hat).reshape(per).mean((1, 3), keepdim=True)
    s2 = (h * hat).reshape(per).mean((1, 3), keepdim=True)
    bound = (he + 16 * E * h).reshape(per) + m1 + hat.reshape(per) * m2 + (xe + 16 * E * hat).reshape(per) * s2
    bound = ((bound + 16 * E * h.reshape(per).mean((1, 3), keepdim=True)) * r).reshape(shape)
    within(dx, wx, bound + roundoff(torch, x.dtype) * wx.abs() + least(torch, x.dtype), "dx " + what)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_two_pass(torch, ops, shape, groups, dtype, act):  # noqa: F811
    dt = dtype_of(torch, dtype)
    x, w, b, dy = inputs(torch, shape, dt, shape[-1] + len(act))
    y, mean, rstd = ops.group_norm(x, groups, w, b, act=act, stats=True)
    assert y.dtype == dt and y.shape == x.shape
    m64, r64, z = check_forward(torch, x, groups, w, b, act, y, mean, rstd, f"{shape} {act}")
    if act == "relu":  # where z is 0 to rounding, the slope may be either side's
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    del z, y
    got = ops.group_norm_backward(dy, x, m64.float(), r64.float(), groups, w, b, act=act)
    check_backward(torch, dy, x, groups, w, b, act, m64, r64, got, f"{shape} {act}")


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_two_pass_in_place(torch, ops, dtype):  # noqa: F811
    x, w, b, dy = inputs(torch, (2, 40001, 320), dtype_of(torch, dtype), 71)
    y, mean, rstd = ops.group_norm(x, 32, w, b, act="gelu", stats=True)
    want = ops.group_norm_backward(dy, x, mean, rstd, 32, w, b, act="gelu")
    over = x.clone()
    assert ops.group_norm(over, 32, w, b, act="gelu", out=over) is over and torch.equal(over, y)
    for into in ("dy", "x"):
        a, e = x.clone(), dy.clone()
        got = ops.group_norm_backward(e, a, mean, rstd, 32, w, b, act="gelu", out=e if into == "dy" else a)
        assert got[0] is (e if into == "dy" else a) and all(torch.equal(p, q) for p, q in zip(got, want))


def test_two_pass_views(torch, ops):  # noqa: F811
    """Channels of wider maps, aligned and not, and pictures apart, into views."""
    g = gen(torch, 72)
    wide = torch.randn((2, 150001, 80), generator=g, device="cuda").half()
    w, b = (torch.randn(64, generator=g, device="cuda") for _ in range(2))
    for first in (8, 2, 3):
        x, dy = wide[..., first:first + 64], wide.flip(1)[..., first + 1:first + 65]
        out = torch.zeros_like(wide)
        y, mean, rstd = ops.group_norm(x, 8, w, b, act="silu", stats=True, out=out[..., 5:69])
        m64, r64, _ = check_forward(torch, x, 8, w, b, "silu", y, mean, rstd, f"from {first}")
        assert not out[..., :5].any() and not out[..., 69:].any()
        got = ops.group_norm_backward(dy, x, m64.float(), r64.float(), 8, w, b, act="silu", out=out[..., 8:72])
        check_backward(torch, dy, x, 8, w, b, "silu", m64, r64, got, f"from {first}")
    one = torch.randn((1, 150001, 64), generator=g, device="cuda").expand(3, -1, -1)  # a picture repeated
    check_forward(torch, one, 8, w, b, "none", ops.group_norm(one, 8, w, b))


def test_two_pass_large_mean_and_outlier(torch, ops):  # noqa: F811
    """The mean a thousand times the spread, and one value a million spreads away: the shifted
    sums keep rstd to the few operations of its partial sums."""
    g = gen(torch, 73)
    one, none = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    for mean in (1e3, -3e4):
        x = torch.randn((1, 200003, 64), generator=g, device="cuda") + mean
        y, m, r = ops.group_norm(x, 4, stats=True)
        check_forward(torch, x, 4, one, none, "none", y, what=f"mean {mean}")
        _, _, r64, _ = norm64(torch, x.double(), 4, one.double(), 0.0, 1e-5, "none")
        within(r, r64, 170 * E * r64, f"rstd, mean {mean}")
    for at in (0, 100001, 200002, 77):
        x = torch.randn((1, 200003, 64), generator=g, device="cuda")
        x[0, at, 5] = 1e6
        _, _, r = ops.group_norm(x, 4, stats=True)
        _, _, r64, _ = norm64(torch, x.double(), 4, one.double(), 0.0, 1e-5, "none")
        within(r, r64, 170 * E * r64, f"rstd, outlier at {at}")


def test_two_pass_nan_and_infinity_stay_in_their_group(torch, ops):  # noqa: F811
    x = torch.randn((2, 60001, 320), generator=gen(torch, 74), device="cuda").half()
    x[0, 59999, 3], x[1, 0, 319] = float("nan"), float("inf")
    bad = ~torch.isfinite(ops.group_norm(x, 32, act="silu"))
    assert bad[0, :, :10].all() and bad[1, :, 310:].all()
    bad[0, :, :10] = False
    bad[1, :, 310:] = False
    assert not bad.any()


def test_two_pass_repeats_and_replays(torch, ops):  # noqa: F811
    x, w, b, dy = inputs(torch, (2, 40001, 320), torch.bfloat16, 75)

    def both():
        y, mean, rstd = ops.group_norm(x, 32, w, b, act="silu", stats=True)
        return (y, mean, rstd, *ops.group_norm_backward(dy, x, mean, rstd, 32, w, b, act="silu"))

    first = both()
    for _ in range(5):
        assert all(torch.equal(p, q) for p, q in zip(first, both()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    x.mul_(0.5)
    dy.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(held, both()))
