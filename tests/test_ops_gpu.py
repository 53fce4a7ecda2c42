"""The block operators against plain 64-bit implementations of their formulas, through the
package's public calls.

Tolerances are bounds, not fits. With u the output type's unit roundoff (2^-24, 2^-11,
2^-8) and e = 2^-24: a float32 chain of k operations on terms of size T is off by at most
about k e T, and the result is rounded once, u |result|. Each test states its T and k.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
ACTS = ["none", "relu", "gelu", "silu"]


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.fixture(scope="module")
def ops(scb, torch):
    return scb.ops


def dtype_of(torch, name):
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def roundoff(torch, dt):
    return {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dt]


def least(torch, dt):
    """Half the spacing of the type's subnormal numbers: what rounding may lose near zero."""
    return {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dt]


def within(got, want, bound, what=""):
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst ratio to the bound "
                           f"{float((d / bound).nan_to_num(1e9).max()):.3g}")


def gen(torch, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------- group norm
def act64(torch, z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def norm64(torch, x, groups, w, b, eps, act):
    n, c = x.shape[0], x.shape[-1]
    per = x.reshape(n, -1, groups, c // groups)
    mean = per.mean((1, 3), keepdim=True)
    var = (per - mean).square().mean((1, 3), keepdim=True)
    hat = ((per - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    z = hat * w + b
    return act64(torch, z, act), mean.reshape(n, groups), torch.sqrt(var + eps).reciprocal().reshape(n, groups), z


def norm_bound(torch, x, groups, w, mean, rstd, z, want, dt):
    """Terms: rstd |w| (|x| + |mean|) and |z|; about 40 operations (partial sums of a thread,
    joins, scale, activation whose slope is below 1.13 and whose own error is a few e)."""
    n, c = x.shape[0], x.shape[-1]
    spread = ((x.reshape(n, -1, groups, c // groups).abs() + mean.abs().reshape(n, 1, groups, 1))
              * rstd.reshape(n, 1, groups, 1)).reshape(x.shape) * w.abs()
    return 40 * E * (spread + z.abs() + 1) + roundoff(torch, dt) * want.abs() + least(torch, dt)


NORM_SHAPES = [  # shape, groups
    ((1, 1, 1), 1), ((1, 1, 8), 8), ((2, 3, 6), 3), ((3, 7, 5, 40), 4), ((1, 64, 512), 32), ((2, 33, 47, 96), 8),
    ((1, 1, 515), 1), ((1, 9, 515), 5), ((2, 11, 2064), 8), ((5, 257, 24), 24), ((1, 5000, 8), 2), ((1, 40000, 64), 16),
    ((70000, 16), 4), ((3, 1, 64), 16), ((1, 4099, 320), 32), ((2, 6, 6, 6, 32), 1), ((1, 700, 1280), 32),
    ((40, 100, 128), 32),
]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape,groups", NORM_SHAPES)
def test_group_norm(torch, ops, shape, groups, dtype):
    dt, g = dtype_of(torch, dtype), gen(torch, sum(shape) + groups)
    act = ACTS[(sum(shape) + len(dtype)) % 4]
    c = shape[-1]
    x = (torch.randn(shape, generator=g, device="cuda") * 2 + torch.randn(c, generator=g, device="cuda")).to(dt)
    w, b = (torch.randn(c, generator=g, device="cuda") for _ in range(2))
    y, mean, rstd = ops.group_norm(x, groups, w, b, act=act, stats=True)
    want, m64, r64, z = norm64(torch, x.double(), groups, w.double(), b.double(), 1e-5, act)
    assert y.dtype == dt and y.shape == x.shape
    within(y, want, norm_bound(torch, x.double(), groups, w.double(), m64, r64, z, want, dt), f"{shape} {act}")
    # mean: a few joins on terms of the group's size; rstd: relative, its variance loses a few e
    big = x.double().reshape(shape[0], -1, groups, c // groups).abs().amax((1, 3))
    within(mean, m64, 20 * E * big + 1e-30, "mean")
    within(rstd, r64, 40 * E * r64 * (1 + (big * r64).square().clamp_max(64)), "rstd")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_group_norm_activations(torch, ops, act, dtype):
    """Every activation over a wide range of its argument, the default scale and shift."""
    dt, g = dtype_of(torch, dtype), gen(torch, 5)
    x = torch.randn((2, 300, 64), generator=g, device="cuda").to(dt)
    w = torch.linspace(-30, 30, 64, device="cuda")
    for weight, bias in ((None, None), (w, None), (None, w), (w, w.flip(0).contiguous())):
        one, zero = torch.ones_like(w).double(), torch.zeros_like(w).double()
        w64, b64 = one if weight is None else weight.double(), zero if bias is None else bias.double()
        y = ops.group_norm(x, 8, weight, bias, eps=1e-3, act=act)
        want, m64, r64, z = norm64(torch, x.double(), 8, w64, b64, 1e-3, act)
        within(y, want, norm_bound(torch, x.double(), 8, w64, m64, r64, z, want, dt), act)


def test_group_norm_large_mean(torch, ops):
    """A mean a thousand times the spread: sums of squares of the values would lose it all."""
    g = gen(torch, 6)
    for mean in (1e3, -3e4):
        x = torch.randn((2, 3000, 64), generator=g, device="cuda") + mean
        y, m, r = ops.group_norm(x, 4, stats=True)
        want, m64, r64, z = norm64(torch, x.double(), 4, torch.ones(64, device="cuda").double(), 0.0, 1e-5, "none")
        one = torch.ones(64, device="cuda").double()
        within(y, want, norm_bound(torch, x.double(), 4, one, m64, r64, z, want, torch.float32), f"mean {mean}")
        within(r, r64, 1e-4 * r64, "rstd")


def test_group_norm_constant_and_special_values(torch, ops):
    # no spread: x - mean is 0, y = act(bias)
    y, m, r = ops.group_norm(torch.full((2, 37, 24), 3.0, device="cuda"), 3, bias=torch.arange(24.0, device="cuda"),
                             stats=True)
    assert torch.equal(y, torch.arange(24.0, device="cuda").expand(2, 37, 24)) and (m == 3).all()
    assert (r - 1e-5 ** -0.5).abs().max() < 1e-2
    # one far outlier, also as a thread's first value, does not spoil the variance
    x = torch.randn((1, 4096, 8), generator=gen(torch, 3), device="cuda")
    x[0, 0, 0] = 1e6
    y, m, r = ops.group_norm(x, 1, stats=True)
    _, m64, r64, _ = norm64(torch, x.double(), 1, 1.0, 0.0, 1e-5, "none")
    within(r, r64, 1e-3 * r64, "outlier rstd")
    # NaN and infinity stay in their picture's group
    x = torch.randn((3, 50, 32), generator=gen(torch, 4), device="cuda").half()
    x[1, 7, 3], x[2, 0, 31] = float("nan"), float("inf")
    y = ops.group_norm(x, 4, act="silu")
    bad = ~torch.isfinite(y)
    assert bad[1, :, :8].all() and bad[2, :, 24:].all()
    bad[1, :, :8] = False
    bad[2, :, 24:] = False
    assert not bad.any()


def test_group_norm_views(torch, ops):
    g = gen(torch, 8)
    wide = torch.randn((3, 5, 9, 100), generator=g, device="cuda").half()
    w, b = (torch.randn(40, generator=g, device="cuda") for _ in range(2))
    cases = {
        "channels of a wider map, aligned": wide[..., 8:48],
        "channels of a wider map, odd start": wide[..., 3:43],
        "one row of pixels": wide[:, :1, :, :40],
        "one column of pixels": wide[:, :, 2:3, :40],
        "a picture repeated": wide[:1, :, :, :40].expand(3, 5, 9, 40),
        "every other picture": wide[::2, :, :, :40],
    }
    for what, x in cases.items():
        want, m64, r64, z = norm64(torch, x.double(), 4, w.double(), b.double(), 1e-5, "silu")
        bound = norm_bound(torch, x.double(), 4, w.double(), m64, r64, z, want, torch.float16)
        within(ops.group_norm(x, 4, w, b, act="silu"), want, bound, what)
        out = torch.zeros((*x.shape[:3], 60), device="cuda").half()[..., 7:47]
        ops.group_norm(x, 4, w, b, act="silu", out=out)
        within(out, want, bound, what + ", into a view")
    x = wide[..., :40].contiguous()
    want = ops.group_norm(x, 4, w, b, act="gelu")
    assert ops.group_norm(x, 4, w, b, act="gelu", out=x) is x and torch.equal(x, want)  # in place


def test_group_norm_empty(torch, ops):
    y, m, r = ops.group_norm(torch.empty((0, 5, 8), device="cuda"), 2, stats=True)
    assert y.shape == (0, 5, 8) and m.shape == (0, 2)
    y, m, r = ops.group_norm(torch.empty((3, 0, 8), device="cuda"), 2, stats=True)
    assert y.shape == (3, 0, 8) and (m == 0).all() and torch.allclose(r, torch.full_like(r, 1e-5 ** -0.5))
    x = torch.empty((3, 0, 8), device="cuda")
    dx, dw, db = ops.group_norm_backward(x, x, m, r, 2)
    assert dx.shape == x.shape and not dw.any() and not db.any()


def test_group_norm_same_result_every_time(torch, ops):
    g = gen(torch, 9)
    x = torch.randn((2, 3001, 320), generator=g, device="cuda").bfloat16()
    dy = torch.randn((2, 3001, 320), generator=g, device="cuda").bfloat16()
    first = ops.group_norm(x, 32, act="silu", stats=True)
    grad = ops.group_norm_backward(dy, x, first[1], first[2], 32, act="silu")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.group_norm(x, 32, act="silu", stats=True)))
        again = ops.group_norm_backward(dy, x, first[1], first[2], 32, act="silu")
        assert all(torch.equal(a, b) for a, b in zip(grad, again))


def norm_grad64(torch, dy, x, groups, w, b, act):
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    y, *_ = norm64(torch, x, groups, w, b, 1e-5, act)
    return torch.autograd.grad(y, (x, w, b), dy)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape,groups", NORM_SHAPES)
def test_group_norm_backward(torch, ops, shape, groups, dtype):
    dt, g = dtype_of(torch, dtype), gen(torch, sum(shape) + groups)
    act = ACTS[(sum(shape) + groups + len(dtype)) % 4]
    n, c = shape[0], shape[-1]
    x = (torch.randn(shape, generator=g, device="cuda") * 2 + torch.randn(c, generator=g, device="cuda")).to(dt)
    dy = torch.randn(shape, generator=g, device="cuda").to(dt)
    w, b = (torch.randn(c, generator=g, device="cuda") for _ in range(2))
    _, m64, r64, z = norm64(torch, x.double(), groups, w.double(), b.double(), 1e-5, act)
    mean, rstd = m64.float(), r64.float()
    if act == "relu":  # where z is 0 to rounding, the slope may be either side's
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    dx, dw, db = ops.group_norm_backward(dy, x, mean, rstd, groups, w, b, act=act)
    wx, ww, wb = norm_grad64(torch, dy.double(), x.double(), groups, w.double(), b.double(), act)
    # xh is off by k1 = 4 e (|x| + |mean|) rstd; slopes change by at most that much times |w|.
    # Sums of m terms in partial sums: at most 64 e times the sum of the terms' sizes.
    per = (n, -1, groups, c // groups)
    xe = ((x.double().reshape(per).abs() + m64.abs().reshape(n, 1, groups, 1)) * r64.reshape(n, 1, groups, 1))
    xe = xe.reshape(shape) * (4 * E)
    hat = (x.double().reshape(per) - m64.reshape(n, 1, groups, 1)) * r64.reshape(n, 1, groups, 1)
    hat = hat.reshape(shape).abs()
    gz, dims = dy.double().abs() * 1.13, tuple(range(len(shape) - 1))
    ge = gz * (xe * w.double().abs() + 16 * E)  # error of a gz
    within(dw, ww, (ge * hat + gz * xe + 64 * E * gz * hat).sum(dims) + 1e-30, "dweight")
    within(db, wb, (ge + 64 * E * gz).sum(dims) + 1e-30, "dbias")
    h, he = gz * w.double().abs(), ge * w.double().abs()
    m1 = (he + 64 * E * h).reshape(per).mean((1, 3), keepdim=True)
    m2 = (he * hat + h * xe + 64 * E * h * hat).reshape(per).mean((1, 3), keepdim=True)
    s2 = (h * hat).reshape(per).mean((1, 3), keepdim=True)
    bound = (he + 16 * E * h).reshape(per) + m1 + hat.reshape(per) * m2 + (xe + 16 * E * hat).reshape(per) * s2
    bound = bound + 16 * E * h.reshape(per).mean((1, 3), keepdim=True)
    bound = (bound * r64.reshape(n, 1, groups, 1)).reshape(shape)
    within(dx, wx, bound + roundoff(torch, dt) * wx.abs() + least(torch, dt), f"dx {shape} {act}")


def test_group_norm_backward_differences(torch, ops):
    """Against central differences of the forward in 64 bits: with step h the formula's third
    derivative leaves h^2, 1e-6 of the gradient's size here."""
    g = gen(torch, 12)
    for act in ("none", "gelu", "silu"):
        x = torch.randn((1, 5, 8), generator=g, device="cuda")
        dy = torch.randn((1, 5, 8), generator=g, device="cuda")
        w, b = (torch.randn(8, generator=g, device="cuda") for _ in range(2))
        _, mean, rstd = ops.group_norm(x, 2, w, b, act=act, stats=True)
        got = ops.group_norm_backward(dy, x, mean, rstd, 2, w, b, act=act)
        at = [x.double(), w.double(), b.double()]
        for k, t in enumerate(at):
            num = torch.empty_like(t)
            for i in range(t.numel()):
                side = []
                for sign in (1, -1):
                    moved = t.clone()
                    moved.view(-1)[i] += sign * 1e-3
                    a = [*at]
                    a[k] = moved
                    side.append((norm64(torch, a[0], 2, a[1], a[2], 1e-5, act)[0] * dy.double()).sum())
                num.view(-1)[i] = (side[0] - side[1]) / 2e-3
            within(got[k], num, 1e-4 * (1 + num.abs().max()), f"{act} input {k}")


def test_group_norm_backward_views_and_autograd(torch, ops):
    g = gen(torch, 13)
    wide = torch.randn((2, 6, 7, 64), generator=g, device="cuda").half()
    x, dy = wide[..., 1:33], wide[..., 32:64]
    w, b = (torch.randn(32, generator=g, device="cuda") for _ in range(2))
    _, mean, rstd = ops.group_norm(x, 4, w, b, act="silu", stats=True)
    want = ops.group_norm_backward(dy.contiguous(), x.contiguous(), mean, rstd, 4, w, b, act="silu")
    got = ops.group_norm_backward(dy, x, mean, rstd, 4, w, b, act="silu")
    within(got[0], want[0].double(), 2 * 2.0 ** -11 * want[0].double().abs() + 1e-5, "dx of views")
    for k in (1, 2):
        within(got[k], want[k].double(), 1e-4 * want[k].double().abs() + 1e-4, "parameters of views")
    same = dy.contiguous()
    assert torch.equal(ops.group_norm_backward(same, x.contiguous(), mean, rstd, 4, w, b, act="silu", out=same)[0],
                       want[0])  # dx over dy
    # autograd: a broadcast gradient (of a sum), parameters given or not
    for wt, bt in ((w, b), (None, None), (w, None)):
        xs = x.float().clone().requires_grad_()
        ps = [None if t is None else t.clone().requires_grad_() for t in (wt, bt)]
        ops.GroupNormAct.apply(xs, 4, ps[0], ps[1], 1e-5, "silu").square().sum().backward()
        ref = x.double().clone().requires_grad_()
        pr = [torch.full((32,), v, device="cuda").double() if t is None else t.double().clone().requires_grad_()
              for t, v in ((wt, 1.0), (bt, 0.0))]
        norm64(torch, ref, 4, pr[0], pr[1], 1e-5, "silu")[0].square().sum().backward()
        within(xs.grad, ref.grad, 1e-4 * (1 + ref.grad.abs()), "autograd dx")
        for p, r in zip(ps, pr):
            assert p is None or (p.grad.double() - r.grad).abs().max() <= 1e-4 * (1 + r.grad.abs().max())


# ---------------------------------------------------------------------------- rotation
def pair_channels(sections, layout):
    pairs, at, out = sum(sections), 0, []
    for m in sections:
        for j in range(m):
            p = at + j
            out.append((2 * p, 2 * p + 1) if layout == "interleaved" else (p, p + pairs) if layout == "half"
                       else (2 * at + j, 2 * at + m + j))
        at += m
    return [p[0] for p in out], [p[1] for p in out]


def rotate64(torch, x, pos, freq, sections, layout, inverse):
    lo, hi = pair_channels(sections, layout)
    axis = [a for a, m in enumerate(sections) for _ in range(m)]
    t = (pos.float()[..., axis] * freq).double()  # the operator's angle is a float32 product
    t = (t if pos.dim() == 3 else t[None])[:, :, None] * (-1 if inverse else 1)
    y = x.double().clone()
    u, v = x.double()[..., lo], x.double()[..., hi]
    y[..., lo], y[..., hi] = u * t.cos() - v * t.sin(), u * t.sin() + v * t.cos()
    return y


def rotate_bound(torch, x, want, dt):
    """sin and cos to 2 ulp, two products and a sum on terms no larger than the pair."""
    return 8 * E * x.double().abs().amax(-1, keepdim=True) + roundoff(torch, dt) * want.abs() + least(torch, dt)


ROT_CASES = [  # b, l, h, hk, d, sections
    (1, 1, 1, 1, 2, (1,)), (1, 1, 16, 4, 64, (16, 16)), (2, 7, 3, 1, 24, (4, 4, 4)), (1, 33, 2, 2, 32, (8, 8)),
    (3, 17, 4, 2, 128, (16, 24, 24)), (2, 5, 1, 1, 40, (5, 7, 3)), (1, 100, 8, 8, 72, (12, 12, 12)),
    (1, 9, 2, 2, 15, (2, 3)), (1, 4, 2, 1, 16, (0, 8)), (2, 1023, 6, 2, 48, (6, 6, 6, 6)), (1, 3, 2, 2, 512, (100, 156)),
    (1, 2049, 12, 4, 128, (22, 20, 20)), (70001, 1, 1, 1, 8, (2, 2)),
]


@pytest.mark.parametrize("layout", ["half", "interleaved", "axial"])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("b,l,h,hk,d,sections", ROT_CASES)
def test_rotate_axes(torch, ops, b, l, h, hk, d, sections, dtype, layout):
    dt, g = dtype_of(torch, dtype), gen(torch, b + l + d)
    q, k = (torch.randn((b, l, n, d), generator=g, device="cuda").to(dt) for n in (h, hk))
    freq = torch.rand(sum(sections), generator=g, device="cuda")
    pos = torch.randint(-300, 300, (l, len(sections)), generator=g, device="cuda", dtype=torch.int32)
    for inverse in (False, True):
        yq, yk = ops.rotate_axes(q, k, pos, freq, sections, layout=layout, inverse=inverse)
        for x, y in ((q, yq), (k, yk)):
            want = rotate64(torch, x, pos, freq, sections, layout, inverse)
            within(y, want, rotate_bound(torch, x, want, dt), f"{layout} {inverse}")
            assert torch.equal(y[..., 2 * sum(sections):], x[..., 2 * sum(sections):])  # the rest is copied


def test_rotate_axes_positions(torch, ops):
    """Position types, per-picture and strided positions, fractions, large values."""
    g = gen(torch, 21)
    q = torch.randn((2, 50, 4, 32), generator=g, device="cuda")
    freq = torch.rand(16, generator=g, device="cuda")
    base = torch.randint(0, 200, (2, 50, 2), generator=g, device="cuda")
    tests = [base, base.int(), base.float() + 0.37, base[0], base[0].float() / 7,
             base.transpose(1, 2).contiguous().transpose(1, 2), base[:1].expand(2, 50, 2), base[:, :, :1].expand(2, 50, 2),
             base.float() * 1e4]
    for pos in tests:
        y, none = ops.rotate_axes(q, None, pos, freq, (9, 7), layout="axial")
        want = rotate64(torch, q, pos, freq, (9, 7), "axial", False)
        assert none is None
        within(y, want, rotate_bound(torch, q, want, torch.float32), f"{pos.dtype} {tuple(pos.stride())}")


@pytest.mark.parametrize("layout", ["half", "interleaved", "axial"])
def test_rotate_axes_views(torch, ops, layout):
    g = gen(torch, 22)
    for dt in (torch.float16, torch.float32):
        qkv = torch.randn((2, 37, 3, 6, 48), generator=g, device="cuda").to(dt)
        pos = torch.randint(0, 99, (37, 3), generator=g, device="cuda")
        freq = torch.rand(24, generator=g, device="cuda")
        wide = torch.randn((2, 37, 6, 51), generator=g, device="cuda").to(dt)
        heads_first = torch.randn((2, 6, 37, 48), generator=g, device="cuda").to(dt).transpose(1, 2)
        for q, k in ((qkv[:, :, 0], qkv[:, :, 1]), (wide[..., 1:49], wide[..., 3:51]), (heads_first, qkv[:, :, 2, :2]),
                     (qkv[:, :1, 0].expand(2, 37, 6, 48), qkv[:, :, 1, :1].expand(2, 37, 5, 48))):
            want = [rotate64(torch, t, pos, freq, (8, 8, 8), layout, False) for t in (q, k)]
            got = ops.rotate_axes(q, k, pos, freq, (8, 8, 8), layout=layout)
            for x, y, w in zip((q, k), got, want):
                within(y, w, rotate_bound(torch, x, w, dt), layout)
        q, k = qkv[:, :, 0], qkv[:, :, 1]
        v = qkv[:, :, 2].clone()
        want = ops.rotate_axes(q, k, pos, freq, (8, 8, 8), layout=layout)
        got = ops.rotate_axes(q, k, pos, freq, (8, 8, 8), layout=layout, out=(q, k))  # in place, inside qkv
        assert got[0] is q and all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(qkv[:, :, 2], v)
        q = torch.randn((1, 4, 2, 50), generator=g, device="cuda").to(dt)[..., 1:49]  # in place, odd alignment
        want = ops.rotate_axes(q, None, pos[:4], freq, (8, 8, 8), layout=layout)[0]
        assert torch.equal(ops.rotate_axes(q, None, pos[:4], freq, (8, 8, 8), layout=layout, out=(q, None))[0], want)


def test_rotate_axes_gradient(torch, ops):
    """The rotation is linear: <R x, y> = <x, R' y>, and turning back restores x."""
    g = gen(torch, 23)
    q, k = (torch.randn((2, 31, n, 32), generator=g, device="cuda") for n in (4, 2))
    pos = torch.randint(0, 60, (31, 2), generator=g, device="cuda")
    freq = torch.rand(14, generator=g, device="cuda")
    for layout in ("half", "interleaved", "axial"):
        a, c = q.clone().requires_grad_(), k.clone().requires_grad_()
        yq, yk = ops.RotateAxes.apply(a, c, pos, freq, (7, 7), layout)
        gq, gk = torch.randn_like(q), torch.randn_like(k)
        ((yq * gq).sum() + (yk * gk).sum()).backward()
        for x, gy in ((a, gq), (c, gk)):
            want = rotate64(torch, gy, pos, freq, (7, 7), layout, True)
            within(x.grad, want, rotate_bound(torch, gy, want, torch.float32), layout)
        # differences: a linear map's are exact, up to the float32 forward's rounding over the step
        back = ops.rotate_axes(yq.detach(), yk.detach(), pos, freq, (7, 7), layout=layout, inverse=True)
        for x, y in ((q, back[0]), (k, back[1])):
            within(y, x.double(), 16 * E * x.double().abs().amax(-1, keepdim=True), "there and back")
        a.grad = None
        ops.RotateAxes.apply(a, c, pos, freq, (7, 7), layout)[0].sum().backward()  # a broadcast gradient, k unused
        want = rotate64(torch, torch.ones_like(q), pos, freq, (7, 7), layout, True)
        within(a.grad, want, 8 * E + E * want.abs(), "broadcast gradient")


def test_rotate_axes_empty(torch, ops):
    freq = torch.ones(4, device="cuda")
    for b, l in ((0, 3), (2, 0)):
        q = torch.empty((b, l, 2, 8), device="cuda")
        yq, yk = ops.rotate_axes(q, q, torch.empty((l, 1), device="cuda"), freq, (4,))
        assert yq.shape == q.shape and yk.shape == q.shape


# ---------------------------------------------------------------------------- attention
def attention64(torch, q, k, v, scale, mask):
    share = q.shape[2] // k.shape[2]
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    if mask is not None:  # hidden keys do not exist
        seen = mask.bool()[:, None, :, None]
        k, v = torch.where(seen, k, 0.0), torch.where(seen, v, 0.0)
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    s = q @ k.transpose(2, 3) * scale
    size = q.abs() @ k.abs().transpose(2, 3) * abs(scale)
    if mask is not None:
        s = s.masked_fill(~mask.bool()[:, None, None, :], -math.inf)
    p = torch.softmax(s, 3).nan_to_num(0.0) if s.shape[3] else s
    return (p @ v).transpose(1, 2), (p @ v.abs()).transpose(1, 2), size.amax((2, 3)) if s.shape[3] else None


def check_attention(torch, ops, q, k, v, mask=None, scale=None, got=None, what=""):
    """Weights: the scores are float32 sums of d products of total size S, off by (d + 8) e S; a
    weight is rounded to the operands' type once, u; numerator and denominator: twice that.
    The output is rounded once."""
    d, dt = q.shape[3], q.dtype
    if got is None:
        got = ops.attention(q, k, v, key_mask=mask, scale=scale)
    want, size, s = attention64(torch, q, k, v, d ** -0.5 if scale is None else scale, mask)
    assert got.shape == q.shape and got.dtype == dt
    u = roundoff(torch, dt)
    off = 0 if s is None else ((d + 8) * E * s)[:, None, :, None]
    within(got, want, (2 * u + 2 * off + 32 * E) * size + u * want.abs() + least(torch, dt), what)


def qkv_of(torch, b, lq, lk, h, hk, d, dt, seed=0, loud=1.0):
    g = gen(torch, 1000 * seed + lq + lk + d)
    q = torch.randn((b, lq, h, d), generator=g, device="cuda") * loud
    k, v = (torch.randn((b, lk, hk, d), generator=g, device="cuda") for _ in range(2))
    return q.to(dt), k.to(dt), (v + 0.3).to(dt)


ATTN_CASES = [  # b, lq, lk, h, hk, d
    (1, 1, 1, 1, 1, 8), (1, 1, 5, 2, 1, 32), (2, 3, 130, 4, 2, 64), (1, 127, 128, 2, 2, 128), (1, 128, 127, 2, 2, 64),
    (2, 129, 129, 3, 1, 32), (1, 257, 300, 2, 2, 96), (1, 64, 1000, 4, 4, 40), (3, 33, 65, 2, 1, 16),
    (1, 500, 513, 1, 1, 80), (2, 1, 4097, 8, 8, 64), (1, 1, 20000, 4, 2, 128), (1, 2, 9000, 16, 1, 64),
    (1, 1000, 1, 2, 2, 64), (1, 16, 16, 2, 2, 72), (1, 9, 31, 2, 1, 7), (1, 40, 70, 2, 2, 256), (1, 30, 50, 1, 1, 129),
    (2, 300, 700, 6, 3, 64), (1, 385, 1025, 2, 1, 128), (1, 31, 1500, 24, 8, 32),
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,lq,lk,h,hk,d", ATTN_CASES)
def test_attention(torch, ops, b, lq, lk, h, hk, d, dtype):
    check_attention(torch, ops, *qkv_of(torch, b, lq, lk, h, hk, d, dtype_of(torch, dtype)))


@pytest.mark.parametrize("b,lq,lk,h,hk,d", [(700, 1, 300, 2, 2, 32), (300, 2, 140, 6, 2, 64), (150, 1, 257, 1, 1, 128),
                                            (40, 130, 200, 4, 4, 64), (1200, 1, 100, 1, 1, 16)])
def test_attention_many_pictures(torch, ops, b, lq, lk, h, hk, d):
    """More pictures and heads than CTAs run at once: several rounds, cut and whole units."""
    check_attention(torch, ops, *qkv_of(torch, b, lq, lk, h, hk, d, torch.float16, seed=7))


def test_attention_free_running_tiles(torch, ops):
    """One query over many keys, several times: the two key streams of a CTA run freely."""
    for heads_first in (False, True):
        q, k, v = qkv_of(torch, 2, 1, 16000, 8, 8, 64, torch.float16, seed=8)
        if heads_first:
            k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
        first = ops.attention(q, k, v)
        check_attention(torch, ops, q, k, v, got=first)
        assert all(torch.equal(first, ops.attention(q, k, v)) for _ in range(50))
    ops.status()


def test_attention_nan_and_infinity_in_visible_keys(torch, ops):
    """A NaN key makes every row that sees it NaN, an infinite score too; no other picture."""
    for lq in (3, 300):
        for bad in (math.nan, math.inf):
            for at in (0, 77, 150):
                q, k, v = qkv_of(torch, 2, lq, 200, 2, 2, 64, torch.float16, seed=9)
                q = q.abs() + 0.1
                k[1, at, 0] = bad
                out = ops.attention(q, k, v)
                assert torch.isnan(out[1, :, 0]).all() and torch.isfinite(out[0]).all()
                assert torch.isfinite(out[1, :, 1]).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,lq,lk,h,hk,d", [(4, 70, 300, 4, 2, 64), (4, 1, 3000, 2, 2, 128), (4, 200, 130, 2, 1, 32),
                                            (4, 5, 6, 1, 1, 7), (4, 140, 520, 2, 2, 40)])
def test_attention_masks(torch, ops, b, lq, lk, h, hk, d, dtype):
    """Masks of every kind in one batch: random, one key, nothing, the last part hidden; hidden
    keys hold NaN, infinities and the type's lowest value."""
    dt = dtype_of(torch, dtype)
    q, k, v = qkv_of(torch, b, lq, lk, h, hk, d, dt, seed=1)
    mask = torch.zeros((b, lk), dtype=torch.bool, device="cuda")
    mask[0] = torch.rand(lk, generator=gen(torch, lk), device="cuda") < 0.5
    mask[0, 0] = False
    mask[1, lk - 1] = True
    mask[3, : lk // 3] = True
    poison = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dt).min], device="cuda").to(dt)
    hidden = (~mask).nonzero()
    for t in (k, v):
        t[hidden[:, 0], hidden[:, 1]] = poison[torch.arange(len(hidden), device="cuda") % 4][:, None, None]
    out = ops.attention(q, k, v, key_mask=mask)
    check_attention(torch, ops, q, k, v, mask, got=out, what="mask")
    assert not out[2].any()  # no visible key: zeros
    assert torch.equal(out, ops.attention(q, k, v, key_mask=mask.to(torch.uint8) * 3))
    none = torch.zeros_like(mask)
    assert not ops.attention(q, k, v, key_mask=none).any()


def test_attention_views(torch, ops):
    for dt in (torch.float16, torch.bfloat16):
        qkv = torch.randn((2, 150, 3, 4, 64), generator=gen(torch, 31), device="cuda").to(dt)
        q, k, v = qkv.unbind(2)
        check_attention(torch, ops, q, k, v, what="packed")
        by_head = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
        check_attention(torch, ops, *by_head, what="heads first")
        odd = torch.randn((2, 150, 4, 67), generator=gen(torch, 32), device="cuda").to(dt)
        check_attention(torch, ops, odd[..., 1:65], odd[..., 2:66], odd[..., 3:67], what="odd alignment")
        check_attention(torch, ops, q, odd[..., 1:65], v, what="one operand of odd alignment")
        check_attention(torch, ops, q, k[:1].expand(2, -1, -1, -1), v[:, :, :1].expand(-1, -1, 4, -1), what="broadcast")
        check_attention(torch, ops, q, k[:, :1].expand(-1, 150, -1, -1), v, what="one key repeated")
        check_attention(torch, ops, q, k[:, ::2], v[:, ::2], what="every other key")
        mask = (torch.rand((2, 161), generator=gen(torch, 33), device="cuda") < 0.6)[:, 3:153]
        check_attention(torch, ops, q, k, v, mask, what="view of a mask")
        check_attention(torch, ops, q, k, v, mask[:1].expand(2, -1), what="shared mask")
        wide = torch.zeros((2, 150, 4, 100), device="cuda").to(dt)
        out = ops.attention(q, k, v, out=wide[..., 5:69])
        check_attention(torch, ops, q, k, v, got=out, what="into a view")
        assert not wide[..., :5].any() and not wide[..., 69:].any()
        out = torch.zeros((2, 4, 150, 64), device="cuda").to(dt).transpose(1, 2)
        check_attention(torch, ops, q, k, v, got=ops.attention(q, k, v, out=out), what="heads first out")


def test_attention_scores(torch, ops):
    """Loud and faint scores, a falling and a rising running maximum, scales of any sign."""
    q, k, v = qkv_of(torch, 1, 200, 900, 2, 2, 64, torch.float16, seed=2, loud=8.0)
    check_attention(torch, ops, q, k, v, what="loud")
    for order in (1, -1):
        ramp = torch.linspace(-4, 4, 900, device="cuda")[None, :, None, None] * order
        check_attention(torch, ops, q.abs(), (k * 0.1 + ramp).half(), v, what="ramp")
    for scale in (0.0, -0.3, 1e-4, 2.0):
        check_attention(torch, ops, q, k, v, scale=scale, what=f"scale {scale}")
    # one key far above all others takes the whole weight
    k2 = k.clone()
    k2[:, 450] = q[:, :1].mean(1) * 0 + 60
    check_attention(torch, ops, q.abs(), k2, v, what="one loud key")


def test_attention_empty(torch, ops):
    q, k, v = qkv_of(torch, 2, 5, 9, 2, 2, 64, torch.float16)
    assert not ops.attention(q, k[:, :0], v[:, :0]).any()
    assert ops.attention(q[:, :0], k, v).shape == (2, 0, 2, 64)
    assert ops.attention(q[:0], k[:0], v[:0]).shape == (0, 5, 2, 64)
    out = torch.full((2, 5, 2, 70), 7.0, device="cuda").half()
    ops.attention(q, k[:, :0], v[:, :0], out=out[..., :64])
    assert not out[..., :64].any() and (out[..., 64:] == 7).all()


def test_attention_same_result_every_time(torch, ops):
    for lq, lk in ((1, 9000), (700, 700)):
        q, k, v = qkv_of(torch, 2, lq, lk, 4, 2, 64, torch.bfloat16, seed=4)
        first = ops.attention(q, k, v)
        assert all(torch.equal(first, ops.attention(q, k, v)) for _ in range(4))


# ---------------------------------------------------------------------------- calls
def test_other_stream_and_graph(torch, ops):
    """On a stream of the user's own, and captured in a graph that is replayed on new inputs."""
    g = gen(torch, 41)
    x = torch.randn((2, 900, 64), generator=g, device="cuda").half()
    q, k, v = qkv_of(torch, 1, 90, 200, 2, 2, 64, torch.float16)
    pos = torch.randint(0, 30, (90, 2), generator=g, device="cuda")
    freq = torch.rand(32, generator=g, device="cuda")

    def everything():
        y, mean, rstd = ops.group_norm(x, 8, act="silu", stats=True)
        dx, dw, db = ops.group_norm_backward(y, x, mean, rstd, 8, act="silu")
        turned, _ = ops.rotate_axes(q, None, pos, freq, (16, 16))
        return y, dx, dw, db, turned, ops.attention(turned, k, v)

    want = everything()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = everything()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = everything()
    for t in (x, q, k, v):
        t.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, everything()))


def test_refusals(torch, ops, scb):
    x = torch.zeros((2, 5, 12), device="cuda").half()
    w = torch.ones(12, device="cuda")
    m = torch.zeros((2, 3), device="cuda")
    q = torch.zeros((2, 5, 4, 16), device="cuda").half()
    pos = torch.zeros((5, 2), device="cuda", dtype=torch.int32)
    f = torch.ones(8, device="cuda")
    bad = [
        lambda: ops.group_norm(x.cpu(), 3), lambda: ops.group_norm(x.double(), 3), lambda: ops.group_norm(x, 5),
        lambda: ops.group_norm(x, 0), lambda: ops.group_norm(x, 3, act="tanh"), lambda: ops.group_norm(x, 3, w.half()),
        lambda: ops.group_norm(x, 3, w[:6]), lambda: ops.group_norm(x, 3, None, w.cpu()),
        lambda: ops.group_norm(x.transpose(1, 2), 1), lambda: ops.group_norm(x, 3, out=x.float()),
        lambda: ops.group_norm(x, 3, out=x[:1].expand(2, 5, 12)), lambda: ops.group_norm(x, 3, eps=-1.0),
        lambda: ops.group_norm(x[0, 0], 3), lambda: ops.group_norm(torch.zeros((2, 4, 6, 12), device="cuda")[:, :3, :5], 3),
        lambda: ops.group_norm_backward(x[:1], x, m, m, 3), lambda: ops.group_norm_backward(x, x, m.half(), m, 3),
        lambda: ops.group_norm_backward(x, x, m[:1], m, 3), lambda: ops.group_norm_backward(x, x, m, m, 4),
        lambda: ops.rotate_axes(q, q, pos, f, (4, 5)), lambda: ops.rotate_axes(q, q, pos, f, (8,)),
        lambda: ops.rotate_axes(q, q, pos.half(), f, (4, 4)), lambda: ops.rotate_axes(q, q, pos, f[:7], (4, 4)),
        lambda: ops.rotate_axes(q, q.float(), pos, f, (4, 4)), lambda: ops.rotate_axes(q, q, pos[:4], f, (4, 4)),
        lambda: ops.rotate_axes(q, q, pos, f, (4, 4), layout="odd"), lambda: ops.rotate_axes(q[0], None, pos, f, (4, 4)),
        lambda: ops.rotate_axes(q, q, pos, f, (9, -1)), lambda: ops.rotate_axes(q, q, pos.cpu(), f, (4, 4)),
        lambda: ops.rotate_axes(q, None, pos, f, (4, 4), out=(q[:, :1].expand(2, 5, 4, 16), None)),
        lambda: ops.rotate_axes(q, None, torch.zeros((5, 5), device="cuda"), f, (2, 2, 2, 1, 1)),
        lambda: ops.rotate_axes(q.transpose(2, 3), None, pos, f, (4, 4)),
        lambda: ops.attention(q.float(), q.float(), q.float()), lambda: ops.attention(q, q[:, :, :3], q[:, :, :3]),
        lambda: ops.attention(q, q, q[:, :4]), lambda: ops.attention(q, q[:1], q[:1]), lambda: ops.attention(q, q, q.cpu()),
        lambda: ops.attention(q, q, q, key_mask=torch.zeros((2, 4), device="cuda")),
        lambda: ops.attention(q, q, q, key_mask=torch.zeros((2, 5), device="cuda")),
        lambda: ops.attention(q, q, q, scale=math.inf), lambda: ops.attention(q, q, q, out=q[:, :1].expand(2, 5, 4, 16)),
        lambda: ops.attention(*[torch.zeros((1, 2, 1, 264), device="cuda").half()] * 3),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(scb.BackendError) as e:
            call()
        assert len(str(e.value)) > 10, k
    torch.cuda.synchronize()
    assert not x.any() and not q.any()  # nothing ran
