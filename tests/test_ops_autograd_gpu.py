"""The block operators and autograd."""
import pytest

from test_ops_gpu import E, gen, ops, qkv_of, rotate64, torch, within  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def positions(torch):  # noqa: F811
    g = gen(torch, 81)
    return (torch.randint(0, 60, (31, 2), generator=g, device="cuda"), torch.rand(14, generator=g, device="cuda"))


def test_rotate_axes_without_k(torch, ops):  # noqa: F811
    pos, freq = positions(torch)
    q = torch.randn((2, 31, 4, 32), generator=gen(torch, 85), device="cuda").requires_grad_()
    y, none = ops.RotateAxes.apply(q, None, pos, freq, (7, 7), "axial")
    assert none is None
    dy = torch.randn_like(y)
    y.backward(dy)
    want = rotate64(torch, dy, pos, freq, (7, 7), "axial", True)
    within(q.grad, want, 8 * E * dy.double().abs().amax(-1, keepdim=True) + E * want.abs(), "dq")


def test_group_norm_has_no_second_derivative(torch, ops):  # noqa: F811
    """A gradient penalty needs it: an error, not a wrong gradient."""
    x = torch.randn((2, 40, 32), generator=gen(torch, 82), device="cuda").requires_grad_()
    w = torch.ones(32, device="cuda", requires_grad=True)
    y = ops.GroupNormAct.apply(x, 4, w, None, 1e-5, "silu")
    dx, = torch.autograd.grad((y * x).sum(), x, create_graph=True)  # x also reaches the loss directly
    with pytest.raises(RuntimeError, match="differentiat"):
        dx.square().sum().backward()
    # without create_graph all is as before
    dx, = torch.autograd.grad(ops.GroupNormAct.apply(x, 4, w, None, 1e-5, "silu").square().sum(), x)
    assert torch.isfinite(dx).all() and not dx.requires_grad


@pytest.mark.parametrize("layout", ["half", "interleaved", "axial"])
def test_rotate_axes_second_derivative(torch, ops, layout):  # noqa: F811
    """The rotation is linear, its gradient is the inverse rotation, and so on."""
    pos, freq = positions(torch)
    q, k = (torch.randn((2, 31, n, 32), generator=gen(torch, 83 + n), device="cuda") for n in (4, 2))

    def penalty(turn, q, k):
        yq, yk = turn(q, k)
        dq, dk = torch.autograd.grad((yq ** 3).sum() + (yk ** 3).sum() + (q ** 2).sum(), (q, k), create_graph=True)
        return torch.autograd.grad(dq.square().sum() + (dk ** 2).sum(), (q, k))

    def plain(q, k):
        return tuple(rotate64(torch, t, pos, freq, (7, 7), layout, False) for t in (q, k))

    got = penalty(lambda a, b: ops.RotateAxes.apply(a, b, pos, freq, (7, 7), layout),
                  q.clone().requires_grad_(), k.clone().requires_grad_())
    want = penalty(plain, q.double().requires_grad_(), k.double().requires_grad_())
    for a, b in zip(got, want):  # a chain of four rotations and some powers: below 100 operations on the row's terms
        within(a, b, 100 * E * (1 + b.abs().amax((2, 3), keepdim=True)), layout)


def test_rotate_axes_inverse_under_autograd(torch, ops):  # noqa: F811
    pos, freq = positions(torch)
    q = torch.randn((2, 31, 4, 32), generator=gen(torch, 86), device="cuda").requires_grad_()
    there = ops.RotateAxes.apply(q, None, pos, freq, (7, 7))[0]
    back = ops.RotateAxes.apply(there, None, pos, freq, (7, 7), "half", True)[0]
    g = torch.randn_like(q)
    back.backward(g)
    within(q.grad, g.double(), 16 * E * g.double().abs().amax(-1, keepdim=True), "identity's gradient")


def test_gradients_that_would_be_lost_are_refused(torch, ops, scb):  # noqa: F811
    pos, freq = positions(torch)
    x = torch.randn((2, 31, 4, 32), generator=gen(torch, 87), device="cuda")
    w = torch.ones(32, device="cuda")
    m = torch.ones((2, 4), device="cuda")
    q, k, v = qkv_of(torch, 1, 40, 50, 2, 2, 64, torch.float16)

    def on(t):
        return t.clone().requires_grad_()

    calls = {
        "GroupNormAct": [lambda: ops.group_norm(on(x), 4), lambda: ops.group_norm(x, 4, on(w)),
                         lambda: ops.group_norm(x, 4, None, on(w)), lambda: ops.group_norm(x, 4, out=on(x))],
        "second": [lambda: ops.group_norm_backward(on(x), x, m, m, 4), lambda: ops.group_norm_backward(x, on(x), m, m, 4),
                   lambda: ops.group_norm_backward(x, x, on(m), m, 4), lambda: ops.group_norm_backward(x, x, m, on(m), 4),
                   lambda: ops.group_norm_backward(x, x, m, m, 4, on(w))],
        "RotateAxes": [lambda: ops.rotate_axes(on(x), None, pos, freq, (7, 7)),
                       lambda: ops.rotate_axes(x, on(x), pos, freq, (7, 7)),
                       lambda: ops.rotate_axes(x, x, pos, freq, (7, 7), out=(x.clone(), on(x)))],
        "inv_freq": [lambda: ops.rotate_axes(x, None, pos.float().requires_grad_(), freq, (7, 7)),
                     lambda: ops.rotate_axes(x, None, pos, on(freq), (7, 7))],
        "attention": [lambda: ops.attention(on(q), k, v), lambda: ops.attention(q, on(k), v),
                      lambda: ops.attention(q, k, on(v)), lambda: ops.attention(q, k, v, out=on(q))],
    }
    for words, some in calls.items():
        for call in some:
            with pytest.raises(scb.BackendError, match=words):
                call()
    with torch.no_grad():  # nobody asks for a gradient: they run
        for some in calls.values():
            for call in some:
                call()
    with torch.inference_mode():
        ops.attention(q, k, v, out=torch.empty_like(q))
    for turn in (lambda: ops.RotateAxes.apply(x, None, pos, on(freq), (7, 7)),
                 lambda: ops.RotateAxes.apply(on(x), x, pos.float().requires_grad_(), freq, (7, 7))):
        with pytest.raises(scb.BackendError, match="inv_freq"):
            turn()[0].sum().backward()
        with torch.no_grad():
            turn()


def test_out_counts_as_written(torch, ops):  # noqa: F811
    """Writing over a tensor that autograd saved is found in the backward pass."""
    pos, freq = positions(torch)
    x = torch.randn((2, 31, 4, 32), generator=gen(torch, 88), device="cuda")
    stats = ops.group_norm(x, 4, stats=True)[1:]
    q, k, v = qkv_of(torch, 1, 40, 50, 2, 2, 64, torch.float16)
    writes = [
        (x, lambda t: ops.group_norm(x, 4, out=t)),
        (x, lambda t: ops.group_norm_backward(x, x, *stats, 4, out=t)),
        (x, lambda t: ops.rotate_axes(x, None, pos, freq, (7, 7), out=(t, None))),
        (x, lambda t: ops.rotate_axes(x, x, pos, freq, (7, 7), out=(torch.empty_like(x), t))),
        (q, lambda t: ops.attention(q, k, v, out=t)),
    ]
    for like, write in writes:
        w = torch.ones_like(like, requires_grad=True)
        saved = like.clone()
        y = (w * saved).sum()
        write(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
