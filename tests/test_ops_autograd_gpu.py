"""The block operators and autograd."""
import pytest

from test_ops_gpu import E, gen, ops, rotate64, torch, within  # noqa: F401 (fixtures)

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
