"""Group norm where the rows that a block takes its shift from are far from all others."""
import pytest

from test_ops_gpu import E, norm64, ops, torch  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def edges(l, row_step, blocks):
    """First and last rows of each of `blocks` ranges, and of walks of `row_step` rows."""
    each = -(-l // blocks)
    rows = {r for k in range(blocks) for r in (k * each, min(l, (k + 1) * each) - 1)}
    return sorted(rows | {0, l - 1} | {r for r in ((l - 1) // row_step * row_step,) if r})


@pytest.mark.parametrize("far", [30.0, 1e3, 1e6])
@pytest.mark.parametrize("l,c,groups,step,blocks", [(200003, 64, 64, 32 * 296, 1), (1088 * 1920, 64, 16, 32 * 296, 1),
                                                    (3000, 64, 4, 1, 8), (40000, 64, 64, 1, 8), (150, 512, 32, 1, 1)])
def test_far_first_and_last_rows(torch, ops, l, c, groups, step, blocks, far):  # noqa: F811
    """Two of the three rows that set the shift lie `far` spreads away. The block then sums about
    its own mean, or accepts a sum of squares of at most 64 times M2: 64 roundings of it and 64
    more of a thread's and the block's partial sums at most, half of that in rstd; the mean
    within a few roundings of `far`."""
    x = torch.randn((1, l, c), generator=torch.Generator(device="cuda").manual_seed(l), device="cuda")
    x[0, edges(l, step, blocks)] = far
    _, mean, rstd = ops.group_norm(x, groups, stats=True)
    _, m64, r64, _ = norm64(torch, x.double(), groups, 1.0, 0.0, 1e-5, "none")
    off = float(((rstd.double() - r64) / r64).abs().max())
    assert off <= 64 * E, off / E
    assert float((mean.double() - m64).abs().max()) <= 64 * E * (1 + far)
