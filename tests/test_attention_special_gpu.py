"""Attention where scores or values are not ordinary numbers, whatever way the work is cut: the
few-row form (every unit leaves pieces), units cut between CTAs, whole units, and the general
kernel."""
import math

import pytest

from test_ops_gpu import check_attention, ops, qkv_of, torch  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu

CUTS = {  # b, lq, lk, h, hk, d
    "few rows, eight units": (2, 1, 3000, 4, 4, 64),
    "few rows, eight units, shared heads, wide": (2, 3, 1025, 8, 4, 128),
    "few rows, many pictures": (160, 2, 500, 1, 1, 32),
    "few rows": (2, 1, 3000, 2, 2, 64),
    "few rows, shared heads, wide": (1, 3, 1025, 4, 2, 128),
    "few rows, one piece a tile": (2, 2, 257, 1, 1, 32),
    "cut units": (1, 300, 1025, 1, 1, 64),
    "cut units, wide": (1, 300, 2049, 2, 1, 128),
    "whole units": (2, 300, 300, 2, 2, 64),
    "whole units, one tile": (3, 40, 100, 2, 1, 32),
    "general kernel": (2, 5, 300, 2, 1, 129),
}
cuts = pytest.mark.parametrize("cut", list(CUTS))


@cuts
def test_nan_query(torch, ops, cut):  # noqa: F811
    """A NaN in a query makes that query's row NaN, and no other row."""
    b, lq, lk, h, hk, d = CUTS[cut]
    q, k, v = qkv_of(torch, b, lq, lk, h, hk, d, torch.float16, seed=51)
    q[0, lq - 1, 0, d - 1] = math.nan
    out = ops.attention(q, k, v)
    bad = torch.isnan(out)
    assert bad[0, lq - 1, 0].all()
    bad[0, lq - 1, 0] = False
    assert not bad.any()


@cuts
@pytest.mark.parametrize("where", ["k", "v"])
def test_nan_key_alone_in_its_piece(torch, ops, cut, where):  # noqa: F811
    """The first keys and the last one are visible, and the last one is NaN: every row is."""
    b, lq, lk, h, hk, d = CUTS[cut]
    q, k, v = qkv_of(torch, b, lq, lk, h, hk, d, torch.float16, seed=52)
    mask = torch.zeros((b, lk), dtype=torch.bool, device="cuda")
    mask[:, :50] = mask[:, -1] = True
    (k if where == "k" else v)[0, -1] = math.nan
    out = ops.attention(q, k, v, key_mask=mask)
    assert torch.isnan(out[0]).all()
    assert torch.isfinite(out[1:]).all()
    mask[:, -1] = False  # hidden, it does not matter
    check_attention(torch, ops, q, k, v, mask)
