"""Scores of minus infinity on visible keys, and values that a weight of zero has to remove."""
import math

import pytest

from test_attention_special_gpu import CUTS, cuts
from test_ops_gpu import check_attention, ops, qkv_of, torch  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def infinite_keys(torch, cut, dt, seed):  # noqa: F811
    """Queries that are positive in channel 0, so that a key with -inf there scores -inf."""
    b, lq, lk, h, hk, d = CUTS[cut]
    q, k, v = qkv_of(torch, b, lq, lk, h, hk, d, dt, seed=seed)
    q[..., 0] = q[..., 0].abs() + 0.5
    return q, k, v


@cuts
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_all_visible_scores_minus_infinity(torch, ops, cut, dtype):  # noqa: F811
    """softmax of nothing but -inf is 0 / 0: NaN, with and without hidden keys beside them; with
    no visible key the row is zero, whatever the hidden keys score."""
    q, k, v = infinite_keys(torch, cut, getattr(torch, dtype), 61)
    ordinary = k.clone()
    k[0, :, :, 0] = -math.inf
    out = ops.attention(q, k, v)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1:]).all()
    mask = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    mask[:, 3] = mask[:, -2] = True
    out = ops.attention(q, k, v, key_mask=mask)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1:]).all()
    mask[0] = False
    out = ops.attention(q, k, v, key_mask=mask)
    assert not out[0].any()
    check_attention(torch, ops, q, ordinary, v, mask, got=out)


@cuts
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("finite", ["first", "last", "some"])
def test_some_scores_minus_infinity(torch, ops, cut, dtype, finite):  # noqa: F811
    """Such keys weigh nothing where a row has a finite score, as hidden keys do."""
    q, k, v = infinite_keys(torch, cut, getattr(torch, dtype), 62)
    lk = k.shape[1]
    keep = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    if finite == "some":
        keep[:] = torch.arange(lk, device="cuda") % 7 == 5
    else:
        keep[:, 0 if finite == "first" else lk - 1] = True
    bad = torch.where(keep[:, :, None, None], k, torch.tensor(-math.inf, device="cuda", dtype=k.dtype))
    bad[..., 1:] = k[..., 1:]
    check_attention(torch, ops, q, k, v, keep, got=ops.attention(q, bad, v))


@cuts
def test_bf16_products_that_overflow(torch, ops, cut):  # noqa: F811
    """Finite operands whose scores overflow to -inf, in every row."""
    q, k, v = infinite_keys(torch, cut, torch.bfloat16, 63)
    q[..., 0], k[..., 0] = 1e30, -1e30
    assert torch.isnan(ops.attention(q, k, v)).all()


@cuts
def test_weights_that_vanish(torch, ops, cut):  # noqa: F811
    """Keys a thousand below the best weigh e^-1000, nothing, even on values of 2^115 (whose
    plain sum still is a float32)."""
    b, lq, lk, h, hk, d = CUTS[cut]
    q = torch.zeros((b, lq, h, d), device="cuda").bfloat16()
    k = torch.zeros((b, lk, hk, d), device="cuda").bfloat16()
    v = torch.full((b, lk, hk, d), 2.0 ** 115, device="cuda").bfloat16()
    q[..., 0], k[..., 0] = 1.0, -1000.0
    k[:, lk // 2, :, 0], v[:, lk // 2] = 0.0, 1.0
    assert (ops.attention(q, k, v, scale=1.0) == 1).all()
