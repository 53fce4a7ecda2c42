"""Scores of minus infinity on visible keys, and values that a weight of zero has to remove."""
import pytest

from test_attention_special_gpu import CUTS, cuts
from test_ops_gpu import ops, torch  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


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
