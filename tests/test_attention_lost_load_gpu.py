"""A load of the attention kernel that never comes (left out on purpose): its waits run out after
a second, the rows it had a part in are NaN, `status` tells, and the next call is as ever."""
import time

import pytest

from test_ops_gpu import ops, qkv_of, torch  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu

# b, lq, lk, h, hk, d; the load; what CTA 0 has a part in, as slices of [b, lq, h]
LOST = {
    "whole units, the first keys": ((2, 300, 300, 2, 2, 64), 0, (0, slice(0, 256), 0)),
    "whole units, the last values": ((2, 300, 300, 2, 2, 32), 5, (0, slice(0, 256), 0)),
    "cut units": ((1, 300, 1025, 1, 1, 128), 3, (0, slice(0, 256), 0)),
    "few rows, eight units": ((2, 1, 3000, 4, 4, 64), 2, (0, 0, 0)),
    "few rows, eight units, shared heads, wide": ((2, 3, 1025, 8, 4, 128), 1, (0, slice(0, 3), slice(0, 2))),
    "few rows": ((2, 1, 3000, 2, 2, 64), 2, (0, 0, 0)),
    "few rows, wide": ((1, 3, 1025, 2, 2, 128), 1, (0, slice(0, 3), 0)),
}


def lost_load(scb, ops, torch, q, k, v, load):  # noqa: F811
    """ops.attention with a load left out."""
    lib, out = scb.load_library(), torch.zeros_like(q)
    b, lq, h, d = q.shape
    _, lk, hk, _ = k.shape
    rows = [scb.backend.ScbRows(t.data_ptr(), *t.stride()[:3]) for t in (q, k, v, out)]
    _work, work, size = ops._workspace("scb_attention_workspace", q, b, lq, lk, h, hk, d)
    rc = lib.scb_probe_attention_lost(*rows, scb.backend.SCB_F16, b, lq, lk, h, hk, d, None, 0, d ** -0.5, work, size,
                                      torch.cuda.current_stream().cuda_stream, load)
    assert rc == 0, lib.scb_last_error(None)
    return out


@pytest.mark.parametrize("case", list(LOST))
def test_lost_load(torch, ops, scb, case):  # noqa: F811
    sizes, load, part = LOST[case]
    q, k, v = qkv_of(torch, *sizes, torch.float16, seed=91)
    want = ops.attention(q, k, v)
    ops.status()
    t = time.perf_counter()
    out = lost_load(scb, ops, torch, q, k, v, load)
    with pytest.raises(scb.BackendError, match="bounded wait"):
        ops.status()
    # one wait runs out, and the wait for the lost load before the CTA ends
    assert time.perf_counter() - t < 4.5
    assert torch.isnan(out[part]).all()
    rest = torch.ones(out.shape[:3], dtype=torch.bool, device="cuda")
    rest[part] = False
    assert torch.equal(out[rest], want[rest])
    assert torch.equal(ops.attention(q, k, v), want)
    ops.status()
