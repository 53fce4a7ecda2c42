"""What a failed call leaves behind."""
import ctypes

import pytest

from test_ops_gpu import check_attention, ops, qkv_of, torch  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def test_an_error_is_reported_once(torch, ops, scb):  # noqa: F811
    """A call that fails leaves no error behind that the next one would report as its own."""
    x = torch.randn((2, 300, 64), device="cuda")
    want = ops.group_norm(x, 4)
    torch.cuda.synchronize()
    # waiting for a stream that is being captured is an error of the runtime
    runtime = ctypes.CDLL("libcudart.so.12")
    stream, graph = torch.cuda.Stream(), ctypes.c_void_p()
    handle = ctypes.c_void_p(stream.cuda_stream)
    assert runtime.cudaStreamBeginCapture(handle, 2) == 0  # relaxed: only this stream's own calls count
    try:
        with pytest.raises(scb.BackendError, match="captur"):
            ops.status(stream)
    finally:
        runtime.cudaStreamEndCapture(handle, ctypes.byref(graph))  # the capture has failed
        runtime.cudaGetLastError()
    assert torch.equal(ops.group_norm(x, 4), want)
    ops.status()
    torch.cuda.synchronize()


def test_few_row_workspace_is_what_is_written(torch, ops):  # noqa: F811
    """One query for each of many pictures: a piece a CTA, 128 rows of two key streams with a
    maximum and a sum each, and no more than that."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    pictures = 2 * sms  # more than one round, so a CTA takes a whole picture
    q = torch.randn((pictures, 1, 1, 128), device="cuda").half()
    k = torch.randn((pictures, 600, 1, 128), device="cuda").half()
    assert ops._work_bytes("scb_attention_workspace", 0, pictures, 1, 600, 1, 1, 128) == pictures * 256 * (128 + 2) * 4
    want = torch.softmax(torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double()) * 128 ** -0.5, 3)
    want = torch.einsum("bhqk,bkhd->bqhd", want, k.double())
    assert (ops.attention(q, k, k).double() - want).abs().max() < 4 * 2.0 ** -11 * 5  # |k| up to 5


@pytest.mark.parametrize("heads,lq,lk,d", [(200, 256, 128, 128), (200, 256, 40, 64), (1200, 1, 100, 16),
                                           (216, 250, 300, 64)])
def test_next_kernel_sees_every_row(torch, ops, heads, lq, lk, d):  # noqa: F811
    """What the stream runs after attention starts when all its rows are there, also where units
    outnumber the CTAs and none is cut."""
    q, k, v = qkv_of(torch, 1, lq, lk, heads, heads, d, torch.float16, seed=95)
    for _ in range(20):
        out = torch.zeros_like(q)
        ops.attention(q, k, v, out=out)
        then = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(then, out)
    check_attention(torch, ops, q, k, v, got=then)
    if lk <= 128:  # whole units leave no pieces
        assert ops._work_bytes("scb_attention_workspace", 0, 1, lq, lk, heads, heads, d) == 0
