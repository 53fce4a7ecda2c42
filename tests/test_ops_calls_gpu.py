"""What a failed call leaves behind."""
import ctypes

import pytest

from test_ops_gpu import ops, torch  # noqa: F401 (fixtures)

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
