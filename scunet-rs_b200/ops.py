"""Block operators on torch CUDA tensors, over the context-free entries of
`include/scunet_b200.h`: what image and video U-Net blocks use beside the network's own.

  group_norm, group_norm_backward   group norm with an activation, channels last
  rotate_axes                       queries and keys rotated by time / row / column
  attention                         attention over all tokens of a map, with a key mask
  status                            wait, and raise if a kernel gave up on a device wait

Every call runs on the current stream of its tensors' device, takes its outputs and its
workspace from torch's caching allocator (so a workspace lives as long as the stream needs
it) and returns before the GPU has finished. Inputs may be views: only the channels have to
be contiguous. An `out` may not overlap an input except where that is said, and counts as
written in place for autograd. `GroupNormAct` and `RotateAxes` are the same for autograd; the
functions themselves, and attention, which has no gradient, refuse tensors that require one
while gradients are recorded. Wrong arguments raise `BackendError`; there is no fallback for
tensors that are not on a CUDA device.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from .backend import (SCB_ACTS, SCB_BF16, SCB_F16, SCB_F32, SCB_I32, SCB_I64, SCB_ROT_LAYOUTS, BackendError, ScbHeads,
                      ScbRows, load_library)

_DTYPES = {torch.float32: SCB_F32, torch.float16: SCB_F16, torch.bfloat16: SCB_BF16}
_POSITIONS = {torch.int32: SCB_I32, torch.int64: SCB_I64, torch.float32: SCB_F32}
_lib = None


def _fail(msg):
    raise BackendError(msg)


def _library():
    global _lib
    if _lib is None:
        _lib = load_library()
    return _lib


# The handle of a device's current stream: torch.cuda.current_stream(index).cuda_stream
# without the Stream object, which costs 2 us a call.
_stream = torch._C._cuda_getCurrentRawStream


def _call(t, fn, *args):
    """fn(*args, stream) on the current stream of t's device; a failure raises its message."""
    index = t.get_device()
    if index == torch.cuda.current_device():
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc != 0:
        _fail(_library().scb_last_error(None).decode())


@functools.lru_cache(maxsize=4096)
def _work_bytes(name, device, *sizes):
    """The workspace of an operator for these sizes on this device."""
    need = ctypes.c_size_t(0)
    with torch.cuda.device(device):
        if getattr(_library(), name)(*sizes, ctypes.byref(need)) != 0:
            _fail(_library().scb_last_error(None).decode())
    return need.value


def _workspace(name, t, *sizes):
    """(tensor to keep until the call is launched, its address, its bytes)"""
    need = _work_bytes(name, t.get_device(), *sizes)
    if not need:
        return None, None, 0
    work = t.new_empty(need, dtype=torch.uint8)
    return work, work.data_ptr(), need


def _dtype(t, what):
    if not t.is_cuda:
        _fail(f"{what} must be on a CUDA device")
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        _fail(f"{what} must be float32, float16 or bfloat16, not {t.dtype}")
    return dt


def _same(t, like, what):
    if t.dtype != like.dtype or t.get_device() != like.get_device() or t.shape != like.shape:
        _fail(f"{what} must be {tuple(like.shape)} {like.dtype} on {like.device}, "
              f"not {tuple(t.shape)} {t.dtype} on {t.device}")


def _params(t, c, like, what):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.get_device() != like.get_device() or t.shape != (c,) or not t.is_contiguous():
        _fail(f"{what} must be {c} contiguous float32 values on {like.device}")
    return t.data_ptr()


_recording = torch.is_grad_enabled


def _no_gradient(why, *tensors):
    """Refuses tensors whose gradient the call would drop from the graph without a word (the
    caller has looked whether gradients are recorded at all)."""
    for t in tensors:
        if t is not None and t.requires_grad:
            _fail(why + " (or call it under torch.no_grad())")


def _rows(t, what):
    """(pictures, rows, channels, picture stride, row stride) of [n][...][c]; the dimensions
    between collapse to rows of one stride."""
    shape, stride = t.shape, t.stride()
    dims = len(shape)
    if dims < 2:
        _fail(f"{what} must be [pictures, ..., channels]")
    if shape[-1] > 1 and stride[-1] != 1:
        _fail(f"{what}: the channels must be contiguous (channels last)")
    if dims == 3:
        return shape[0], shape[1], shape[2], stride[0], stride[1]
    rows, sl = 1, 0
    for size, st in zip(reversed(shape[1:-1]), reversed(stride[1:-1])):
        if size == 1:
            continue
        if rows > 1 and st != sl * rows:
            _fail(f"{what}: the dimensions between pictures and channels must have one common row stride")
        if rows == 1:
            sl = st
        rows *= size
    return shape[0], rows, shape[-1], stride[0], sl


def _out(out, like, what="out"):
    """`out`, checked, or new contiguous memory of like's shape."""
    if out is None:
        return like.new_empty(like.shape)
    _same(out, like, what)
    return out


def _ptr(t):
    return None if t is None else t.data_ptr()


def _act(act):
    if act not in SCB_ACTS:
        _fail(f"unknown activation {act!r}")
    return SCB_ACTS[act]


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, act="none", out=None, stats=False):
    """act((x - mean) / sqrt(var + eps) * weight + bias) of x [n, ..., c], channels last.

    Mean and variance are those of each picture's c / groups neighbouring channels; weight
    and bias are float32 [c]; act is "none", "relu", "gelu" (exact) or "silu". `out` may be x.
    With stats=True also returns mean and 1 / sqrt(var + eps), float32 [n, groups]."""
    dt = _dtype(x, "x")
    if _recording():
        _no_gradient("group_norm gives no gradient: use GroupNormAct.apply", x, weight, bias, out)
    n, l, c, sn, sl = _rows(x, "x")
    y = _out(out, x)
    yn, yl = (l * c, c) if out is None else _rows(y, "out")[3:]
    mean = rstd = None
    if stats:
        mean, rstd = (x.new_empty((n, max(groups, 1)), dtype=torch.float32) for _ in range(2))
    _work, work, size = _workspace("scb_group_norm_workspace", x, n, l, c, groups)
    _call(x, _library().scb_group_norm, x.data_ptr(), sn, sl, dt, n, l, c, groups, _params(weight, c, x, "weight"),
          _params(bias, c, x, "bias"), eps, _act(act), y.data_ptr(), yn, yl, _ptr(mean), _ptr(rstd), work, size)
    if out is not None:
        increment_version(out)
    return (y, mean, rstd) if stats else y


def group_norm_backward(dy, x, mean, rstd, groups, weight=None, bias=None, *, act="none", out=None):
    """(dx, dweight, dbias) of group_norm from dy, its x and its mean and rstd (stats=True).
    dweight and dbias are float32 [c] whether or not weight and bias are given; `out` (dx) may
    be dy or x."""
    dt = _dtype(x, "x")
    if _recording():
        _no_gradient("group_norm has no second derivative", dy, x, mean, rstd, weight, bias, out)
    n, l, c, sn, sl = _rows(x, "x")
    _same(dy, x, "dy")
    _, _, _, dn, dl = _rows(dy, "dy")
    dx = _out(out, x)
    xn, xl = (l * c, c) if out is None else _rows(dx, "out")[3:]
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        if t.dtype != torch.float32 or t.get_device() != x.get_device() or t.shape != (n, groups) \
                or not t.is_contiguous():
            _fail(f"{what} must be contiguous float32 [{n}, {groups}] on {x.device}")
    dw, db = x.new_empty(c, dtype=torch.float32), x.new_empty(c, dtype=torch.float32)
    _work, work, size = _workspace("scb_group_norm_workspace", x, n, l, c, groups)
    _call(x, _library().scb_group_norm_backward, dy.data_ptr(), dn, dl, x.data_ptr(), sn, sl, dt, n, l, c, groups,
          mean.data_ptr(), rstd.data_ptr(), _params(weight, c, x, "weight"), _params(bias, c, x, "bias"), _act(act),
          dx.data_ptr(), xn, xl, dw.data_ptr(), db.data_ptr(), work, size)
    if out is not None:
        increment_version(out)
    return dx, dw, db


@functools.lru_cache(maxsize=256)
def _sections(sections):
    """(C array, pairs) of the axes' sections."""
    return (ctypes.c_int * len(sections))(*sections), sum(sections)


_NO_POSITIONS = "the rotation has no gradient with respect to positions and inv_freq"


def _heads(x, out, what):
    if x.dim() != 4:
        _fail(f"{what} must be [pictures, tokens, heads, channels]")
    xb, xl, xh, xd = x.stride()
    yb, yl, yh, yd = out.stride()
    if x.shape[3] > 1 and (xd != 1 or yd != 1):
        _fail(f"{what}: the channels must be contiguous")
    return ScbHeads(x.data_ptr(), out.data_ptr(), x.shape[2], xb, xl, xh, yb, yl, yh)


def rotate_axes(q, k, positions, inv_freq, sections, *, layout="half", inverse=False, out=None):
    """(q, k) rotated by their tokens' positions on 1 to 4 axes (k may be None).

    q is [b, l, h, d], k [b, l, hk, d]; positions [l, axes] or [b, l, axes], int32, int64 or
    float32; inv_freq float32 [sum(sections)]: sections[a] channel pairs turn by
    positions[..., a] * inv_freq. layout: "half" pairs channels (p, p + P), "interleaved"
    (2p, 2p + 1), "axial" the halves of each axis's own channels; channels past 2 P are
    copied. inverse=True turns back, which is the gradient. `out` is a pair of tensors, which
    may be (q, k) themselves."""
    dt = _dtype(q, "q")
    if _recording():
        _no_gradient("rotate_axes gives no gradient: use RotateAxes.apply", q, k, *(out or ()))
        if positions.requires_grad or inv_freq.requires_grad:
            _fail(_NO_POSITIONS)
    if layout not in SCB_ROT_LAYOUTS:
        _fail(f"unknown layout {layout!r}")
    if q.dim() != 4:
        _fail("q must be [pictures, tokens, heads, channels]")
    b, l, _, d = q.shape
    if k is not None and (k.dtype != q.dtype or k.get_device() != q.get_device() or k.dim() != 4
                          or k.shape[:2] != (b, l) or k.shape[3] != d):
        _fail(f"k must be [{b}, {l}, heads, {d}] {q.dtype} on {q.device}")
    axes = len(sections)
    c_sections, pairs = _sections(tuple(sections))
    if positions.dtype not in _POSITIONS or positions.get_device() != q.get_device():
        _fail(f"positions must be int32, int64 or float32 on {q.device}")
    if positions.shape == (l, axes):
        pb, (pl, pa) = 0, positions.stride()
    elif positions.shape == (b, l, axes):
        pb, pl, pa = positions.stride()
    else:
        _fail(f"positions must be [{l}, {axes}] or [{b}, {l}, {axes}], not {tuple(positions.shape)}")
    _params(inv_freq, pairs, q, "inv_freq")
    yq = _out(None if out is None else out[0], q, "out[0]")
    yk = None if k is None else _out(None if out is None else out[1], k, "out[1]")
    _call(q, _library().scb_rotate_axes, _heads(q, yq, "q"), None if k is None else _heads(k, yk, "k"), dt, b, l, d,
          positions.data_ptr(), _POSITIONS[positions.dtype], pb, pl, pa, inv_freq.data_ptr(),
          c_sections, axes, SCB_ROT_LAYOUTS[layout], bool(inverse))
    if out is not None:
        for y in (yq,) if k is None else (yq, yk):
            increment_version(y)
    return yq, yk


def attention(q, k, v, *, scale=None, key_mask=None, out=None):
    """softmax(scale q k^T over the visible keys) v, float16 or bfloat16.

    q is [b, lq, h, d], k and v [b, lk, hk, d] with d at most 256; query head i reads key head
    i / (h / hk). key_mask is bool or uint8 [b, lk], nonzero = visible: what hidden keys hold
    does not matter, and queries with no visible key give zeros (with nothing but scores of -inf
    NaN, as 0 / 0 is). scale defaults to 1 / sqrt(d). Fast (tensor cores) for d up to 128 and
    16-byte aligned rows of k and v. Forward only: there is no gradient. A lost wait on the device
    makes the rows it had a part in NaN; `status` tells."""
    dt = _dtype(q, "q")
    if _recording():
        _no_gradient("attention has no gradient", q, k, v, out)
    for t, what in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() != 4 or t.dtype != q.dtype or t.get_device() != q.get_device():
            _fail(f"{what} must be [pictures, tokens, heads, channels] {q.dtype} on {q.device}")
        if t.shape[3] > 1 and t.stride(3) != 1:
            _fail(f"{what}: the channels must be contiguous")
    b, lq, h, d = q.shape
    _, lk, hk, _ = k.shape
    if k.shape != (b, lk, hk, d) or v.shape != k.shape:
        _fail(f"k and v must be [{b}, keys, heads, {d}] alike, not {tuple(k.shape)} and {tuple(v.shape)}")
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.get_device() != q.get_device() \
                or key_mask.shape != (b, lk) or (lk > 1 and key_mask.stride(1) != 1):
            _fail(f"key_mask must be bool or uint8 [{b}, {lk}] on {q.device}, its rows contiguous")
    o = _out(out, q)
    if d > 1 and o.stride(3) != 1:
        _fail("out: the channels must be contiguous")
    rows = []
    for t in (q, k, v, o):
        sb, sl, sh, _ = t.stride()
        rows.append(ScbRows(t.data_ptr(), sb, sl, sh))
    _work, work, size = _workspace("scb_attention_workspace", q, b, lq, lk, h, hk, d)
    _call(q, _library().scb_attention, *rows, dt, b, lq, lk, h, hk, d, _ptr(key_mask),
          0 if key_mask is None else key_mask.stride(0), d ** -0.5 if scale is None else scale, work, size)
    if out is not None:
        increment_version(out)
    return o


def status(stream=None):
    """Wait for the stream (default: the current one) and raise if an operator's kernel gave up
    on a bounded wait since the last call. The operators themselves do not wait: call this where
    the program waits anyway."""
    stream = stream or torch.cuda.current_stream()
    with torch.cuda.device(stream.device):
        if _library().scb_op_status(stream.cuda_stream) != 0:
            _fail(_library().scb_last_error(None).decode())


class GroupNormAct(torch.autograd.Function):
    """group_norm under autograd: GroupNormAct.apply(x, groups, weight, bias, eps, act). It has
    no second derivative: differentiating its gradient raises RuntimeError."""

    @staticmethod
    def forward(ctx, x, groups, weight, bias, eps=1e-5, act="none"):
        y, mean, rstd = group_norm(x, groups, weight, bias, eps=eps, act=act, stats=True)
        ctx.save_for_backward(x, mean, rstd, weight, bias)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, weight, bias = ctx.saved_tensors
        dy = dy.contiguous()  # a gradient may come broadcast
        dx, dw, db = group_norm_backward(dy, x, mean, rstd, ctx.groups, weight, bias, act=ctx.act)
        return dx, None, dw if weight is not None else None, db if bias is not None else None, None, None


class RotateAxes(torch.autograd.Function):
    """rotate_axes under autograd: RotateAxes.apply(q, k, positions, inv_freq, sections, layout,
    inverse). Its gradient is the rotation by the opposite angles, under autograd again, so it
    has derivatives of every order."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, sections, layout="half", inverse=False):
        ctx.save_for_backward(positions, inv_freq)
        ctx.sections, ctx.layout, ctx.inverse = tuple(sections), layout, bool(inverse)
        return rotate_axes(q, k, positions, inv_freq, sections, layout=layout, inverse=inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
            _fail(_NO_POSITIONS)
        dk = None if dk is None else dk.contiguous()  # there was no k
        dq, dk = RotateAxes.apply(dq.contiguous(), dk, positions, inv_freq, ctx.sections, ctx.layout, not ctx.inverse)
        return dq, dk, None, None, None, None, None
