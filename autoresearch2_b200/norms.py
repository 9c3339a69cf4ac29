"""RMS norms before and after a block, fused with its gate and residual add.

    residual_norm(x, y, pre_weight=, post_weight=, gate=, post_norm=, residual_scale=, eps=)
        -> (x_new, h)

    x_new = residual_scale * x + gate * (rms(y) * post_weight  or  y)
    h     = rms(x_new) * pre_weight          rms(v) = v / sqrt(mean(v^2) + eps)

x is the residual stream, y the output of the block that was fed h, and the
new h feeds the next block: one kernel reads x and y and writes x_new and h.
The backward recomputes x_new from x and y (no copy of either is kept) and
gives every gradient in one pass plus a small join of the weight gradients,
whose order of addition is fixed: equal inputs give equal bits.  Forward-mode
tangents and second derivatives are refused.
"""
import math

import torch

from . import _lib
from ._lib import address as ptr
from ._lib import call, stream_handle

__all__ = ["residual_norm", "WIDTH_MAX"]

WIDTH_MAX = 16384  # elements of a row
F32_MAX = torch.finfo(torch.float32).max


def _matrix(t, width):
    """t as [rows, width] with dense rows (a view where the strides allow one)."""
    t = t.reshape(-1, width) if t.dim() != 2 else t
    return t if width == 1 or t.stride(1) == 1 else t.contiguous()


def _check_groups(x, gate, groups):
    """The ops' way to say what _gate_groups found."""
    rows = x.numel() // x.shape[-1]
    if groups < 1 or (rows and rows % groups) or (gate is not None and rows and gate.numel() != groups * x.shape[-1]):
        raise ValueError(f"a gate of {groups} rows does not divide {rows} rows evenly")


def _check_backward(x, y, dx_new, dh, stats, out_dtype):
    for name, t, like, dtype in (("dx_new", dx_new, x, x.dtype), ("dh", dh, x, out_dtype)):
        if t is not None and (t.shape != like.shape or t.dtype != dtype or t.device != x.device):
            raise ValueError(f"{name} must be {dtype} of shape {tuple(like.shape)} on {x.device}")
    if (stats.numel() != 2 * (x.numel() // x.shape[-1]) or stats.dtype != torch.float32 or not stats.is_contiguous()
            or stats.device != x.device):
        raise ValueError(f"stats are the forward's: float32, contiguous, two a row, on {x.device}")


def _empty(t, dtype=None):
    """Contiguous, of t's shape (two thirds of the time that new_empty takes)."""
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _code(t):
    return _lib._DTYPES[t.dtype] if t is not None else 0


def _gate_groups(gate, x):
    """Runs of equal length into which the gate's rows split x's rows."""
    rows = x.numel() // x.shape[-1]
    if gate.shape[-1:] != x.shape[-1:]:
        raise ValueError(f"gate's last dimension must be {x.shape[-1]}, got shape {tuple(gate.shape)}")
    if gate.dim() == 1:
        return 1
    groups = math.prod(gate.shape[:-1])
    if gate.dim() == 2:
        if groups < 1 or rows % groups:
            raise ValueError(f"a gate of {groups} rows does not divide {rows} rows evenly")
        return groups
    lead = gate.shape[:-1]
    while lead and lead[-1] == 1:
        lead = lead[:-1]
    if gate.dim() != x.dim() or lead != x.shape[:len(lead)]:
        raise ValueError(f"gate {tuple(gate.shape)} must be x's leading dimensions {tuple(x.shape[:-1])} up to some "
                         "dimension, ones after it, then the width")
    return groups


def _forward(x, y, pre, post, gate, groups, post_norm, scale, eps, out_dtype, keep):
    """(x_new or None, h, stats or None)."""
    width, codes = x.shape[-1], _lib._DTYPES
    x2 = _matrix(x, width)
    rows, dev = x2.shape[0], x.device
    x_new, py, y_ld = None, None, 0
    if y is not None:
        y2 = _matrix(y, width)
        x_new, py, y_ld = _empty(x), y2.data_ptr(), y2.stride(0)
    h = _empty(x, out_dtype)
    stats = x.new_empty((rows, 2), dtype=torch.float32) if keep else None
    if rows:
        pre, post, gate = _dense(pre), _dense(post), _dense(gate)
        call("sffn_residual_norm", x2.data_ptr(), codes[x.dtype], x2.stride(0), py, codes[out_dtype], y_ld, rows, width,
             ptr(pre), _code(pre), ptr(post), _code(post), ptr(gate), _code(gate), rows // groups, int(post_norm), scale,
             eps, ptr(x_new), h.data_ptr(), ptr(stats), _lib.status_word(dev).data_ptr(), stream_handle(dev))
    return x_new, h, stats


def _backward(x, y, pre, post, gate, groups, post_norm, scale, out_dtype, stats, dx_new, dh, want):
    """Gradients of (x, y, pre, post, gate); None where `want` is false."""
    _lib.bind_thread(x.device)
    width, codes = x.shape[-1], _lib._DTYPES
    x2 = _matrix(x, width)
    rows, dev = x2.shape[0], x.device
    py, y_ld, dy = None, 0, None
    if y is not None:
        y2 = _matrix(y, width)
        py, y_ld = y2.data_ptr(), y2.stride(0)
        dy = _empty(y) if want[1] else None
    dx = _empty(x) if want[0] else None
    dpre = _empty(pre) if pre is not None and want[2] else None
    dpost = _empty(post) if post is not None and want[3] else None
    dgate = _empty(gate) if gate is not None and want[4] else None
    if not rows:
        for g in (dpre, dpost, dgate):
            if g is not None:
                g.zero_()
        return dx, dy, dpre, dpost, dgate
    pre, post, gate, dx_new, dh = _dense(pre), _dense(post), _dense(gate), _dense(dx_new), _dense(dh)
    ws, ws_bytes = None, 0
    if dpre is not None or dpost is not None or dgate is not None:
        per = rows // groups if dpost is not None or dgate is not None else 0
        ws_bytes = _lib.load().sffn_residual_norm_bwd_workspace_bytes(rows, width, per)
        ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    call("sffn_residual_norm_bwd", x2.data_ptr(), codes[x.dtype], x2.stride(0), py, codes[out_dtype], y_ld, rows, width,
         ptr(pre), _code(pre), ptr(post), _code(post), ptr(gate), _code(gate), rows // groups, int(post_norm), scale,
         stats.data_ptr(), ptr(dx_new), ptr(dh), ptr(dx), ptr(dy), ptr(dpre), ptr(dpost), ptr(dgate), ptr(ws), ws_bytes,
         _lib.status_word(dev).data_ptr(), stream_handle(dev))
    return dx, dy, dpre, dpost, dgate


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, pre, post, gate, groups, post_norm, scale, eps, out_dtype):
        x_new, h, stats = _forward(x, y, pre, post, gate, groups, post_norm, scale, eps, out_dtype, True)
        ctx.save_for_backward(x, y, pre, post, gate, stats)
        ctx.args = groups, post_norm, scale, out_dtype
        ctx.set_materialize_grads(False)
        return x_new, h

    @staticmethod
    def backward(ctx, dx_new, dh):
        _lib.once_differentiable("residual_norm")
        x, y, pre, post, gate, stats = ctx.saved_tensors
        groups, post_norm, scale, out_dtype = ctx.args
        grads = _backward(x, y, pre, post, gate, groups, post_norm, scale, out_dtype, stats, dx_new, dh,
                          ctx.needs_input_grad[:5])
        return *grads, None, None, None, None, None


def _check(x, y, pre_weight, post_weight, gate, post_norm, residual_scale, eps, out_dtype):
    """h's type, of arguments that are refused otherwise (the gate's rows: _gate_groups)."""
    for t in (x, y, pre_weight, post_weight, gate):
        if t is not None:
            _lib.require_cuda(t)
            _lib.dtype_code(t)
            if t.device != x.device:
                raise ValueError(f"a tensor is on {t.device}, x on {x.device}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= WIDTH_MAX:
        raise ValueError(f"residual_norm takes x [..., D] with 1 <= D <= {WIDTH_MAX}, got {tuple(x.shape)}")
    if y is None:
        if post_norm or post_weight is not None or gate is not None or residual_scale != 1.0:
            raise ValueError("post_norm, post_weight, gate and residual_scale go with a block output y")
        out_dtype = x.dtype if out_dtype is None else out_dtype
    else:
        if y.shape != x.shape:
            raise ValueError(f"y must have x's shape {tuple(x.shape)}, got {tuple(y.shape)}")
        if out_dtype not in (None, y.dtype):
            raise TypeError(f"h has y's type {y.dtype}; out_dtype is for calls without y")
        out_dtype = y.dtype
    if out_dtype != x.dtype and (out_dtype not in _lib._DTYPES or x.dtype != torch.float32):
        raise TypeError(f"x is {x.dtype}: h may be of the same type, or x float32 and h bfloat16 or float16")
    for name, t in (("pre_weight", pre_weight), ("post_weight", post_weight)):
        if t is not None and t.shape != x.shape[-1:]:
            raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(t.shape)}")
    if post_weight is not None and not post_norm:
        raise ValueError("post_weight goes with post_norm=True")
    if not (abs(residual_scale) <= F32_MAX and 2.0 ** -126 <= eps <= F32_MAX):
        raise ValueError(f"residual_scale must be finite and eps positive, got {residual_scale!r}, {eps!r}")
    return out_dtype


def residual_norm(x, y=None, pre_weight=None, post_weight=None, gate=None, post_norm=False, residual_scale=1.0,
                  eps=1e-6, out_dtype=None):
    """(x_new, h): the residual stream after a block, and its norm for the next.

    x [..., D], D <= 16384; y of x's shape, or None (the first norm of a stack:
    x_new is x itself).  x and y share a type, or x is float32 and y bfloat16
    or float16; x_new has x's type and h y's (out_dtype, or x's, without y).
    pre_weight and post_weight [D] (post_weight only with post_norm) and gate
    may each have any of the three types, and None for ones.

    gate is [D]; or [G, D], each row for one of G equal runs of x's rows; or
    x's leading dimensions up to some one, then ones, then D (for x [B, T, D]
    one gate a sequence is [B, 1, D]).  A [G, D] gate is not broadcast against
    x's last two dimensions.

    Rows are read in place where one stride fits them all.  Arithmetic,
    statistics and sums are float32 (the blocks' sums of a weight gradient 64
    bits), each output is rounded once; h comes from the unrounded x_new."""
    out_dtype = _check(x, y, pre_weight, post_weight, gate, post_norm, residual_scale, eps, out_dtype)
    groups = _gate_groups(gate, x) if gate is not None and x.numel() else 1
    args = (x, y, pre_weight, post_weight, gate, groups, bool(post_norm), float(residual_scale), float(eps), out_dtype)
    if torch.compiler.is_compiling():
        x_new, h, _ = torch.ops.sparseffn.residual_norm(*args)
    elif _lib.tracked(*args[:5]):
        x_new, h = _ResidualNorm.apply(*args)
    else:
        x_new, h, _ = _forward(*args, False)
    return (x_new if y is not None else x), h
