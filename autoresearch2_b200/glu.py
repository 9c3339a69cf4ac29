"""The gated feed-forward block, forward and backward.

    gated_ffn(x, Wg, Wu, W2, activation="silu", checkpoint=None)

    g = x Wg^T, u = x Wu^T, h = act(g) * u, y = h W2^T

One kernel computes both projections, the activation and the product; g and u
never make a trip through memory on the way to h.  The backward works from x, g
and u as the forward kept them -- in the inputs' type, or with
checkpoint="fp8" in the 8-bit block format of fp8.py, half the bytes:

    dh = dy W2, dg = dh * u * act'(g), du = dh * act(g)
    dW2 = dy^T (act(g) * u), dWg = dg^T x, dWu = du^T x, dx = dg Wg + du Wu

dh's kernel reads g and u and writes dg, du and act(g) * u; dx is one product
over both pairs.  Products sum in float32; h, dg and du are rounded to the
inputs' type, in which the tensor cores read them.
"""
import torch

from . import _lib, fp8
from ._lib import address as ptr
from ._lib import call, stream_handle
from .parallel import submit_grad

__all__ = ["ACTIVATIONS", "gated_ffn"]

ACTIVATIONS = {"relu": 0, "relu2": 1, "silu": 2, "gelu": 3}
KEEP = {None: 1, "fp8": 2}


def _kept_ld(F, keep):
    return (F + 15) // 16 * 16 if keep == 2 else (F + 7) // 8 * 8


def _forward(x, Wg, Wu, W2, act, keep):
    """(y, g, u, g_tiles, u_tiles, x_values, x_tiles): keep 0 keeps nothing, 1 g
    and u in x's type, 2 all three in 8 bits; what is not kept is None."""
    x2, Wg, Wu, W2 = fp8._rows(x), fp8._rows(Wg), fp8._rows(Wu), fp8._rows(W2)
    T, D = x2.shape
    F, dev, code = Wg.shape[0], x.device, _lib._DTYPES[x.dtype]
    g = u = gt = ut = xv = xt = None
    if keep == 0 and 0 < T <= fp8.FEW_ROWS:
        h, y = x2.new_empty((T, (F + 7) // 8 * 8)), x2.new_empty((T, D))
        call("sffn_few_rows_ffn", code, act, x2.data_ptr(), fp8._ld(x2), Wg.data_ptr(), fp8._ld(Wg), Wu.data_ptr(),
             fp8._ld(Wu), W2.data_ptr(), fp8._ld(W2), T, D, F, h.data_ptr(), h.shape[1], y.data_ptr(), D,
             _lib.status_word(dev).data_ptr(), stream_handle(dev))
        return y if x.dim() == 2 else y.view(x.shape), g, u, gt, ut, xv, xt
    if keep == 2:
        g, u = (fp8._empty_values(T, F, dev) for _ in range(2))
        gt, ut = (fp8._empty_tiles(T, F, dev) for _ in range(2))
    elif keep == 1:
        g, u = (fp8._empty_rows(x2, T, F, 8) for _ in range(2))
    if T == 0:
        if keep == 2:
            xv, xt = fp8._pack(x2)
        return x.new_empty(x.shape), g, u, gt, ut, xv, xt
    if T <= fp8.FEW_ROWS:  # kept, so the tensor cores' tiles: W2's product is the few-row kernel's
        xa, ga, ua = fp8._align(x2, Wg, Wu)
    else:
        xa, ga, ua, W2a = fp8._align(x2, Wg, Wu, W2)
    h = fp8._empty_rows(x2, T, F, 8)
    ldh = (F + 7) // 8 * 8
    call("sffn_glu_up", code, act, xa[0].data_ptr(), xa[1], ga[0].data_ptr(), ga[1], ua[0].data_ptr(), ua[1], T, D, F,
         h.data_ptr(), ldh, keep, ptr(g), ptr(u), _kept_ld(F, keep), ptr(gt), ptr(ut),
         _lib.status_word(dev).data_ptr(), stream_handle(dev))
    if T <= fp8.FEW_ROWS:
        y = fp8._few_rows(h, W2)
    else:
        y = fp8._mm_into(x2.new_empty((T, D)), (h, ldh), 0, W2a, 0)
    if keep == 2:
        xv, xt = fp8._pack(xa[0])
    return y if x.dim() == 2 else y.view(x.shape), g, u, gt, ut, xv, xt


def _backward(dy, x, Wg, Wu, W2, g, u, gt, ut, xv, xt, act, want, apart=False):
    """Gradients of (x, Wg, Wu, W2); None where `want` is false.  x is None with 8-bit
    checkpoints.  apart: dWg and dWu do not share their storage."""
    _lib.bind_thread(dy.device)
    dy2, Wg, Wu, W2 = fp8._rows(dy), fp8._rows(Wg), fp8._rows(Wu), fp8._rows(W2)
    T, D = dy2.shape
    F, dev, code = Wg.shape[0], dy.device, _lib._DTYPES[dy.dtype]
    dx = dWg = dWu = dW2 = None
    if T == 0:
        return (dy.new_empty(dy.shape) if want[0] else None,
                *(submit_grad(w.new_zeros(w.shape)) if n else None for w, n in zip((Wg, Wu, W2), want[1:])))
    keep = 2 if xv is not None else 1
    ld = (F + 7) // 8 * 8
    d, h = dy2.new_empty((T, 2 * ld)), fp8._empty_rows(dy2, T, F, 8)  # d: dg | du, their weights' gradient is one product
    dg, du = (d[:, :F], 2 * ld), (d[:, ld:ld + F], 2 * ld)
    if want[0]:
        dya, W2a, ga, ua = fp8._align(dy2, W2, Wg, Wu)
    else:
        dya, W2a = fp8._align(dy2, W2)
    call("sffn_glu_dgrad", code, act, dya[0].data_ptr(), dya[1], W2a[0].data_ptr(), W2a[1], T, D, F, keep, g.data_ptr(),
         u.data_ptr(), _kept_ld(F, keep), ptr(gt), ptr(ut), dg[0].data_ptr(), du[0].data_ptr(), 2 * ld, h.data_ptr(), ld,
         _lib.status_word(dev).data_ptr(), stream_handle(dev))
    if want[3]:
        dW2 = submit_grad(fp8._mm_into(dy2.new_empty((D, F)), dya, 1, (h, ld), 1))
    del h
    if want[1] or want[2]:
        if keep == 2:
            xk = fp8._unpack(xv, xt, fp8._empty_rows(dy2, T, D, 8), D), (D + 7) // 8 * 8
        else:
            xk, = fp8._align(fp8._rows(x))
        if want[1] and want[2] and not apart:
            dW = fp8._mm_into(dy2.new_empty((2 * ld, D)), (d, 2 * ld), 1, xk, 1)
            dWg, dWu = submit_grad(dW[:F]), submit_grad(dW[ld:ld + F])
        else:
            dWg = submit_grad(fp8._mm_into(dy2.new_empty((F, D)), dg, 1, xk, 1)) if want[1] else None
            dWu = submit_grad(fp8._mm_into(dy2.new_empty((F, D)), du, 1, xk, 1)) if want[2] else None
        del xk
    if want[0]:
        dx = fp8._mm_into(dy2.new_empty((T, D)), dg, 0, ga, 1, (du, ua)).view(dy.shape)
    return dx, dWg, dWu, dW2


def _check_kept(dy, x, F, g, u, gt, ut, xv, xt):
    """The backward op's: what it is given is what a forward keeps."""
    rows, D = dy.numel() // dy.shape[-1], dy.shape[-1]
    if x is not None:
        ok = x.shape == dy.shape and x.dtype == dy.dtype and x.device == dy.device and all(
            t.shape == (rows, F) and t.dtype == dy.dtype and t.device == dy.device and t.data_ptr() % 16 == 0
            and (rows <= 1 or t.stride() == (_kept_ld(F, 1), 1)) for t in (g, u))
    else:
        ok = True
        for v, t, width in ((g, gt, F), (u, ut, F), (xv, xt, D)):
            fp8.Fp8Tensor(v, t)
            ok = ok and v.shape == (rows, width) and v.device == dy.device and (rows <= 1 or v.stride(0) == _kept_ld(width, 2))
    if not ok:
        raise ValueError("x, g and u are not as the forward kept them")


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, Wg, Wu, W2, act, keep):
        y, *kept = _forward(x, Wg, Wu, W2, act, keep)
        ctx.save_for_backward(x if keep == 1 else None, Wg, Wu, W2, *kept)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, dy):
        _lib.once_differentiable("gated_ffn")
        return *_backward(dy, *ctx.saved_tensors, ctx.act, ctx.needs_input_grad[:4]), None, None


def _check(x, Wg, Wu, W2):
    _lib.require_cuda(x, Wg, Wu, W2)
    D = x.shape[-1] if x.dim() else 0
    F = Wg.shape[0] if Wg.dim() else 0
    if not (x.dtype in fp8.OUT_TYPES and D and F and fp8._fits(x, Wg, F, D) and fp8._fits(x, Wu, F, D)
            and fp8._fits(x, W2, D, F)):
        fp8._check_weights(x, Wg=(Wg, (F, D)), Wu=(Wu, (F, D)), W2=(W2, (D, F)))


def gated_ffn(x, Wg, Wu, W2, activation="silu", checkpoint=None):
    """y [..., D] of x [..., D], Wg and Wu [F, D], W2 [D, F] (nn.Linear layout),
    all bfloat16 or all float16.

    activation: "silu", "gelu" (exact), "relu" or "relu2".  checkpoint=None keeps
    x, x Wg^T and x Wu^T for the backward in their type, "fp8" in 8 bits; the
    output is the same.  Nothing is kept where no gradient is wanted; calls of up
    to 32 rows then take the few-row kernels.  Weight gradients are handed to an
    attached parallel.GradAllReduce as they are produced.  Differentiable once,
    in reverse mode."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if checkpoint not in KEEP:
        raise ValueError(f"checkpoint must be None or 'fp8', got {checkpoint!r}")
    _check(x, Wg, Wu, W2)
    act, keep = ACTIVATIONS[activation], KEEP[checkpoint]
    tracked = _lib.tracked(x, Wg, Wu, W2)
    if torch.compiler.is_compiling():
        return torch.ops.sparseffn.gated_ffn(x, Wg, Wu, W2, act, keep if tracked else 0)[0]
    if tracked:
        return _GatedFFN.apply(x, Wg, Wu, W2, act, keep)
    return _forward(x, Wg, Wu, W2, act, 0)[0]
