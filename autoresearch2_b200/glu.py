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
import functools

import torch

from . import _lib, fp8
from ._lib import address as ptr
from ._lib import call, stream_handle
from .parallel import current, submit_grad

__all__ = ["ACTIVATIONS", "gated_ffn"]

ACTIVATIONS = {"relu": 0, "relu2": 1, "silu": 2, "gelu": 3}
KEEP = {None: 1, "fp8": 2}
DGRAD, DW2, DWGU, DX = 1, 2, 4, 8  # steps of the backward
JOINT, APART = 16, 32  # dWg and dWu as one product, or as two


def _kept_ld(F, keep):
    return (F + 15) // 16 * 16 if keep == 2 else (F + 7) // 8 * 8


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(backward, keep, odd, want, T, D, F):
    return _lib.load().sffn_gated_ffn_workspace_bytes(backward, keep, odd, want, T, D, F)


def _forward(x, Wg, Wu, W2, act, keep):
    """(y, g, u, g_tiles, u_tiles, x_values, x_tiles): keep 0 keeps nothing, 1 g
    and u in x's type, 2 all three in 8 bits; what is not kept is None."""
    x2, Wg, Wu, W2 = fp8._rows(x), fp8._rows(Wg), fp8._rows(Wu), fp8._rows(W2)
    T, D = x2.shape
    F, dev = Wg.shape[0], x.device
    g = u = gt = ut = xv = xt = None
    if keep == 2:
        g, u, xv = fp8._empty_values(T, F, dev), fp8._empty_values(T, F, dev), fp8._empty_values(T, D, dev)
        gt, ut, xt = fp8._empty_tiles(T, F, dev), fp8._empty_tiles(T, F, dev), fp8._empty_tiles(T, D, dev)
    elif keep == 1:
        g, u = fp8._empty_rows(x2, T, F, 8), fp8._empty_rows(x2, T, F, 8)
    y = x2.new_empty((T, D))
    if T:
        (ldx, ox), (ldg, og), (ldu, ou), (ld2, o2) = (fp8._row_stride(x2, 1), fp8._row_stride(Wg, 2),
                                                      fp8._row_stride(Wu, 4), fp8._row_stride(W2, 8))
        odd = ox | og | ou | o2
        n = _workspace_bytes(0, keep, odd, 0, T, D, F)
        ws = fp8._workspace(n, dev)
        call("sffn_gated_ffn", _lib._DTYPES[x.dtype], act, keep, x2.data_ptr(), ldx, Wg.data_ptr(), ldg, Wu.data_ptr(), ldu,
             W2.data_ptr(), ld2, odd, T, D, F, y.data_ptr(), ptr(g), ptr(u), ptr(gt), ptr(ut), ptr(xv), ptr(xt), ptr(ws), n,
             _lib.status_word(dev).data_ptr(), stream_handle(dev))
    return (y if x.dim() == 2 else y.view(x.shape)), g, u, gt, ut, xv, xt


def _backward(dy, x, Wg, Wu, W2, g, u, gt, ut, xv, xt, act, want, apart=False):
    """Gradients of (x, Wg, Wu, W2); None where `want` is false.  x is None with 8-bit
    checkpoints.  apart: dWg and dWu do not share their storage."""
    dev = dy.device
    _lib.bind_thread(dev)
    dy2, Wg, Wu, W2 = fp8._rows(dy), fp8._rows(Wg), fp8._rows(Wu), fp8._rows(W2)
    T, D = dy2.shape
    F, keep = Wg.shape[0], 1 if xv is None else 2
    dx = dWg = dWu = dW2 = None
    if want[0]:
        dx = dy2.new_empty(dy.shape)
    if not T:
        return (dx, *(submit_grad(w.new_zeros(w.shape)) if n else None for w, n in zip((Wg, Wu, W2), want[1:])))
    how = APART
    if want[1] and want[2] and not apart:  # one product, rows of dWu after F rounded up to 8 of dWg
        ld = (F + 7) // 8 * 8
        both = dy2.new_empty((2 * ld, D))
        dWg, dWu = both[:F], both[ld:ld + F]
        how = JOINT
    else:
        dWg, dWu = (dy2.new_empty((F, D)) if w else None for w in want[1:3])
    if want[3]:
        dW2 = dy2.new_empty((D, F))
    x2, (ldx, ox) = None, (0, 0)
    if keep == 1:
        x2 = fp8._rows(x)
        ldx, ox = fp8._row_stride(x2, 16)
    (ldy, oy), (ldg, og), (ldu, ou), (ld2, o2) = (fp8._row_stride(dy2, 1), fp8._row_stride(Wg, 2), fp8._row_stride(Wu, 4),
                                                  fp8._row_stride(W2, 8))
    odd = oy | og | ou | o2 | ox
    n = _workspace_bytes(1, keep, odd, want[0] + 2 * want[1] + 4 * want[2] + 8 * want[3], T, D, F)
    ws = fp8._workspace(n, dev)
    code, status, stream = _lib._DTYPES[dy.dtype], _lib.status_word(dev).data_ptr(), stream_handle(dev)

    def run(steps):
        call("sffn_gated_ffn_bwd", code, act, keep, steps | how, dy2.data_ptr(), ldy, ptr(x2), ldx, Wg.data_ptr(), ldg, Wu.data_ptr(),
             ldu, W2.data_ptr(), ld2, odd, g.data_ptr(), u.data_ptr(), ptr(gt), ptr(ut), ptr(xv), ptr(xt), T, D, F, ptr(dx),
             ptr(dWg), ptr(dWu), ptr(dW2), ptr(ws), n, status, stream)

    if current() is None:
        run(DGRAD | DW2 | DWGU | DX)
    else:  # each weight gradient's reduction beside what follows it
        run(DGRAD | DW2)
        submit_grad(dW2)
        run(DWGU)
        submit_grad(dWg)
        submit_grad(dWu)
        run(DX)
    return dx, dWg, dWu, dW2


def _as_kept(dy, x, F, g, u, gt, ut, xv, xt):
    """(x, g, u, g_tiles, u_tiles, x_values, x_tiles) on the strides that the kernels read,
    which a forward gives them and a copy by saved-tensor hooks does not; refused
    where they are not what was kept.  x is None with 8-bit checkpoints, the
    last four without."""
    rows, D, dev = dy.numel() // dy.shape[-1], dy.shape[-1], dy.device
    if x is None:
        kept = fp8._kept_rows
        return (None, kept(g, rows, F, fp8.E4M3, dev, 16), kept(u, rows, F, fp8.E4M3, dev, 16), fp8._kept_tiles(gt, rows, F, dev),
                fp8._kept_tiles(ut, rows, F, dev), kept(xv, rows, D, fp8.E4M3, dev, 16), fp8._kept_tiles(xt, rows, D, dev))
    if x.shape != dy.shape or x.dtype is not dy.dtype or x.device != dev:
        raise ValueError(f"the kept x must be {dy.dtype} {tuple(dy.shape)} on {dev}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x, *(fp8._kept_rows(t, rows, F, dy.dtype, dev, 8) for t in (g, u)), None, None, None, None


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
        x, Wg, Wu, W2, *kept = ctx.saved_tensors
        _check(dy, Wg, Wu, W2)
        x, *kept = _as_kept(dy, x, Wg.shape[0], *kept)
        return *_backward(dy, x, Wg, Wu, W2, *kept, ctx.act, ctx.needs_input_grad[:4]), None, None


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
    to 16 rows (64 where the weights' rows are on 16 bytes) then take the few-row
    kernels.  Weight gradients are handed to an
    attached parallel.GradAllReduce as they are produced; those of Wg and Wu share
    one storage where both are wanted (clone one to keep or save it alone).
    h, dg and du are rounded to the inputs' type: in float16 they overflow beyond
    65504 ("relu2" soon does) and lose digits below 6e-5, so scale the loss there
    as for any float16 layer.  Differentiable once, in reverse mode."""
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
