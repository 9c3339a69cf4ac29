"""Matrices in 8 bits: activations kept between forward and backward, and products.

    fp8_pack(x) -> Fp8Tensor            fp8_unpack(q, dtype) -> tensor
    fp8_matmul(a, b, out_dtype=)        a b^T of two of them
    ckpt_linear(x, W)                   y = x W^T, keeping x in 8 bits

The format: float8_e4m3fn values and one power-of-two scale for each 128
elements of a row: 2^e with the smallest integer e such that the block's largest
finite magnitude is at most 448 * 2^e, e >= -118 (1 for a block of zeros).
Values are rounded once, to nearest, ties to even; infinities and NaN become
NaN.  A power of two adds no rounding, dequantised values are exact in bfloat16
and float32, and the tensor cores apply such scales themselves.
"""
import functools

import torch

from . import _lib
from ._lib import address as ptr
from ._lib import call, stream_handle
from .parallel import current, submit_grad

__all__ = ["BLOCK", "Fp8Tensor", "fp8_pack", "fp8_unpack", "fp8_matmul", "ckpt_linear"]

BLOCK = 128
E4M3 = torch.float8_e4m3fn
FEW_ROWS = 64  # products of at most so many rows go by the few-row kernels
OUT_TYPES = (torch.bfloat16, torch.float16)


def _cdiv(a, b):
    return -(-a // b)


class Fp8Tensor:
    """A tensor in the 8-bit block format.

    values       float8_e4m3fn [rows, width], rows dense and 16 bytes apart in
                 multiples (a view of wider rows where width is not one)
    scale_tiles  uint8 [rows/128, blocks/4, 32, 4, 4], rounded up: the exponent
                 byte e + 127 of row r, block k at
                 [r // 128, k // 4, r % 32, r % 128 // 32, k % 4]
    shape        of the tensor it stands for, [..., width]
    """

    __slots__ = ("values", "scale_tiles", "shape")

    def __init__(self, values, scale_tiles, shape=None):
        if values.dtype != E4M3 or values.dim() != 2 or values.shape[1] < 1:
            raise ValueError(f"values must be float8_e4m3fn [rows, width], got {values.dtype} {tuple(values.shape)}")
        rows, width = values.shape
        if width > 1 and values.stride(1) != 1 or rows > 1 and (values.stride(0) % 16 or values.stride(0) < width):
            raise ValueError("values must have dense rows, a multiple of 16 bytes apart")
        want = _tile_shape(rows, width)
        if scale_tiles.dtype != torch.uint8 or tuple(scale_tiles.shape) != want or not scale_tiles.is_contiguous():
            raise ValueError(f"scale_tiles must be uint8 {want}, contiguous")
        if scale_tiles.device != values.device:
            raise ValueError(f"scale_tiles are on {scale_tiles.device}, values on {values.device}")
        shape = torch.Size((rows, width) if shape is None else shape)
        if not shape or shape[-1] != width or shape.numel() != rows * width:
            raise ValueError(f"shape {tuple(shape)} is not {rows} rows of {width}")
        self.values, self.scale_tiles, self.shape = values, scale_tiles, shape

    @property
    def device(self):
        return self.values.device

    @property
    def exponents(self):
        """e of every block, int32 [rows, blocks]."""
        rows, width = self.values.shape
        t = self.scale_tiles.permute(0, 3, 2, 1, 4).reshape(self.scale_tiles.shape[0] * 128, -1)
        return t[:rows, :_cdiv(width, BLOCK)].int() - 127

    def to_dense(self, dtype=torch.bfloat16):
        return fp8_unpack(self, dtype)

    def vram_size(self):
        """Bytes held."""
        return self.values.shape[0] * _stride(self.values) + self.scale_tiles.numel()

    def __repr__(self):
        return f"Fp8Tensor(shape={tuple(self.shape)}, device={self.device})"


def _tile_shape(rows, width):
    return (rows + 127) // 128, (width + 511) // 512, 32, 4, 4


def _stride(values):
    """Bytes between rows (one row's stride says nothing)."""
    return values.stride(0) if values.shape[0] > 1 else _cdiv(values.shape[1], 16) * 16


def _rows(t):
    """t as [rows, width] with dense rows (a view where the strides allow one)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t
    rows, width = t.shape
    dense = (width == 1 or t.stride(1) == 1) and (rows <= 1 or t.stride(0) >= width)
    return t if dense else t.contiguous()


def _ld(t):
    """Elements between the rows of a matrix with dense rows."""
    rows, width = t.shape
    return t.stride(0) if rows > 1 else width


def _row_stride(t, bit):
    """(row stride, bit if the matrix's rows are not on 16 bytes, as TMA reads them) of a
    16-bit matrix with dense rows."""
    rows, width = t.shape
    ld = t.stride(0) if rows > 1 else width
    return ld, bit if t.data_ptr() % 16 or (rows > 1 and ld % 8) else 0


def _empty_rows(t, rows, cols, multiple):
    """[rows, cols] of t's type, its rows padded to a multiple of so many elements."""
    ld = -(-cols // multiple) * multiple
    out = t.new_empty((rows, ld))
    return out if ld == cols else out.narrow(1, 0, cols)


def _empty_values(rows, width, device, multiple=16):
    ld = -(-width // multiple) * multiple
    out = torch.empty((rows, ld), dtype=E4M3, device=device)
    return out if ld == width else out.narrow(1, 0, width)


def _empty_tiles(rows, width, device):
    return torch.empty(_tile_shape(rows, width), dtype=torch.uint8, device=device)


def _kept_rows(t, rows, width, dtype, device, multiple):
    """A matrix that a forward kept, its rows padded to a multiple of so many elements.
    Saved-tensor hooks (save_on_cpu and the like) may give back a dense copy,
    which is laid out again; what is not that matrix is refused."""
    if t.shape != (rows, width) or t.dtype is not dtype or t.device != device:
        raise ValueError(f"a kept tensor must be {dtype} {(rows, width)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    ld = -(-width // multiple) * multiple
    if (rows <= 1 or t.stride(0) == ld) and (width <= 1 or t.stride(1) == 1) and t.data_ptr() % 16 == 0:
        return t
    return t.new_empty((rows, ld)).narrow(1, 0, width).copy_(t)


def _kept_tiles(t, rows, width, device):
    if t.shape != _tile_shape(rows, width) or t.dtype is not torch.uint8 or t.device != device:
        raise ValueError(f"kept scale_tiles must be uint8 {_tile_shape(rows, width)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.contiguous()


def _pack(x):
    """(values, scale tiles) of x [..., width]."""
    x2 = _rows(x)
    rows, width = x2.shape
    dev = x.device
    values, tiles = _empty_values(rows, width, dev), _empty_tiles(rows, width, dev)
    if rows:
        call("sffn_fp8_pack", x2.data_ptr(), _lib._DTYPES[x.dtype], rows, width, _ld(x2), values.data_ptr(),
             -(-width // 16) * 16, tiles.data_ptr(), stream_handle(dev))
    return values, tiles


def _unpack(values, tiles, out, width):
    """Into out, whose rows are dense; returns it."""
    rows = values.shape[0]
    if rows:
        ldo = out.stride(0) if out.dim() == 2 and rows > 1 else width
        call("sffn_fp8_unpack", values.data_ptr(), _stride(values), tiles.data_ptr(), rows, width, _lib._DTYPES[out.dtype],
             out.data_ptr(), ldo, stream_handle(values.device))
    return out


def _check_pack(x):
    _lib.require_cuda(x)
    _lib.dtype_code(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"the 8-bit format takes [..., width] with width >= 1, got {tuple(x.shape)}")


def _refuse_grad(name, *tensors):
    if _lib.tracked(*tensors):
        raise RuntimeError(f"{name} has no gradient: detach its input or call it under torch.no_grad()")


def fp8_pack(x):
    """x [..., width] (float32, bfloat16 or float16, any strides) as an Fp8Tensor."""
    _check_pack(x)
    _refuse_grad("fp8_pack", x)
    values, tiles = torch.ops.sparseffn.fp8_pack(x) if torch.compiler.is_compiling() else _pack(x)
    q = Fp8Tensor.__new__(Fp8Tensor)
    q.values, q.scale_tiles, q.shape = values, tiles, x.shape
    return q


def fp8_unpack(q, dtype=torch.bfloat16):
    """The tensor an Fp8Tensor stands for, in float32, bfloat16 or float16.
    Exact in the first two; values beyond the type's range become its largest."""
    _lib.require_cuda(q.values)
    if dtype not in _lib._DTYPES:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, bfloat16 or float16")
    if torch.compiler.is_compiling():
        return torch.ops.sparseffn.fp8_unpack(q.values, q.scale_tiles, q.shape, dtype)
    return _unpack(q.values, q.scale_tiles, torch.empty(q.shape, dtype=dtype, device=q.values.device), q.shape[-1])


# ---------------------------------------------------------------------------
# The product
# ---------------------------------------------------------------------------
@functools.lru_cache(maxsize=4096)
def _product_workspace(packed, M, N, K):
    return getattr(_lib.load(), "sffn_fp8_mm_workspace_bytes" if packed else "sffn_fp8_linear_workspace_bytes")(M, N, K)


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _matmul(av, at, bv, bt, out_dtype):
    M, K = av.shape
    N = bv.shape[0]
    dev = av.device
    out = torch.empty((M, N), dtype=out_dtype, device=dev)
    if not (M and N):
        return out
    code, status, stream = _lib._DTYPES[out_dtype], _lib.status_word(dev).data_ptr(), stream_handle(dev)
    if M <= FEW_ROWS:
        call("sffn_few_rows_fp8", av.data_ptr(), _stride(av), at.data_ptr(), bv.data_ptr(), _stride(bv), bt.data_ptr(), M, N,
             K, out.data_ptr(), code, N, status, stream)
    else:
        n = _product_workspace(True, M, N, K)
        ws = _workspace(n, dev)
        call("sffn_fp8_mm", av.data_ptr(), _stride(av), at.data_ptr(), bv.data_ptr(), _stride(bv), bt.data_ptr(), M, N, K,
             out.data_ptr(), code, N, ptr(ws), n, status, stream)
    return out


def _pack_matmul(x, bv, bt, out_dtype):
    """x [..., K] packed on the way, in one call."""
    x2 = _rows(x)
    M, K = x2.shape
    N = bv.shape[0]
    dev = x.device
    out = torch.empty((M, N), dtype=out_dtype, device=dev)
    if M and N:
        n = _product_workspace(False, M, N, K)
        ws = _workspace(n, dev)
        call("sffn_fp8_linear", x2.data_ptr(), _lib._DTYPES[x.dtype], _ld(x2), bv.data_ptr(), _stride(bv), bt.data_ptr(), M, N,
             K, out.data_ptr(), _lib._DTYPES[out_dtype], N, ws.data_ptr(), n, _lib.status_word(dev).data_ptr(),
             stream_handle(dev))
    return out


def _check_product(av, bv, out_dtype):
    _lib.require_cuda(av, bv)
    if out_dtype not in OUT_TYPES:
        raise TypeError(f"out_dtype must be bfloat16 or float16, got {out_dtype}")
    if av.shape[-1] != bv.shape[-1]:
        raise ValueError(f"a has rows of {av.shape[-1]}, b of {bv.shape[-1]}")
    if av.device != bv.device:
        raise ValueError(f"a is on {av.device}, b on {bv.device}")
    if bv.data_ptr() % 16 or (av.dtype == E4M3 and av.data_ptr() % 16):
        raise ValueError("values must start on 16 bytes")


def fp8_matmul(a, b, out_dtype=None):
    """a b^T: [..., K] with [N, K] -> [..., N], in bfloat16 or float16.

    b is an Fp8Tensor [N, K] (weights, packed once); a is one [..., K], or a
    float32, bfloat16 or float16 tensor, which is packed first.  out_dtype: a's
    own type where that is one of the two, else bfloat16.  Sums are float32,
    scales are applied to them block by block, the result is rounded once.
    Not differentiable."""
    if not isinstance(b, Fp8Tensor) or len(b.shape) != 2:
        raise TypeError("b must be an Fp8Tensor [N, K]")
    packed = isinstance(a, Fp8Tensor)
    if not packed:
        _check_pack(a)
        _refuse_grad("fp8_matmul", a)
        if out_dtype is None and a.dtype in OUT_TYPES:
            out_dtype = a.dtype
    out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    if torch.compiler.is_compiling():
        av, at = (a.values, a.scale_tiles) if packed else torch.ops.sparseffn.fp8_pack(a)
        out = torch.ops.sparseffn.fp8_matmul(av, at, b.values, b.scale_tiles, out_dtype)
    elif packed:
        _check_product(a.values, b.values, out_dtype)
        out = _matmul(a.values, a.scale_tiles, b.values, b.scale_tiles, out_dtype)
    else:
        _check_product(a, b.values, out_dtype)
        out = _pack_matmul(a, b.values, b.scale_tiles, out_dtype)
    return out if len(a.shape) == 2 else out.view(*a.shape[:-1], b.shape[0])


# ---------------------------------------------------------------------------
# A linear layer that keeps its input in 8 bits
# ---------------------------------------------------------------------------
def _fits(x, w, rows, cols):
    return w.dtype is x.dtype and w.is_cuda and w.device == x.device and w.shape == (rows, cols)


def _check_weights(x, **weights):
    """x [..., D] against weights {name: (tensor, shape)}: CUDA, one 16-bit type, one device."""
    ts = [w for w, _ in weights.values()]
    _lib.require_cuda(x, *ts)
    if x.dtype not in OUT_TYPES:
        raise TypeError(f"unsupported dtype {x.dtype}; expected bfloat16 or float16")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., width] with width >= 1, got {tuple(x.shape)}")
    for name, (w, shape) in weights.items():
        if w.dtype != x.dtype:
            raise TypeError(f"{name} is {w.dtype}, x {x.dtype}")
        if w.device != x.device:
            raise ValueError(f"{name} is on {w.device}, x on {x.device}")
        if w.dim() != 2 or tuple(w.shape) != shape or 0 in shape:
            raise ValueError(f"{name} must be {shape}, got {tuple(w.shape)}")


def _check_linear(x, W):
    if not (isinstance(x, torch.Tensor) and isinstance(W, torch.Tensor) and x.is_cuda and x.dim() and W.dim() == 2
            and x.dtype in OUT_TYPES and x.shape[-1] and W.shape[0] and _fits(x, W, W.shape[0], x.shape[-1])):
        _lib.require_cuda(x, W)
        _check_weights(x, W=(W, (W.shape[0] if W.dim() else 0, x.shape[-1] if x.dim() else 0)))


@functools.lru_cache(maxsize=4096)
def _linear_workspace(backward, odd, want, T, N, K):
    return _lib.load().sffn_ckpt_linear_workspace_bytes(backward, odd, want, T, N, K)


def _linear_forward(x, W, keep):
    """(y, values, tiles) -- the last two None without keep."""
    x2, W2 = _rows(x), _rows(W)
    T, K = x2.shape
    N, dev = W2.shape[0], x.device
    y = x2.new_empty((T, N))
    values = tiles = None
    if keep:
        values, tiles = _empty_values(T, K, dev), _empty_tiles(T, K, dev)
    if T:
        (ldx, ox), (ldw, ow) = _row_stride(x2, 1), _row_stride(W2, 2)
        n = _linear_workspace(0, ox | ow, 0, T, N, K)
        ws = _workspace(n, dev)
        call("sffn_ckpt_linear", _lib._DTYPES[x.dtype], x2.data_ptr(), ldx, W2.data_ptr(), ldw, ox | ow, T, N, K, y.data_ptr(),
             ptr(values), ptr(tiles), ptr(ws), n, _lib.status_word(dev).data_ptr(), stream_handle(dev))
    return (y if x.dim() == 2 else y.view(*x.shape[:-1], N)), values, tiles


def _linear_backward(dy, W, values, tiles, x_shape, want_x, want_W):
    dev = dy.device
    _lib.bind_thread(dev)
    dy2, W2 = _rows(dy), _rows(W)
    T, N = dy2.shape
    K = x_shape[-1]
    dx = dy2.new_empty(x_shape) if want_x else None
    if not T:
        return dx, submit_grad(W.new_zeros((N, K))) if want_W else None
    dW = dy2.new_empty((N, K)) if want_W else None
    (ldy, oy), (ldw, ow) = _row_stride(dy2, 1), _row_stride(W2, 2)
    dtype, status, stream = _lib._DTYPES[dy.dtype], _lib.status_word(dev).data_ptr(), stream_handle(dev)

    def run(dx, dW):
        n = _linear_workspace(1, oy | ow, (dx is not None) + 2 * (dW is not None), T, N, K)
        ws = _workspace(n, dev)
        call("sffn_ckpt_linear_bwd", dtype, dy2.data_ptr(), ldy, W2.data_ptr(), ldw, oy | ow, ptr(values),
             _stride(values) if dW is not None else 0, ptr(tiles), T, N, K, ptr(dx), ptr(dW), ptr(ws), n, status, stream)

    if want_x and want_W and current() is not None:  # dW's reduction beside dx
        run(None, dW)
        submit_grad(dW)
        run(dx, None)
    else:
        run(dx, dW)
        submit_grad(dW)
    return dx, dW


def _check_backward(dy, W, x_shape):
    if not _fits(dy, W, dy.shape[-1], x_shape[-1]):
        _check_weights(dy, W=(W, (dy.shape[-1], x_shape[-1])))


def _kept_input(dy, values, tiles, x_shape):
    """x as kept, on the strides that the kernels read."""
    rows, width = dy.numel() // dy.shape[-1], x_shape[-1]
    return _kept_rows(values, rows, width, E4M3, dy.device, 16), _kept_tiles(tiles, rows, width, dy.device)


class _CkptLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W):
        y, values, tiles = _linear_forward(x, W, ctx.needs_input_grad[1])
        ctx.save_for_backward(W, values, tiles)
        ctx.x_shape = x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        _lib.once_differentiable("ckpt_linear")
        W, values, tiles = ctx.saved_tensors
        _check_backward(dy, W, ctx.x_shape)
        if values is not None:
            values, tiles = _kept_input(dy, values, tiles, ctx.x_shape)
        return _linear_backward(dy, W, values, tiles, ctx.x_shape, *ctx.needs_input_grad)


def ckpt_linear(x, W):
    """y = x W^T for x [..., K], W [N, K], both bfloat16 or float16.

    Between forward and backward only W and x in 8 bits are kept (half a 16-bit
    x): the output and x's gradient are those of a linear layer, the weight's
    gradient is dy^T times the kept x.  Differentiable once, in reverse mode."""
    _check_linear(x, W)
    if torch.compiler.is_compiling():
        return torch.ops.sparseffn.ckpt_linear(x, W, torch.is_grad_enabled() and W.requires_grad)[0]
    if _lib.tracked(x, W):
        return _CkptLinear.apply(x, W)
    return _linear_forward(x, W, False)[0]
