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
import torch

from . import _lib
from ._lib import address as ptr
from ._lib import call, stream_handle
from .parallel import submit_grad

__all__ = ["BLOCK", "Fp8Tensor", "fp8_pack", "fp8_unpack", "fp8_matmul", "ckpt_linear"]

BLOCK = 128
E4M3 = torch.float8_e4m3fn
FEW_ROWS = 32  # products of at most so many rows read the weights by the few-row kernel
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
    return _cdiv(rows, 128), _cdiv(_cdiv(width, BLOCK), 4), 32, 4, 4


def _stride(values):
    """Bytes between rows (one row's stride says nothing)."""
    return values.stride(0) if values.shape[0] > 1 else _cdiv(values.shape[1], 16) * 16


def _rows(t):
    """t as [rows, width] with dense rows (a view where the strides allow one)."""
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    rows, width = t.shape
    dense = (width == 1 or t.stride(1) == 1) and (rows <= 1 or t.stride(0) >= width)
    return t if dense else t.contiguous()


def _ld(t):
    """Elements between the rows of a matrix with dense rows."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _aligned(t):
    """A 16-bit matrix with rows on 16 bytes, as TMA reads them, and its row
    stride: t, or a copy with padded rows."""
    ld = t.stride(0)
    if t.shape[0] == 1:
        ld = _cdiv(t.shape[1], 8) * 8
    if ld % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, ld
    ld = _cdiv(t.shape[1], 8) * 8
    out = t.new_empty((t.shape[0], ld))
    out[:, :t.shape[1]] = t
    return out[:, :t.shape[1]], ld


def _empty_values(rows, width, device, multiple=16):
    return torch.empty((rows, _cdiv(width, multiple) * multiple), dtype=E4M3, device=device)[:, :width]


def _empty_tiles(rows, width, device):
    return torch.empty(_tile_shape(rows, width), dtype=torch.uint8, device=device)


def _pack(x):
    """(values, scale tiles) of x [..., width]."""
    x2 = _rows(x)
    rows, width = x2.shape
    values, tiles = _empty_values(rows, width, x.device), _empty_tiles(rows, width, x.device)
    if rows:
        call("sffn_fp8_pack", x2.data_ptr(), _lib._DTYPES[x.dtype], rows, width, _ld(x2), values.data_ptr(),
             _stride(values), tiles.data_ptr(), stream_handle(x.device))
    return values, tiles


def _unpack(values, tiles, shape, dtype):
    out = torch.empty(shape, dtype=dtype, device=values.device)
    rows, width = values.shape
    if rows:
        call("sffn_fp8_unpack", values.data_ptr(), _stride(values), tiles.data_ptr(), rows, width, _lib._DTYPES[dtype],
             out.data_ptr(), width, stream_handle(values.device))
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
    return Fp8Tensor(values, tiles, x.shape)


def fp8_unpack(q, dtype=torch.bfloat16):
    """The tensor an Fp8Tensor stands for, in float32, bfloat16 or float16.
    Exact in the first two; values beyond the type's range become its largest."""
    _lib.require_cuda(q.values)
    if dtype not in _lib._DTYPES:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, bfloat16 or float16")
    if torch.compiler.is_compiling():
        return torch.ops.sparseffn.fp8_unpack(q.values, q.scale_tiles, q.shape, dtype)
    return _unpack(q.values, q.scale_tiles, q.shape, dtype)


# ---------------------------------------------------------------------------
# The product
# ---------------------------------------------------------------------------
def _matmul(av, at, bv, bt, out_dtype):
    M, K = av.shape
    N = bv.shape[0]
    dev = av.device
    out = torch.empty((M, N), dtype=out_dtype, device=dev)
    if not out.numel():
        return out
    if M <= FEW_ROWS:
        call("sffn_few_rows_fp8", av.data_ptr(), _stride(av), at.data_ptr(), bv.data_ptr(), _stride(bv), bt.data_ptr(), M, N,
             K, out.data_ptr(), _lib._DTYPES[out_dtype], N, stream_handle(dev))
    else:
        call("sffn_fp8_mm", av.data_ptr(), _stride(av), at.data_ptr(), bv.data_ptr(), _stride(bv), bt.data_ptr(), M, N, K,
             out.data_ptr(), _lib._DTYPES[out_dtype], N, _lib.status_word(dev).data_ptr(), stream_handle(dev))
    return out


def _check_product(av, bv, out_dtype):
    _lib.require_cuda(av, bv)
    if out_dtype not in OUT_TYPES:
        raise TypeError(f"out_dtype must be bfloat16 or float16, got {out_dtype}")
    if av.shape[-1] != bv.shape[-1]:
        raise ValueError(f"a has rows of {av.shape[-1]}, b of {bv.shape[-1]}")
    if av.device != bv.device:
        raise ValueError(f"a is on {av.device}, b on {bv.device}")
    if av.data_ptr() % 16 or bv.data_ptr() % 16:
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
    if not isinstance(a, Fp8Tensor):
        _check_pack(a)
        _refuse_grad("fp8_matmul", a)
        if out_dtype is None and a.dtype in OUT_TYPES:
            out_dtype = a.dtype
        if a.shape[-1] != b.shape[-1]:
            raise ValueError(f"a has rows of {a.shape[-1]}, b of {b.shape[-1]}")
        a = fp8_pack(a)
    out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    if torch.compiler.is_compiling():
        out = torch.ops.sparseffn.fp8_matmul(a.values, a.scale_tiles, b.values, b.scale_tiles, out_dtype)
    else:
        _check_product(a.values, b.values, out_dtype)
        out = _matmul(a.values, a.scale_tiles, b.values, b.scale_tiles, out_dtype)
    return out.view(*a.shape[:-1], b.shape[0])


# ---------------------------------------------------------------------------
# 16-bit products on the tensor cores
# ---------------------------------------------------------------------------
def _mm_into(out, A, a_mn, B, b_mn, second=None):
    """out [M, N] = A B^T; A is [M, K], or with a_mn [K, M]; B [N, K] or [K, N];
    plus second = (A2, B2), likewise, added within the product."""
    M, N = out.shape
    A, lda = _aligned(A)
    B, ldb = _aligned(B)
    K = A.shape[0] if a_mn else A.shape[1]
    A2 = B2 = None
    lda2 = ldb2 = K2 = 0
    if second is not None:
        (A2, lda2), (B2, ldb2) = map(_aligned, second)
        K2 = A2.shape[0] if a_mn else A2.shape[1]
    ws_bytes = _lib.load().sffn_gemm16_workspace_bytes(M, N, K, K2)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=out.device) if ws_bytes else None
    call("sffn_gemm16", _lib._DTYPES[out.dtype], A.data_ptr(), lda, int(a_mn), B.data_ptr(), ldb, int(b_mn), ptr(A2), lda2,
         ptr(B2), ldb2, K2, M, N, K, out.data_ptr(), _ld(out), ptr(ws), ws_bytes, _lib.status_word(out.device).data_ptr(),
         stream_handle(out.device))
    return out


def _linear(x, W):
    """x [T, K] W [N, K]^T in their type."""
    T, N = x.shape[0], W.shape[0]
    out = x.new_empty((T, N))
    if T == 0:
        return out
    if T <= FEW_ROWS:
        call("sffn_few_rows_mm", _lib._DTYPES[x.dtype], x.data_ptr(), _ld(x), W.data_ptr(), _ld(W), T, N, x.shape[1],
             out.data_ptr(), N, stream_handle(x.device))
        return out
    return _mm_into(out, x, False, W, False)


# ---------------------------------------------------------------------------
# A linear layer that keeps its input in 8 bits
# ---------------------------------------------------------------------------
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


def _linear_forward(x, W, keep):
    """(y, values, tiles) -- the last two None without keep."""
    x2 = _rows(x)
    y = _linear(x2, _rows(W)).view(*x.shape[:-1], W.shape[0])
    return (y, *_pack(x2)) if keep else (y, None, None)


def _linear_backward(dy, W, values, tiles, x_shape, want_x, want_W):
    _lib.bind_thread(dy.device)
    dy2, width = _rows(dy), x_shape[-1]
    dx = dW = None
    if want_W:
        dW = W.new_empty((dy2.shape[1], width))
        if dy2.shape[0]:
            kept = _unpack(values, tiles, values.shape, dy.dtype)
            _mm_into(dW, dy2, True, kept, True)
            del kept
        else:
            dW.zero_()
        submit_grad(dW)
    if want_x:
        dx = dy.new_empty(x_shape)
        if dy2.shape[0]:
            _mm_into(dx.view(-1, width), dy2, False, _rows(W), True)
    return dx, dW


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
        return _linear_backward(dy, W, values, tiles, ctx.x_shape, *ctx.needs_input_grad)


def ckpt_linear(x, W):
    """y = x W^T for x [..., K], W [N, K], both bfloat16 or float16.

    Between forward and backward only W and x in 8 bits are kept (half a 16-bit
    x): the output and x's gradient are those of a linear layer, the weight's
    gradient is dy^T times the kept x.  Differentiable once, in reverse mode."""
    _check_weights(x, W=(W, (W.shape[0] if W.dim() else 0, x.shape[-1] if x.dim() else 0)))
    if torch.compiler.is_compiling():
        return torch.ops.sparseffn.ckpt_linear(x, W)[0]
    if _lib.tracked(x, W):
        return _CkptLinear.apply(x, W)
    return _linear_forward(x, W, False)[0]
