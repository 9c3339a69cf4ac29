"""torch.library custom ops (namespace ``sparseffn``) over the CUDA library.

torch.compile and torch.export trace through these ops without graph breaks;
the reference's own attempt to register its kernels as ops is commented out
(old/lib_sparse/sparse.py:212-298).  Each op's kernel is this package's
eager API, so it runs the same CUDA code; each fake kernel gives only the
outputs' shapes and dtypes, so tracing needs no device.

    sparseffn::bitsparse_pack(dense) -> (vals, packed_mask)
        old/sparse_pack.py:66-106; len(vals) = nnz is data-dependent (an
        unbacked size while tracing)
    sparseffn::bitsparse_unpack(vals, packed_mask, shape) -> dense
        old/sparse_unpack.py:57-97
    sparseffn::tile_pack(dense, vals!, offset!, block_m, block_n) -> (bitmask, prefix, vals_offset)
        dense_to_tilesparse, old/lib_sparse/sparse.py:154-210; writes the vals
        arena and advances its cursor in place
    sparseffn::tile_unpack(vals, bitmask, prefix, vals_offset, shape, block_m, block_n, square)
        -> dense, old/lib_sparse/sparse_unpack.py:5-55
    sparseffn::ffn_fwd(x, W1, W2, b1?, vals!, offset!, act)
        -> (out, bitmask, prefix, vals_offset, row_offsets, kb_list, kb_count)
    sparseffn::ffn_bwd(grad_output, x, W1, W2, vals, bitmask, prefix, vals_offset, row_offsets,
                       kb_list, kb_count, fused, has_bias, act) -> (grad_x, grad_W1, grad_W2, grad_b1)
        the forward and backward of FFNSparse / FFNSpRelu2 (sparse.py:56-151),
        which call them; act is 0 (ReLU) or 1 (ReLU^2).  The ops that write the
        arena carry no autograd formula (torch.library allows none on a
        mutating op): the autograd.Function classes in ffn.py hold that.
    sparseffn::codec15_compress(data) -> stream
    sparseffn::codec15_uncompress(stream, shape, dtype) -> data
        the 15-bit sign-strip codec, bitshifting/code.py:129-177
    sparseffn::token_logprobs(logits, targets?, top_k, temperature, ignore_index)
        -> (logp, entropy, top_ids, top_logp, stats)
    sparseffn::distill_topk(logits, ids, scores, temperature, tail) -> (loss, stats)
    sparseffn::residual_norm(x, y?, pre?, post?, gate?, groups, post_norm, scale, eps, out_dtype)
        -> (x_new, h, stats)
        the operators of logits.py and norms.py (without counterpart in the
        reference), with their autograd formulas over the ops named *_bwd;
        their functions call these ops while torch.compile traces.  Outputs
        that a call leaves out are empty tensors here.

The fused bf16 path (ffn._fused_ok, decided from dtypes, contiguity and
shapes alone) keeps z in 128x128 tiles and returns per-row value offsets and
K-block lists; the float32 / float16 path keeps 64x64 tiles and returns
those three as empty tensors, as it does grad_b1 when there is no bias.
"""
from typing import Optional

import torch
from torch import Tensor

from . import bitshift
from . import bitsparse as bs
from . import ffn, logits, norms

__all__ = ["OPS"]

OPS = ("bitsparse_pack", "bitsparse_unpack", "tile_pack", "tile_unpack", "ffn_fwd", "ffn_bwd",
       "codec15_compress", "codec15_uncompress", "token_logprobs", "token_logprobs_bwd", "distill_topk",
       "distill_topk_bwd", "residual_norm", "residual_norm_bwd")


def _cdiv(a, b):
    return (a + b - 1) // b


def _i32(like, *shape):
    return torch.empty(shape, dtype=torch.int32, device=like.device)


# ---------------------------------------------------------------------------
# Flat format
# ---------------------------------------------------------------------------
@torch.library.custom_op("sparseffn::bitsparse_pack", mutates_args=())
def bitsparse_pack(dense: Tensor) -> tuple[Tensor, Tensor]:
    return bs.bitsparse_pack(dense)


@bitsparse_pack.register_fake
def _(dense):
    nnz = torch.library.get_ctx().new_dynamic_size()
    return dense.new_empty(nnz), dense.new_empty(_cdiv(dense.numel(), 8), dtype=torch.uint8)


@torch.library.custom_op("sparseffn::bitsparse_unpack", mutates_args=())
def bitsparse_unpack(vals: Tensor, packed_mask: Tensor, shape: list[int]) -> Tensor:
    return bs.bitsparse_unpack(vals, packed_mask, shape)


@bitsparse_unpack.register_fake
def _(vals, packed_mask, shape):
    return vals.new_empty(shape)


# ---------------------------------------------------------------------------
# Tiled format
# ---------------------------------------------------------------------------
@torch.library.custom_op("sparseffn::tile_pack", mutates_args=("vals", "offset"))
def tile_pack(dense: Tensor, vals: Tensor, offset: Tensor, block_m: int,
              block_n: int) -> tuple[Tensor, Tensor, Tensor]:
    x = bs.dense_to_tilesparse(dense, vals, offset, block_m, block_n)
    return x.bitmask, x.prefix, x.vals_offset


@tile_pack.register_fake
def _(dense, vals, offset, block_m, block_n):
    nt = _cdiv(dense.shape[0], block_m) * _cdiv(dense.shape[1], block_n)
    return (dense.new_empty(nt * block_m * block_n // 8, dtype=torch.uint8), _i32(dense, nt + 1),
            _i32(dense, 1))


@torch.library.custom_op("sparseffn::tile_unpack", mutates_args=())
def tile_unpack(vals: Tensor, bitmask: Tensor, prefix: Tensor, vals_offset: Tensor, shape: list[int],
                block_m: int, block_n: int, square: bool) -> Tensor:
    M, N = shape
    x = bs.BitsparseTensor(vals, bitmask, prefix, vals_offset, _cdiv(M, block_m), _cdiv(N, block_n),
                           block_m, block_n, (M, N))
    return bs.tile_unpack(x, square=square)


@tile_unpack.register_fake
def _(vals, bitmask, prefix, vals_offset, shape, block_m, block_n, square):
    return vals.new_empty(shape)


# ---------------------------------------------------------------------------
# FFN forward / backward
# ---------------------------------------------------------------------------
@torch.library.custom_op("sparseffn::ffn_fwd", mutates_args=("vals", "offset"))
def ffn_fwd(x: Tensor, W1: Tensor, W2: Tensor, b1: Optional[Tensor], vals: Tensor, offset: Tensor,
            act: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    if ffn._fused_ok(x, W1, W2, b1, vals):
        return ffn._fused_forward(x, W1, W2, vals, offset, b1, act)
    out, z = ffn._unfused_forward(x, W1, W2, vals, offset, b1, act)
    return out, z.bitmask, z.prefix, z.vals_offset, _i32(x, 0), _i32(x, 0, 0), _i32(x, 0)


@ffn_fwd.register_fake
def _(x, W1, W2, b1, vals, offset, act):
    T, Fd, D = x.shape[0], W1.shape[0], W2.shape[0]
    fused = ffn._fused_ok(x, W1, W2, b1, vals)
    bm = 128 if fused else 64
    nt = _cdiv(T, bm) * _cdiv(Fd, bm)
    out = x.new_empty(T, D)
    bitmask = x.new_empty(nt * bm * bm // 8, dtype=torch.uint8)
    if fused:
        aux = (_i32(x, nt * 128), _i32(x, _cdiv(T, 256), _cdiv(Fd, 64)), _i32(x, _cdiv(T, 256)))
    else:
        aux = (_i32(x, 0), _i32(x, 0, 0), _i32(x, 0))
    return (out, bitmask, _i32(x, nt + 1), _i32(x, 1)) + aux


@torch.library.custom_op("sparseffn::ffn_bwd", mutates_args=())
def ffn_bwd(grad_output: Tensor, x: Tensor, W1: Tensor, W2: Tensor, vals: Tensor, bitmask: Tensor,
            prefix: Tensor, vals_offset: Tensor, row_offsets: Tensor, kb_list: Tensor,
            kb_count: Tensor, fused: bool, has_bias: bool,
            act: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    T, Fd = x.shape[0], W1.shape[0]
    bm = 128 if fused else 64
    z = bs.BitsparseTensor(vals, bitmask, prefix, vals_offset, _cdiv(T, bm), _cdiv(Fd, bm), bm, bm,
                           (T, Fd))
    if fused:
        grads = ffn._fused_backward(grad_output, x, W1, W2, z, row_offsets, kb_list, kb_count,
                                    has_bias, act)
    else:
        grads = ffn._unfused_backward(grad_output, x, W1, W2, z, has_bias, act)
    grad_x, grad_W1, grad_W2, grad_b1 = grads
    if grad_b1 is None:
        grad_b1 = x.new_empty(0)
    return grad_x, grad_W1, grad_W2, grad_b1


@ffn_bwd.register_fake
def _(grad_output, x, W1, W2, vals, bitmask, prefix, vals_offset, row_offsets, kb_list, kb_count,
      fused, has_bias, act):
    return (x.new_empty(x.shape), W1.new_empty(W1.shape), W2.new_empty(W2.shape),
            x.new_empty(W1.shape[0] if has_bias else 0))


# ---------------------------------------------------------------------------
# 15-bit sign-strip codec
# ---------------------------------------------------------------------------
@torch.library.custom_op("sparseffn::codec15_compress", mutates_args=())
def codec15_compress(data: Tensor) -> Tensor:
    return bitshift.compress_fn(data)


@codec15_compress.register_fake
def _(data):
    return data.new_empty(bitshift.padded_bytes(data.numel()), dtype=torch.uint8)


@torch.library.custom_op("sparseffn::codec15_uncompress", mutates_args=())
def codec15_uncompress(compressed: Tensor, shape: list[int], dtype: torch.dtype) -> Tensor:
    return bitshift.uncompress_fn(compressed, shape, dtype)


@codec15_uncompress.register_fake
def _(compressed, shape, dtype):
    return compressed.new_empty(shape, dtype=dtype)


# ---------------------------------------------------------------------------
# Output distribution (parameters are named x: the module `logits` stays reachable)
# ---------------------------------------------------------------------------
@torch.library.custom_op("sparseffn::token_logprobs", mutates_args=())
def token_logprobs(x: Tensor, targets: Optional[Tensor], top_k: int, temperature: float,
                   ignore_index: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    logits._check_score(x, targets, top_k, temperature)
    return logits._score_forward(x, targets, top_k, temperature, ignore_index)


@token_logprobs.register_fake
def _(x, targets, top_k, temperature, ignore_index):
    lead = x.shape[:-1]
    f32 = dict(dtype=torch.float32)
    return (x.new_empty(lead if targets is not None else (0,), **f32), x.new_empty(lead, **f32),
            x.new_empty((*lead, top_k), dtype=torch.int64), x.new_empty((*lead, top_k), **f32),
            x.new_empty((*lead, 2), **f32))


@torch.library.custom_op("sparseffn::token_logprobs_bwd", mutates_args=())
def token_logprobs_bwd(x: Tensor, targets: Optional[Tensor], top_ids: Tensor, entropy: Tensor, stats: Tensor,
                       g_logp: Optional[Tensor], g_entropy: Optional[Tensor], g_top: Optional[Tensor],
                       temperature: float, ignore_index: int) -> Tensor:
    lead, k = x.shape[:-1], top_ids.shape[-1]
    logits._check_score(x, targets, k, temperature)
    for name, t, shape in (("entropy", entropy, lead), ("stats", stats, (*lead, 2)), ("g_logp", g_logp, lead),
                           ("g_entropy", g_entropy, lead), ("g_top", g_top, (*lead, k))):
        logits._check_kept(name, t, shape, x.device)
    logits._check_kept("top_ids", top_ids, (*lead, k), x.device, torch.int64)
    return logits._score_backward(x, targets, top_ids.contiguous(), entropy.contiguous(), stats.contiguous(), g_logp,
                                  g_entropy, g_top, temperature, ignore_index).contiguous()


@token_logprobs_bwd.register_fake
def _(x, targets, top_ids, entropy, stats, g_logp, g_entropy, g_top, temperature, ignore_index):
    return x.new_empty(x.shape)


def _score_setup(ctx, inputs, output):
    x, targets, _, temperature, ignore_index = inputs
    _, entropy, top_ids, _, stats = output
    ctx.save_for_backward(x, targets, top_ids, entropy, stats)
    ctx.args = temperature, ignore_index
    ctx.mark_non_differentiable(top_ids, stats)
    ctx.set_materialize_grads(False)


def _score_bwd(ctx, g_logp, g_entropy, _ids, g_top, _stats):
    x, targets, top_ids, entropy, stats = ctx.saved_tensors
    grad = token_logprobs_bwd(x, targets, top_ids, entropy, stats, g_logp if targets is not None else None,
                              g_entropy, g_top, *ctx.args)
    return grad, None, None, None, None


token_logprobs.register_autograd(_score_bwd, setup_context=_score_setup)


@torch.library.custom_op("sparseffn::distill_topk", mutates_args=())
def distill_topk(x: Tensor, ids: Tensor, scores: Tensor, temperature: float, tail: str) -> tuple[Tensor, Tensor]:
    logits._check_distill(x, ids, scores, temperature, tail)
    return logits._distill_forward(x, ids, scores, temperature, tail)


@distill_topk.register_fake
def _(x, ids, scores, temperature, tail):
    return x.new_empty(x.shape[:-1], dtype=torch.float32), x.new_empty((*x.shape[:-1], 4), dtype=torch.float32)


@torch.library.custom_op("sparseffn::distill_topk_bwd", mutates_args=())
def distill_topk_bwd(x: Tensor, ids: Tensor, scores: Tensor, stats: Tensor, g_loss: Tensor, temperature: float,
                     tail: str) -> Tensor:
    logits._check_distill(x, ids, scores, temperature, tail)
    logits._check_kept("stats", stats, (*x.shape[:-1], 4), x.device)
    logits._check_kept("g_loss", g_loss, x.shape[:-1], x.device)
    return logits._distill_backward(x, ids, scores, stats.contiguous(), g_loss, temperature, tail).contiguous()


@distill_topk_bwd.register_fake
def _(x, ids, scores, stats, g_loss, temperature, tail):
    return x.new_empty(x.shape)


def _distill_setup(ctx, inputs, output):
    x, ids, scores, temperature, tail = inputs
    ctx.save_for_backward(x, ids, scores, output[1])
    ctx.args = temperature, tail
    ctx.mark_non_differentiable(output[1])


def _distill_bwd(ctx, g_loss, _stats):
    return distill_topk_bwd(*ctx.saved_tensors, g_loss, *ctx.args), None, None, None, None


distill_topk.register_autograd(_distill_bwd, setup_context=_distill_setup)


# ---------------------------------------------------------------------------
# Norms around a block
# ---------------------------------------------------------------------------
def _or_empty(like, ts):
    return tuple(t if t is not None else like.new_empty(0) for t in ts)


@torch.library.custom_op("sparseffn::residual_norm", mutates_args=())
def residual_norm(x: Tensor, y: Optional[Tensor], pre: Optional[Tensor], post: Optional[Tensor],
                  gate: Optional[Tensor], groups: int, post_norm: bool, scale: float, eps: float,
                  out_dtype: torch.dtype) -> tuple[Tensor, Tensor, Tensor]:
    norms._check(x, y, pre, post, gate, post_norm, scale, eps, out_dtype)
    norms._check_groups(x, gate, groups)
    return _or_empty(x, norms._forward(x, y, pre, post, gate, groups, post_norm, scale, eps, out_dtype, True))


@residual_norm.register_fake
def _(x, y, pre, post, gate, groups, post_norm, scale, eps, out_dtype):
    return (x.new_empty(x.shape if y is not None else (0,)), x.new_empty(x.shape, dtype=out_dtype),
            x.new_empty((x.numel() // x.shape[-1], 2), dtype=torch.float32))


@torch.library.custom_op("sparseffn::residual_norm_bwd", mutates_args=())
def residual_norm_bwd(x: Tensor, y: Optional[Tensor], pre: Optional[Tensor], post: Optional[Tensor],
                      gate: Optional[Tensor], groups: int, post_norm: bool, scale: float, out_dtype: torch.dtype,
                      stats: Tensor, dx_new: Optional[Tensor], dh: Optional[Tensor],
                      want: list[bool]) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    norms._check(x, y, pre, post, gate, post_norm, scale, 1.0, out_dtype)
    norms._check_groups(x, gate, groups)
    norms._check_backward(x, y, dx_new, dh, stats, out_dtype)
    return _or_empty(x, norms._backward(x, y, pre, post, gate, groups, post_norm, scale, out_dtype, stats, dx_new,
                                        dh, want))


@residual_norm_bwd.register_fake
def _(x, y, pre, post, gate, groups, post_norm, scale, out_dtype, stats, dx_new, dh, want):
    return tuple(t.new_empty(t.shape) if t is not None and w else x.new_empty(0)
                 for t, w in zip((x, y, pre, post, gate), want))


def _norm_setup(ctx, inputs, output):
    x, y, pre, post, gate, groups, post_norm, scale, eps, out_dtype = inputs
    ctx.save_for_backward(x, y, pre, post, gate, output[2])
    ctx.args = groups, post_norm, scale, out_dtype
    ctx.mark_non_differentiable(output[2])
    ctx.set_materialize_grads(False)


def _norm_bwd(ctx, dx_new, dh, _stats):
    x, y, pre, post, gate, stats = ctx.saved_tensors
    want = [t is not None and w for t, w in zip((x, y, pre, post, gate), ctx.needs_input_grad)]
    grads = residual_norm_bwd(x, y, pre, post, gate, *ctx.args, stats, dx_new if y is not None else None, dh, want)
    return *(g if w else None for g, w in zip(grads, want)), None, None, None, None, None


residual_norm.register_autograd(_norm_bwd, setup_context=_norm_setup)
