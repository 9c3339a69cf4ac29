"""Operators on a model's output distribution.

    token_logprobs(logits, targets, top_k=, temperature=)
        log probabilities of given tokens, the entropy of every row and its
        top alternatives, in one pass over the logits
    distill_topk(logits, teacher_ids, teacher_scores, temperature=, tail=)
        the divergence of a student's logits from a teacher's top log
        probabilities (what token_logprobs(top_k=) of the teacher gives)

Both take logits [..., V] in float32, bfloat16 or float16 (rows of any stride
whose last dimension is dense; two leading strides are read in place, more
are copied), compute in float32, and carry their gradient with respect to the
logits (once, and in reverse mode: forward-mode tangents are refused).  Nothing
of the logits' size is written in the forward, and only the gradient in the
backward.
"""
import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import address as ptr
from ._lib import call, stream_handle

__all__ = ["TokenLogprobs", "token_logprobs", "distill_topk", "TOP_MAX"]

TOP_MAX = 128  # alternatives a row
TAILS = {"renorm": 0, "bucket": 1}


class TokenLogprobs(NamedTuple):
    """What token_logprobs gives: float32 logp [...] (None without targets),
    float32 entropy [...], int64 top_ids [..., top_k], float32 top_logp [..., top_k]."""
    logp: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logp: torch.Tensor


def _rows(logits):
    """(logits or a copy, rows, inner, s_outer, s_inner): row r starts at
    s_outer * (r // inner) + s_inner * (r % inner)."""
    V = logits.shape[-1]
    if logits.is_contiguous():
        rows = logits.numel() // V
        return logits, rows, rows, 0, V
    if V > 1 and logits.stride(-1) != 1:
        logits = logits.contiguous()
    dims = []  # merged (size, stride) of the leading dimensions
    for n, st in zip(logits.shape[:-1], logits.stride()[:-1]):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * st:
            dims[-1] = (dims[-1][0] * n, st)
        else:
            dims.append((n, st))
    if len(dims) > 2:
        logits = logits.contiguous()
        dims = [(logits.numel() // V, V)]
    if not dims:
        dims = [(1, V)]
    rows = math.prod(n for n, _ in dims)
    inner, s_inner = dims[-1]
    return logits, rows, inner, (dims[0][1] if len(dims) == 2 else 0), s_inner


def _grad_like(logits, rows, s_inner):
    """An uninitialised gradient of logits' shape, its rows one stride apart,
    and that stride.  Rows lie to 16-byte boundaries as the logits' rows do, so
    the kernel's 16-byte accesses of the two go together (contiguous logits
    get a contiguous gradient)."""
    V, n = logits.shape[-1], 16 // logits.element_size()
    ld = V + (s_inner - V) % n if rows > 1 else V
    at = logits.data_ptr() % 16 // logits.element_size()
    if ld == V and at == 0:
        return torch.empty_like(logits, memory_format=torch.contiguous_format), V
    flat = logits.new_empty(at + rows * ld)
    strides, step = [1], ld
    for k in reversed(logits.shape[:-1]):
        strides.append(step)
        step *= k
    return flat.as_strided(logits.shape, strides[::-1], at), ld


def _check_logits(name, logits, temperature):
    _lib.require_cuda(logits)
    _lib.dtype_code(logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{name} takes logits [..., V] with V >= 1, got {tuple(logits.shape)}")
    if not (isinstance(temperature, (int, float)) and 1e-30 <= temperature <= 1e30):  # ln p / T stays finite in float32
        raise ValueError(f"temperature must be a number in [1e-30, 1e30], got {temperature!r}")


def _check_index(name, t, shape, device):
    _lib.require_cuda(t)
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be int64 or int32, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the logits on {device}")


def _check_kept(name, t, shape, device, dtype=torch.float32):
    """What a backward op is given of the forward and of upstream gradients."""
    if t is not None and (tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device):
        raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)} on {device}")


# ---------------------------------------------------------------------------
# token_logprobs
# ---------------------------------------------------------------------------
def _score_forward(logits, targets, top_k, temperature, ignore_index, keep=True):
    """(logp or an empty tensor, entropy, top_ids, top_logp, stats [..., 2]; None without keep)."""
    dev, lead = logits.device, logits.shape[:-1]
    x, rows, inner, so, si = _rows(logits)
    f32 = torch.float32
    entropy = x.new_empty(lead, dtype=f32)
    logp = torch.empty_like(entropy) if targets is not None else x.new_empty(0, dtype=f32)
    stats = x.new_empty((*lead, 2), dtype=f32) if keep else None
    top_ids = x.new_empty((*lead, top_k), dtype=torch.int64)
    top_logp = torch.empty_like(top_ids, dtype=f32)
    if rows:
        t = targets.contiguous() if targets is not None else None
        call("sffn_token_logprobs", ptr(x), _lib.dtype_code(x), rows, x.shape[-1], inner, so, si, ptr(t),
             t.element_size() if t is not None else 0, ignore_index, top_k, 1.0 / temperature,
             ptr(logp), ptr(entropy), ptr(stats), ptr(top_ids), ptr(top_logp), ptr(_lib.status_word(dev)),
             stream_handle(dev))
    return logp, entropy, top_ids, top_logp, stats


def _score_backward(logits, targets, top_ids, entropy, stats, g_logp, g_entropy, g_top, temperature, ignore_index):
    _lib.bind_thread(logits.device)
    x, rows, inner, so, si = _rows(logits)
    grad, ld = _grad_like(x, rows, si)
    if rows:
        t = targets.contiguous() if targets is not None else None
        g_logp, g_entropy, g_top = (g.contiguous() if g is not None else None for g in (g_logp, g_entropy, g_top))
        call("sffn_token_logprobs_bwd", ptr(x), _lib.dtype_code(x), rows, x.shape[-1], inner, so, si, ptr(t),
             t.element_size() if t is not None else 0, ignore_index, ptr(top_ids), top_ids.shape[-1],
             1.0 / temperature, ptr(stats), ptr(entropy), ptr(g_logp), ptr(g_entropy), ptr(g_top), ptr(grad), ld,
             stream_handle(x.device))
    return grad


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature, ignore_index):
        logp, entropy, top_ids, top_logp, stats = _score_forward(logits, targets, top_k, temperature, ignore_index)
        ctx.save_for_backward(logits, targets, top_ids, entropy, stats)
        ctx.args = temperature, ignore_index
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_ids)
        return logp, entropy, top_ids, top_logp

    @staticmethod
    def backward(ctx, g_logp, g_entropy, _, g_top):
        _lib.once_differentiable("token_logprobs")
        logits, targets, top_ids, entropy, stats = ctx.saved_tensors
        if targets is None:
            g_logp = None
        return (_score_backward(logits, targets, top_ids, entropy, stats, g_logp, g_entropy, g_top, *ctx.args),
                None, None, None, None)


def _check_score(logits, targets, top_k, temperature):
    _check_logits("token_logprobs", logits, temperature)
    V = logits.shape[-1]
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 0 <= top_k <= min(V, TOP_MAX):
        raise ValueError(f"top_k must be an integer in [0, {min(V, TOP_MAX)}], got {top_k!r}")
    if targets is not None:
        _check_index("targets", targets, logits.shape[:-1], logits.device)


def token_logprobs(logits, targets=None, top_k=0, temperature=1.0, ignore_index=-100) -> TokenLogprobs:
    """Log probabilities of `targets` under softmax(logits / temperature), the
    entropy of each row, and its top_k (<= 128) alternatives, largest first,
    equal logits by lower index.

    logits [..., V]; targets [...] int64 or int32, or None for no logp.  logp,
    entropy and top_logp are float32 and differentiable with respect to the
    logits.  Rows whose target is ignore_index are left out: logp and entropy
    0, ids -1, top_logp -inf, gradient 0 (distill_topk takes such a list as
    empty).  Logits of -inf have probability 0; a row of nothing else has logp
    -inf, entropy 0, gradient 0.  A row holding NaN or +inf has NaN.  Another
    target outside [0, V) gives NaN and sets the library's status word
    (check_status() reports it); its logp has no gradient (the row's entropy
    and top_logp keep theirs), so that one bad target does not spoil the
    weights before the status is looked at."""
    _check_score(logits, targets, top_k, temperature)
    if torch.compiler.is_compiling():
        r = torch.ops.sparseffn.token_logprobs(logits, targets, top_k, temperature, ignore_index)
    elif _lib.tracked(logits):
        r = _TokenLogprobs.apply(logits, targets, top_k, temperature, ignore_index)
    else:
        r = _score_forward(logits, targets, top_k, temperature, ignore_index, keep=False)
    return TokenLogprobs(r[0] if targets is not None else None, r[1], r[2], r[3])


# ---------------------------------------------------------------------------
# distill_topk
# ---------------------------------------------------------------------------
def _distill_forward(logits, ids, scores, temperature, tail, keep=True):
    """(loss, stats [..., 4]; None without keep)."""
    dev, lead = logits.device, logits.shape[:-1]
    x, rows, inner, so, si = _rows(logits)
    loss = x.new_empty(lead, dtype=torch.float32)
    stats = x.new_empty((*lead, 4), dtype=torch.float32) if keep else None
    if rows:
        ids, scores = ids.contiguous(), scores.contiguous()
        call("sffn_distill_topk", ptr(x), _lib.dtype_code(x), rows, x.shape[-1], inner, so, si, ptr(ids),
             ids.element_size(), ptr(scores), _lib.dtype_code(scores), ids.shape[-1], TAILS[tail],
             1.0 / temperature, ptr(loss), ptr(stats), ptr(_lib.status_word(dev)), stream_handle(dev))
    return loss, stats


def _distill_backward(logits, ids, scores, stats, g_loss, temperature, tail):
    _lib.bind_thread(logits.device)
    x, rows, inner, so, si = _rows(logits)
    grad, ld = _grad_like(x, rows, si)
    if rows:
        ids, scores, g_loss = ids.contiguous(), scores.contiguous(), g_loss.contiguous()
        call("sffn_distill_topk_bwd", ptr(x), _lib.dtype_code(x), rows, x.shape[-1], inner, so, si, ptr(ids),
             ids.element_size(), ptr(scores), _lib.dtype_code(scores), ids.shape[-1], TAILS[tail],
             1.0 / temperature, ptr(stats), ptr(g_loss), ptr(grad), ld, stream_handle(x.device))
    return grad


class _DistillTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, scores, temperature, tail):
        loss, stats = _distill_forward(logits, ids, scores, temperature, tail)
        ctx.save_for_backward(logits, ids, scores, stats)
        ctx.args = temperature, tail
        return loss

    @staticmethod
    def backward(ctx, g_loss):
        _lib.once_differentiable("distill_topk")
        logits, ids, scores, stats = ctx.saved_tensors
        return _distill_backward(logits, ids, scores, stats, g_loss, *ctx.args), None, None, None, None


def _check_distill(logits, teacher_ids, teacher_scores, temperature, tail):
    _check_logits("distill_topk", logits, temperature)
    if tail not in TAILS:
        raise ValueError(f"tail must be one of {sorted(TAILS)}, got {tail!r}")
    if not isinstance(teacher_ids, torch.Tensor) or teacher_ids.dim() < 1 or not 1 <= teacher_ids.shape[-1] <= TOP_MAX:
        raise ValueError(f"teacher_ids must be [..., K] with 1 <= K <= {TOP_MAX}")
    shape = (*logits.shape[:-1], teacher_ids.shape[-1])
    _check_index("teacher_ids", teacher_ids, shape, logits.device)
    _lib.require_cuda(teacher_scores)
    _lib.dtype_code(teacher_scores)
    if tuple(teacher_scores.shape) != shape or teacher_scores.device != logits.device:
        raise ValueError(f"teacher_scores must have shape {shape} on {logits.device}, got "
                         f"{tuple(teacher_scores.shape)} on {teacher_scores.device}")


def distill_topk(logits, teacher_ids, teacher_scores, temperature=1.0, tail="renorm"):
    """float32 [...]: for each row the divergence sum q (ln q - ln p) of the
    student's distribution p = softmax(logits / temperature) from a teacher's
    list of K <= 128 entries, differentiable with respect to the logits.

    teacher_ids [..., K] int64 or int32 (-1: absent), teacher_scores [..., K]
    float32, bfloat16 or float16: the teacher's log probabilities at its
    temperature, as token_logprobs(teacher, top_k=K, temperature=T) gives them
    (they are not divided by `temperature` again, and no gradient flows to
    them).  tail says what becomes of the probability the list leaves out:

      "renorm"  the listed mass is scaled to one, q = softmax(teacher_scores);
                scores may then be the teacher's logits / T themselves
      "bucket"  q = exp(teacher_scores), and the rest, 1 - sum q, is one more
                class, compared with the student's mass off the list (a rest
                below 2^-20 is the scores' own rounding and counts as none)

    A row without an entry of positive weight (ids all -1, scores all -inf)
    has loss 0 and gradient 0.  An id listed twice counts with both weights.
    Where the student gives a listed class no probability (a logit of -inf, not
    one that is only far below) the loss is +inf; with "bucket" also where it
    has -inf for every class off the list and a rest is left.
    Other ids outside [0, V) count as absent and set the library's status word
    (check_status() reports it).  The loss carries no factor T^2."""
    _check_distill(logits, teacher_ids, teacher_scores, temperature, tail)
    if teacher_scores.requires_grad and torch.is_grad_enabled():
        raise ValueError("no gradient flows to teacher_scores: detach them")
    if torch.compiler.is_compiling():
        return torch.ops.sparseffn.distill_topk(logits, teacher_ids, teacher_scores, temperature, tail)[0]
    if _lib.tracked(logits):
        return _DistillTopk.apply(logits, teacher_ids, teacher_scores, temperature, tail)
    return _distill_forward(logits, teacher_ids, teacher_scores, temperature, tail, keep=False)[0]
