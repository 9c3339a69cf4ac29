"""GPU checks of distill_topk's bucket where what the teacher's list leaves, the
rest 1 - sum q, is small or the student's mass off the list is, against float64.

u = 2^-24.  The rest r is summed in 64 bits and rounded once (u r).  Off the list
the gradient is softmax_off(j) (p_r - r), p_r the student's mass there: p_r and
softmax_off are quotients of sums of exponentials, each within e = (300 + n) u of
itself for n additions to an accumulator (exponents up to 40 in base 2 with 3
roundings each: 83 u, as much again for a change of the reference; 6 u an
exponential).  So an element is within softmax_off(j) (p_r + r) (2 e + 8 u),
whatever p_r - r leaves."""
import math

import pytest
import torch

import autoresearch2_b200 as sf

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F64 = torch.float64


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed), device=DEV)


def definition(x, ids, scores, T=1.0):
    """(loss, gradient, softmax off the list (0 on it), ln p_r, rest), float64; distinct ids."""
    lp = torch.log_softmax(x.detach().to(F64) / T, -1)
    c = scores.to(F64)
    q = c.exp()
    rest = 1.0 - q.sum(-1, keepdim=True)
    rest = torch.where(rest < 2.0 ** -20, 0.0, rest)
    off = lp.scatter(1, ids, -math.inf)
    ln_pr = off.logsumexp(-1, keepdim=True)
    soft = (off - ln_pr).exp()
    loss = (q * (c - lp.gather(1, ids))).sum(-1, keepdim=True)
    loss = loss + torch.where(rest > 0, rest * (rest.log() - ln_pr), 0.0)
    Q = q.sum(-1, keepdim=True) + rest
    grad = (soft * (Q * ln_pr.exp() - rest)).scatter(1, ids, Q * lp.gather(1, ids).exp() - q) / T
    return loss[:, 0], grad, soft, ln_pr, rest


def a_list(rows, V, K, rest, seed):
    """Random classes and log probabilities that leave about `rest`."""
    ids = torch.rand(rows, V, generator=gen(seed), device=DEV).argsort(-1)[:, :K].contiguous()
    w = torch.softmax(randn(rows, K, seed=seed + 1).to(F64), -1)
    return ids, (w * (1.0 - rest)).log().float()


def additions(V):
    return V // 64 + 40


def within(got, want, tol, dtype=torch.float32):
    fi = torch.finfo(dtype)
    tol = tol + want.abs() * (fi.eps / 2) * (1 + 2 ** -10) + fi.smallest_normal * fi.eps / 2
    err = (got.detach().to(F64) - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3g} of the tolerance"


@pytest.mark.parametrize("rest", [3e-6, 1e-5, 1e-3])
@pytest.mark.parametrize("rows,V,K", [(6, 1000, 128), (1300, 900, 100), (3, 50304, 128)])
def test_a_small_rest_keeps_its_digits(rows, V, K, rest):
    """The student too has little off the list, so that p_r - r turns on the rest."""
    ids, scores = a_list(rows, V, K, rest, 1)
    x = randn(rows, V, seed=3)
    x.scatter_add_(1, ids, torch.full_like(scores, math.log(V / K / rest) + 1.0))
    x.requires_grad_()
    got = sf.distill_topk(x, ids, scores, tail="bucket")
    g, = torch.autograd.grad(got.sum(), x)
    loss, grad, soft, ln_pr, r = definition(x, ids, scores)
    e = (300 + additions(V)) * U
    outside = torch.ones_like(g, dtype=torch.bool).scatter_(1, ids, False)
    tol = soft * (ln_pr.exp() + r) * (2 * e + 8 * U)
    within(g[outside], grad[outside], tol[outside])
    assert float((tol[outside] / grad[outside].abs()).median()) < 1e-3
