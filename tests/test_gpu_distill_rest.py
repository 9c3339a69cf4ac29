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


def check_bucket(x, ids, scores, T):
    """Loss and gradient.  A logarithm l of a probability is within (300 + n) u + 4 u |l|
    (its sum's logarithm; its exponent's three roundings and the last difference), q = e^c
    within (4 + |c|) u of itself; the terms' products and sums take 20 u of them."""
    x = x.detach().requires_grad_()
    got = sf.distill_topk(x, ids, scores, temperature=T, tail="bucket")
    g, = torch.autograd.grad(got.sum(), x)
    loss, grad, soft, ln_pr, r = definition(x, ids, scores, T)
    lp = torch.log_softmax(x.detach().to(F64) / T, -1).gather(1, ids)
    c = scores.to(F64)
    q, n = c.exp(), additions(x.shape[-1])
    e = (300 + n) * U
    tol = (q * (e + 4 * U * lp.abs() + 4 * U * c.abs() + (24 + c.abs()) * U * (c - lp).abs())).sum(-1, keepdim=True)
    ln_r = torch.where(r > 0, r.log(), 0.0)
    tol = tol + r * (e + 4 * U * ln_pr.abs() + 24 * U * (ln_r - ln_pr).abs())
    assert bool(loss.isfinite().all())
    within(got, loss, tol[:, 0])
    tol = soft * (ln_pr.exp() + r) * (2 * e + 8 * U)
    on = lp.exp() * (2 * e + 4 * U * lp.abs()) + q * (8 + 2 * c.abs()) * U
    within(g, grad, tol.scatter(1, ids, on) / T, x.dtype)
    return got, g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1.0, 0.05])
@pytest.mark.parametrize("gap", [20.0, 80.0, 90.0, 104.0, 300.0, 1000.0])
@pytest.mark.parametrize("rows,V,K", [(5, 700, 6), (1200, 257, 20), (2, 50304, 64)])
def test_students_far_from_the_rest(rows, V, K, gap, T, dtype):
    """The listed classes stand `gap` nats above the others: the mass off the list is
    far below float32's smallest, its logarithm and the shares in it are not."""
    ids, scores = a_list(rows, V, K, 1e-3 if gap < 100 else 0.2, 7)
    x = randn(rows, V, seed=9).scatter_(1, ids, gap + randn(rows, K, seed=10)) * T
    check_bucket(x.to(dtype), ids, scores, T)


@pytest.mark.parametrize("gap", [90.0, 500.0])
def test_students_far_below_the_rest(gap):
    """The other way about: the listed classes have nothing, and no term is lost."""
    ids, scores = a_list(4, 900, 9, 0.01, 21)
    x = randn(4, 900, seed=22).scatter_(1, ids, -gap + randn(4, 9, seed=23))
    check_bucket(x, ids, scores, 1.0)


def test_a_rest_that_the_student_cannot_have():
    """Nothing but -inf off the list: +inf, gradients of the list's classes alone; a NaN
    stays one."""
    ids, scores = a_list(3, 200, 5, 0.1, 31)
    x = torch.full((3, 200), -math.inf, device=DEV).scatter_(1, ids, randn(3, 5, seed=32))
    x[1, ids[1, 2]] = math.nan
    x[2] = -math.inf
    x.requires_grad_()
    got = sf.distill_topk(x, ids, scores, tail="bucket")
    assert got[0] == math.inf and got[1].isnan() and got[2] == math.inf
    g, = torch.autograd.grad(got.sum(), x)
    outside = torch.ones(200, dtype=torch.bool, device=DEV)
    outside[ids[0]] = False
    p, q = torch.softmax(x.detach()[0].to(F64), -1)[ids[0]], scores[0].to(F64).exp()
    assert bool((g[0][outside] == 0).all()) and bool((g[2] == 0).all())
    within(g[0][ids[0]], p - q, 40 * U * (p + q))


def test_gradient_of_a_far_student_against_differences():
    """Central differences of the loss's own value 30 nats apart, h = 2^-6: the third
    derivative of the loss is at most 6, and its rounding 60 (300 + n) u a difference."""
    ids, scores = a_list(1, 12, 4, 0.25, 41)
    x = randn(1, 12, seed=42).scatter_(1, ids, 30.0 + randn(1, 4, seed=43)).requires_grad_()
    f = lambda z: float(sf.distill_topk(z, ids, scores, tail="bucket"))  # noqa: E731
    g, = torch.autograd.grad(sf.distill_topk(x, ids, scores, tail="bucket").sum(), x)
    base, h = x.detach(), 2.0 ** -6
    want = torch.zeros_like(base, dtype=F64)
    for j in range(12):
        step = torch.zeros_like(base)
        step[0, j] = h
        want[0, j] = (f(base + step) - f(base - step)) / (2 * h)
    within(g, want, torch.tensor(h * h + 60 * 340 * U / (2 * h), dtype=F64, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_student_near_its_teacher(dtype):
    """Equal logits: s = V and s_off = V - K are exact, ln p = -ln V, and the loss, some
    10^-4 and less, turns on ln(q_r / p_r) near 0.  Its argument has three roundings, the
    rest one, the logarithm and the product one each: 6 u.  The listed classes have a
    share near K / V of the terms, each within 60 u (ln V, c and their difference)."""
    for V in list(range(300, 320)) + [1000 + 37 * i for i in range(20)] + [20011 * i for i in range(1, 8)]:
        K = 4
        x = torch.zeros(3, V, device=DEV, dtype=dtype)
        ids = torch.arange(K, device=DEV).repeat(3, 1) * 7
        scores = (torch.tensor([[0.9], [1.0], [1.2]], device=DEV, dtype=F64) / V).log().float().expand(3, K).contiguous()
        got = sf.distill_topk(x, ids, scores, tail="bucket")
        loss = definition(x, ids, scores)[0]
        within(got, loss, torch.tensor(6 * U + 1.2 * K / V * 60 * U, dtype=F64, device=DEV))


@pytest.mark.parametrize("rows,V,dtype", [(600, 1400000, torch.bfloat16), (600, 700001, torch.bfloat16), (593, 1000000, torch.float32),
                                          (200, 1400000, torch.bfloat16), (3, 1400000, torch.float32)])
def test_the_longest_lists_of_bits(rows, V, dtype):
    """Up to the largest vocabulary, with one block to a row and with several."""
    K, check = 32, 3
    ids, scores = (t.repeat(-(-rows // check), 1)[:rows].contiguous() for t in a_list(check, V, K, 0.3, 51))
    ids[:, 0], ids[:, 1] = 0, V - 1
    x = torch.empty(rows, V, device=DEV, dtype=dtype)
    for at in range(0, rows, check):
        x[at:at + check] = randn(min(check, rows - at), V, seed=at % 9)
    got = sf.distill_topk(x, ids, scores, tail="bucket")
    for at in (0, rows - check):
        part = slice(at, at + check)
        loss, *_ = definition(x[part], ids[part], scores[part])
        lp = torch.log_softmax(x[part].to(F64), -1).gather(1, ids[part])
        c, e = scores[part].to(F64), (300 + additions(V)) * U
        tol = (c.exp() * (e + 30 * U * (lp.abs() + c.abs() + 1))).sum(-1) + e + 40 * U
        within(got[part], loss, tol)
    assert bool(got.isfinite().all())
