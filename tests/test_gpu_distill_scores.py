"""GPU checks of distill_topk's renorm on scores that are no log probabilities: a
teacher's logits, of any size, give what their softmax over the list gives.

u = 2^-24.  c - max c has one rounding of the scores' distance, the sum's logarithm
4 u and its terms 6 u each over at most K additions, the difference and the
exponential 6 u: q is within (K + 20 + 2 |ln q|) u of itself, however large the
scores are; an error of q counts (|ln q - ln p| + 1) times in the loss.  ln p is within
(300 + n) u + 4 u |ln p| for n additions to an accumulator."""
import pytest
import torch

import autoresearch2_b200 as sf

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F64 = torch.float64


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


@pytest.mark.parametrize("offset", [0.0, -200.0, 200.0, -3000.0, 1e4])
@pytest.mark.parametrize("rows,V,K", [(6, 50, 1), (9, 1000, 16), (1300, 700, 128), (2, 50304, 64)])
def test_logits_as_scores(rows, V, K, offset):
    x = randn(rows, V, seed=1).mul_(2.5).requires_grad_()
    ids = torch.rand(rows, V, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).argsort(-1)[:, :K].contiguous()
    scores = randn(rows, K, seed=3) * 3 + offset
    got = sf.distill_topk(x, ids, scores)
    g, = torch.autograd.grad(got.sum(), x)
    lp = torch.log_softmax(x.detach().to(F64), -1)
    on, lnq = lp.gather(1, ids), torch.log_softmax(scores.to(F64), -1)
    q = lnq.exp()
    n = V // 64 + 40
    e_q, e_p = (K + 20 + 2 * lnq.abs()) * U, (300 + n) * U + 4 * U * on.abs()
    err = (got.detach().to(F64) - (q * (lnq - on)).sum(-1)).abs()
    tol = (q * (e_q * ((lnq - on).abs() + 1) + e_p)).sum(-1) + 2 * K * U
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3g} of the tolerance"
    p = lp.exp()
    want = p.scatter_add(1, ids, -q)
    err = (g.to(F64) - want).abs()
    tol = (p * ((300 + n) * U + 4 * U * lp.abs())).scatter_add(1, ids, q * e_q) + 2 * U * want.abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3g} of the tolerance"


def test_far_entries_of_a_list():
    """Scores 200 apart: the far ones weigh nothing; all near -200: what they are among themselves."""
    x = randn(4, 60, seed=5)
    ids = torch.arange(3, device=DEV).repeat(4, 1)
    scores = torch.tensor([[0.0, -200.0, -190.0], [-192.25, -191.5, -1e30], [1e30, 0.0, 5.0], [-3e38, -3e38, -3e38]], device=DEV)
    lp = torch.log_softmax(x.to(F64), -1)[:, :3]
    lnq = torch.log_softmax(scores.to(F64), -1)
    q = lnq.exp()
    want = torch.where(q > 0, q * (lnq - lp), 0.0).sum(-1)
    err = (sf.distill_topk(x, ids, scores).to(F64) - want).abs()
    assert bool((err <= 400 * U * (1 + want.abs())).all())
