"""GPU checks of token_logprobs and distill_topk on confident rows: one peak over
noise, wherever it stands, against float64.

Bounds, u = 2^-24.  With the row's maximum as reference the peak is exactly 1 in
s = sum e^d and 0 in w = sum e^d d, and S = s - 1 is small.  To the accumulator
that holds the peak every later addition, of a thread or of the tree, costs at
most u (s < 2): a thread adds at most V / 64 terms to each of its accumulators (32
threads, two accumulators; rows above 32 KB have at least 64 threads, V / 128),
the tree 1 + 5 + 16 + 8 more.  So with n of these additions

    |error of s| <= n u + S e,    e = (300 + n) u

e the relative error of one small term: its exponent, at most 40 in base 2, has 3
roundings (3 u 40 ln 2 = 83 u), the rescaling by a new maximum the same, each of
its steps and the exponential itself some 6 u, and n additions.  ln s, below S, has
2 u of its own, and ln p = -ln s at the peak.  H = ln s + |w| / s adds terms of one
sign: |w| <= H carries 2 e (e^d and d), n u, and the factor 1 / s.
The bounds do not grow with what the peak stands above the noise: a reference that
lags behind the maximum costs up to 100 u here, whatever n."""
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


def peaked(rows, V, height, dtype, seed, T=1.0):
    """(logits, places): normal noise and in each row one element `height` above zero, a
    third of them among the last, a third among the first elements."""
    x = torch.randn(rows, V, generator=gen(seed), device=DEV)
    at = torch.randint(0, V, (rows,), generator=gen(seed + 1), device=DEV)
    at[::3] = V - 1 - at[::3] % 9
    at[1::3] = at[1::3] % 9
    x[torch.arange(rows, device=DEV), at] = height
    return (x * T).to(dtype), at


def additions(V, dtype):
    small = V * torch.finfo(dtype).bits // 8 <= 32768
    return -(-V // (64 if small else 128)) + 30


def within(got, want, tol):
    worst = ((got.detach().to(F64) - want).abs() / tol).max()
    assert float(worst) <= 1.0, f"worst {float(worst):.3g} of the tolerance"


CASES = [(24, 1024, 20.0), (1300, 1024, 20.0), (1300, 1024, 15.0), (24, 8192, 18.0), (1300, 8192, 18.0), (24, 50304, 22.0),
         (24, 50304, 18.0), (3, 200003, 19.0), (2000, 301, 17.0), (1, 100, 21.0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("k", [0, 5])
@pytest.mark.parametrize("rows,V,height", CASES)
def test_scores_of_confident_rows(rows, V, height, k, dtype):
    for T in (1.0, 0.5):
        x, at = peaked(rows, V, height, dtype, V, T)
        x.requires_grad_()
        r = sf.token_logprobs(x, at, top_k=k, temperature=T)
        lp = torch.log_softmax(x.detach().to(F64) / T, -1)
        logp = lp.gather(1, at[:, None])[:, 0]
        H = -(lp.exp() * lp).sum(-1)
        S, n = torch.expm1(-logp), additions(V, dtype)
        e = (300 + n) * U
        tol = n * U + S * e + 2 * U * S
        within(r.logp, logp, tol)
        within(r.entropy, H, tol + H * (3 * e + n * U))
        assert float(r.logp.detach().max()) <= 0.0 and float(r.entropy.detach().min()) >= 0.0
        if k:
            assert torch.equal(r.top_ids[:, 0], at) and torch.equal(r.top_logp[:, 0], r.logp)
        if dtype == torch.float32:  # the gradient at the peak, 1 - p: p = 1 / s and two roundings
            g, = torch.autograd.grad(r.logp, x, torch.ones_like(r.logp))
            within(g.gather(1, at[:, None])[:, 0], -torch.expm1(logp) / T, (tol + 4 * U) / T)


@pytest.mark.parametrize("rows,V,height", [(40, 1024, 20.0), (1300, 8192, 18.0)])
def test_statistics_hold_the_maximum(rows, V, height):
    """The op's statistics are the row's largest logit itself and the sum from it."""
    x, at = peaked(rows, V, height, torch.float32, 5)
    for k in (0, 3):
        stats = torch.ops.sparseffn.token_logprobs(x, at, k, 1.0, -100)[4]
        assert torch.equal(stats[:, 0], x.amax(-1)) and float(stats[:, 1].min()) >= 1.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tail", ["renorm", "bucket"])
@pytest.mark.parametrize("rows,V,height", [(24, 1024, 20.0), (1300, 1024, 16.0), (1300, 8192, 18.0)])
def test_confident_students(rows, V, height, tail, dtype):
    """The loss from a teacher as confident in the same class: errors of ln p as above,
    4 u of each |ln p| and |ln q|, and q's own (4 + |ln q|) u."""
    x, at = peaked(rows, V, height, dtype, V + 1)
    teacher, _ = peaked(rows, V, height - 2.0, torch.float32, V + 1)
    scores, ids = torch.topk(torch.log_softmax(teacher.to(F64), -1), 8, dim=-1)
    scores = scores.float()
    c = scores.to(F64)
    lp = torch.log_softmax(x.to(F64), -1)
    lnq = torch.log_softmax(c, -1) if tail == "renorm" else c
    q, on = lnq.exp(), lp.gather(1, ids)
    loss = (q * (lnq - on)).sum(-1)
    S, n = torch.expm1(-lp.amax(-1)), additions(V, dtype)
    tol = n * U + S * (302 + n) * U + (q * U * (4 * on.abs() + 4 * lnq.abs() + (4 + lnq.abs()) * (lnq - on).abs())).sum(-1) + 8 * U
    if tail == "bucket":
        rest = 1.0 - q.sum(-1)
        off = lp.scatter(1, ids, -math.inf).logsumexp(-1)
        rest = torch.where(rest < 2.0 ** -20, 0.0, rest)
        loss = loss + torch.where(rest > 0, rest * (rest.log() - off), 0.0)
        # the rest's own error: of a float32 sum of eight terms (16 u), as of a longer one
        tol = tol + torch.where(rest > 0, 16 * U * (rest.log() - off).abs() + rest * (300 + n) * U, 0.0)
    within(sf.distill_topk(x, ids, scores, tail=tail), loss, tol)
