"""GPU checks of token_logprobs and distill_topk against the definitions in
float64 (softmax, entropy, stable sort, the divergence and its gradient written
out below), at the sizes, masks and strides where such kernels go wrong, and of
their gradients against the formula and against central differences.

Tolerances.  u = 2^-24 is half a float32 step.  One thread adds at most
V / 128 + 64 terms to each of its two sums before the tree of a block (by 32
threads V / 64, at the sizes below no more), the exponential is
within 2^-22 = 4 u, and an exponent d carries 3 roundings, 3 u |d|, whose mean
under p is at most 3 u ln V.  So ln s is within

    E(V) = u (V / 128 + 64 + 5 ln V + 40)

and a log probability within E + 4 u |logp|; the entropy, ln s plus a mean of
|d|, within (2 + 2 ln V) E.  A gradient element is a sum of terms p * (upstream)
whose exponentials carry the same errors: E times the upstream's magnitude, then
one rounding to the type, finfo.eps / 2 of the value (or half its smallest
subnormal)."""
import math

import pytest
import torch

import autoresearch2_b200 as sf
from autoresearch2_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
INF = math.inf
F64 = torch.float64
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _status():
    yield
    sf.check_status()


def E(V):
    return U * (V / 128 + 64 + 5 * math.log(V) + 40)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def half_step(want, dtype):
    """The rounding to dtype of a value near `want`."""
    fi = torch.finfo(dtype)
    return want.abs() * (fi.eps / 2) * (1 + 2 ** -10) + fi.smallest_normal * fi.eps / 2


# ---------------------------------------------------------------------------
# token_logprobs: the definition
# ---------------------------------------------------------------------------
def log_p(logits, T):
    """ln p in float64; -inf throughout a row of -inf.  The maximum goes first: next
    to logits of 3e38 float64 too would lose the sum's logarithm."""
    x = logits.detach().to(F64)
    m = x.amax(-1, keepdim=True)
    z = (x - torch.where(m == -INF, 0.0, m)) / T
    return torch.where(m == -INF, -INF, z - torch.logsumexp(z, -1, keepdim=True))


def score_want(logits, targets, k, T, ignore=-100):
    lp = log_p(logits, T)
    p = lp.exp()
    skip = targets == ignore
    t = torch.where(skip, 0, targets.long())
    logp = torch.where(skip, 0.0, lp.gather(-1, t[..., None])[..., 0])
    ent = torch.where(skip, 0.0, -torch.special.xlogy(p, p).sum(-1))
    ids = torch.sort(logits.detach().float(), dim=-1, descending=True, stable=True)[1][..., :k]
    top = torch.where(skip[..., None], -INF, lp.gather(-1, ids))
    return logp, ent, torch.where(skip[..., None], -1, ids), top


def score_grad_want(logits, targets, ids, T, g, gh, gt, ignore=-100):
    """(gradient in float64, magnitude of the upstream per row)."""
    lp = log_p(logits, T)
    p = lp.exp()
    H = -torch.special.xlogy(p, p).sum(-1, keepdim=True)
    live = (targets != ignore)[..., None] & (lp > -INF).any(-1, keepdim=True)
    g, gh, gt = (a.to(F64) for a in (g, gh, gt))
    t = torch.where(targets == ignore, 0, targets.long())
    grad = -p * (g + gt.sum(-1))[..., None] - gh[..., None] * (torch.special.xlogy(p, p) + p * H)
    grad.scatter_add_(-1, t[..., None], g[..., None])
    grad.scatter_add_(-1, ids.clamp_min(0), gt)
    mag = (g.abs() + gt.abs().sum(-1) + gh.abs() * (2 + 2 * math.log(p.shape[-1] + 1)))[..., None] / T
    return torch.where(live, grad / T, 0.0), mag


def close(got, want, tol):
    got, want = got.detach().to(F64), want.to(F64)
    fine = torch.isfinite(want)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    err = (got - want)[fine].abs()
    tol = torch.as_tensor(tol, device=got.device, dtype=F64).expand(want.shape)[fine]
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.3g} of the tolerance"


def check_score(logits, targets, k, T=1.0, grad=True):
    V = logits.shape[-1]
    x = logits.detach().requires_grad_(grad)
    r = sf.token_logprobs(x, targets, top_k=k, temperature=T)
    logp, ent, ids, top = score_want(logits, targets, k, T)
    assert r.logp.dtype == r.entropy.dtype == r.top_logp.dtype == torch.float32 and r.top_ids.dtype == torch.int64
    assert r.logp.shape == targets.shape and r.top_ids.shape == (*targets.shape, k)
    close(r.logp, logp, E(V) + 4 * U * torch.where(logp.isfinite(), logp.abs(), 0))
    close(r.entropy, ent, (2 + 2 * math.log(V + 1)) * E(V))
    assert torch.equal(r.top_ids, ids)
    close(r.top_logp, top, E(V) + 4 * U * torch.where(top.isfinite(), top.abs(), 0))
    if not grad:
        return
    g, gh, gt = randn(*targets.shape, seed=7), randn(*targets.shape, seed=8), randn(*targets.shape, k, seed=9)
    outs, gs = [r.logp, r.entropy] + [r.top_logp] * (k > 0), [g, gh] + [gt] * (k > 0)
    got, = torch.autograd.grad(outs, x, gs)
    want, mag = score_grad_want(logits, targets, ids, T, g, gh, gt)
    assert got.dtype == logits.dtype and got.shape == logits.shape
    close(got, want, half_step(want, logits.dtype) + E(V) * mag)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,k,T", [(1, 1, 1, 1.0), (1, 2, 1, 0.5), (3, 7, 7, 2.0), (5, 33, 8, 1.0),
                                        (130, 300, 128, 1.0), (2, 1000, 100, 0.7), (9, 4097, 64, 1.0),
                                        (3, 16391, 1, 1.0), (2, 50257, 65, 1.3), (1, 262147, 128, 1.0),
                                        (400, 2048, 0, 1.0), (600, 5003, 5, 1.0)])
def test_score(dtype, rows, V, k, T):
    logits = randn(rows, V, seed=V + k, scale=3.0, dtype=dtype)
    targets = torch.randint(0, V, (rows,), generator=gen(1), device=DEV)
    check_score(logits, targets, k, T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", [(1301, 771), (1301, 5003), (1190, 16411)])
def test_many_rows(dtype, rows, V):
    """Rows enough for a small block each."""
    x = randn(rows, V, seed=V, scale=2.5, dtype=dtype)
    x[::7, ::2] = -INF
    x[5] = -INF
    t = torch.randint(0, V, (rows,), generator=gen(2), device=DEV)
    t[::5] = -100
    check_score(x, t, 0)
    ids, scores = teacher_list(x, 70)
    ids[3::4, 1::3] = -1
    for tail in ("renorm", "bucket"):
        check_distill(x, ids, scores, tail)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [9, 500, 4500, 60001])
def test_score_ties_go_to_the_lowest_index(dtype, V):
    """Few distinct values (both zeros among them), a constant row, rising and
    falling rows, one row whose largest values stand together."""
    k = min(V, 100)
    x = torch.randint(-2, 3, (6, V), generator=gen(V), device=DEV).float()
    x[0] = torch.where(torch.rand(V, generator=gen(3), device=DEV) < 0.5, -0.0, 0.0)
    x[1] = 1.25
    x[2] = torch.arange(V, device=DEV) % 1000 / 8.0
    x[3] = -(torch.arange(V, device=DEV) / V * 64)
    x[4, V // 2:V // 2 + k] = 7.0
    check_score(x.to(dtype), torch.arange(6, device=DEV) % V, k)


def test_score_sorted_rows_put_every_alternative_in_one_place():
    """Rows sorted either way, and long runs of larger values: the alternatives
    stand in few threads' shares of the row."""
    V = 70003
    x = torch.sort(randn(3, V, seed=4), dim=-1)[0]
    x[1] = x[1].flip(0)
    x[2] = randn(V, seed=5)
    x[2, 30000:50000] += 100.0
    check_score(x, torch.tensor([0, V - 1, 30001], device=DEV), 128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [17, 3001, 40960])
def test_score_masked_rows(dtype, V):
    """Rows of -inf alone, of one or a few finite logits, of the type's lowest
    value alone, and of a mask by it."""
    x = randn(6, V, seed=V, scale=2.0, dtype=dtype)
    low = torch.finfo(dtype).min
    x[0] = -INF
    x[1] = -INF
    x[1, V // 3] = 1.5
    x[2, torch.rand(V, generator=gen(6), device=DEV) < 0.9] = -INF
    x[2, 0] = 0.25
    x[3] = low
    x[4, 1:] = low
    x[5, V - 1] = -INF
    targets = torch.tensor([0, V // 3, 0, V - 1, 0, V - 1], device=DEV)
    check_score(x, targets, min(V, 70))


def test_score_extreme_float32_logits():
    """Differences beyond float32: the lowest value beside large ones, and low temperatures."""
    x = randn(3, 1000, seed=2)
    x[0, 5], x[0, 6] = 3e38, -3e38
    x[1] = torch.linspace(-3e38, 3e38, 1000, device=DEV)
    check_score(x, torch.tensor([5, 999, 3], device=DEV), 4, grad=False)
    check_score(x[2:], torch.tensor([3], device=DEV), 4, T=1e-3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_score_at_the_limits_of_the_temperature(dtype):
    """So hot that every class is alike; so cold that the largest logit has all."""
    V = 3001
    x = (torch.randperm(V, generator=gen(14), device=DEV) / 1024).repeat(3, 1).to(dtype)
    x[1, 7] = 5.0
    x[:, 90] = 8.0
    t = torch.full((3,), 90, device=DEV)
    x.requires_grad_()
    r = sf.token_logprobs(x, t, top_k=1, temperature=1e30)
    close(r.logp, torch.full((3,), -math.log(V), dtype=F64, device=DEV), torch.tensor(E(V) + 4 * U * math.log(V), device=DEV))
    close(r.entropy, torch.full((3,), math.log(V), dtype=F64, device=DEV), torch.tensor((2 + 2 * math.log(V)) * E(V), device=DEV))
    r = sf.token_logprobs(x, t, top_k=1, temperature=1e-30)
    assert r.logp.tolist() == r.entropy.tolist() == r.top_logp[:, 0].tolist() == [0.0] * 3
    assert r.top_ids[:, 0].tolist() == [90] * 3
    if dtype == torch.float32:  # 1 / T is in the range of the gradient's type
        assert not torch.autograd.grad(r.logp.sum() + r.entropy.sum(), x)[0].any()


@pytest.mark.parametrize("V", [100, 20000])
def test_score_nan_and_inf_rows(V):
    x = randn(3, V, seed=1)
    x[0, V // 2] = math.nan
    x[1, V - 1] = INF
    r = sf.token_logprobs(x, torch.zeros(3, dtype=torch.long, device=DEV), top_k=5)
    assert r.logp[:2].isnan().all() and r.entropy[:2].isnan().all() and r.logp[2].isfinite()
    assert r.top_ids[0, 0] == V // 2 and r.top_ids[1, 0] == V - 1  # NaN above all, then +inf
    assert torch.equal(r.top_ids[0, 1:], torch.sort(torch.nan_to_num(x[0], nan=-INF), descending=True, stable=True)[1][:4])


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_score_rows_left_out_are_not_read(index):
    x = randn(40, 3000, seed=3)
    targets = torch.randint(0, 3000, (40,), generator=gen(2), device=DEV)
    out = torch.arange(40, device=DEV) % 3 == 0
    targets[out] = -100
    check_score(x, targets, 6)
    y = x.clone()
    y[out] = math.nan
    y.requires_grad_()
    a, b = sf.token_logprobs(x, targets, top_k=6), sf.token_logprobs(y, targets.to(index), top_k=6)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    (b.logp.sum() + b.entropy.sum() + b.top_logp[~out].sum()).backward()
    assert bool((y.grad[out] == 0).all()) and bool(y.grad[~out].isfinite().all())
    other = torch.where(out, 7, targets)
    c = sf.token_logprobs(x, other, top_k=6, ignore_index=7)
    assert torch.equal(c.logp[out], torch.zeros(int(out.sum()), device=DEV)) and (c.top_ids[out] == -1).all()


def test_score_target_outside_the_vocabulary():
    x = randn(4, 50, seed=1).requires_grad_()
    for bad in (50, -1, 2 ** 40):
        t = torch.tensor([3, bad, 4, 5], device=DEV)
        r = sf.token_logprobs(x, t)
        assert r.logp.isnan().tolist() == [False, True, False, False] and r.entropy.isfinite().all()
        with pytest.raises(_lib.SparseFFNError, match="outside the vocabulary"):
            sf.check_status()
        g, = torch.autograd.grad(r.logp, x, torch.ones(4, device=DEV))
        assert bool((g[1] == 0).all()) and bool(g.isfinite().all())


def test_score_without_targets_and_without_rows():
    x = randn(2, 3, 100, seed=1)
    r = sf.token_logprobs(x, top_k=4)
    assert r.logp is None and r.top_ids.shape == (2, 3, 4)
    full = sf.token_logprobs(x, torch.zeros(2, 3, dtype=torch.long, device=DEV), top_k=4)
    assert torch.equal(r.entropy, full.entropy) and torch.equal(r.top_logp, full.top_logp)
    e = torch.empty(0, 100, device=DEV, requires_grad=True)
    r = sf.token_logprobs(e, torch.empty(0, dtype=torch.long, device=DEV), top_k=4)
    assert r.logp.shape == (0,) and r.top_ids.shape == (0, 4)
    r.logp.sum().backward()
    assert e.grad.shape == (0, 100)
    one = sf.token_logprobs(x[0, 0], torch.tensor(3, device=DEV), top_k=2)
    assert one.logp.shape == () and one.top_ids.shape == (2,)


def strided(base):
    """Views of one [4, 6, 1024 + pad] tensor, each with its own strides."""
    return {"padded": base[..., :1001], "shifted": base[:, :-1, 3:900], "one_row_each": base[:, 2],
            "first_last": base[:, :, 1:], "transposed_rows": base.transpose(0, 1)[..., :777],
            "expanded": base[:1, :, :640].expand(4, 6, 640), "copied": base.transpose(1, 2),
            "four": base.view(2, 2, 6, -1)[:, :, 1:4, :500]}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(strided(torch.empty(4, 6, 1029))))
def test_strides(dtype, name):
    base = randn(4, 6, 1029, seed=5, scale=2.0, dtype=dtype)
    x = strided(base)[name]
    V = x.shape[-1]
    targets = torch.randint(0, V, x.shape[:-1], generator=gen(1), device=DEV)
    k = min(V, 6)
    check_score(x, targets, k)
    ids = torch.rand(*x.shape[:-1], V, generator=gen(2), device=DEV).argsort(-1)[..., :k]
    check_distill(x, ids, randn(*ids.shape, seed=3), "bucket")


def central_difference(f, x, eps=2 ** -6):
    """Gradient of the float64 sum f(x) at float32 x, by central differences of the kernel's own forward."""
    g = torch.empty_like(x, dtype=F64)
    flat = g.view(-1)
    for i in range(x.numel()):
        hi, lo = x.clone(), x.clone()
        hi.view(-1)[i] += eps
        lo.view(-1)[i] -= eps
        flat[i] = (f(hi) - f(lo)) / (hi.view(-1)[i].double() - lo.view(-1)[i].double())
    return g


def test_score_gradient_against_differences():
    """Step h = 2^-6: the error of the difference is h^2 / 6 of a third derivative
    (below 10 for these weights) plus the forward's E / h."""
    x = randn(2, 19, seed=8)
    t = torch.tensor([3, 17], device=DEV)
    w = randn(2, 2 + 3, seed=9).double()

    def f(z):
        r = sf.token_logprobs(z, t, top_k=3, temperature=1.5)
        return (torch.cat([r.logp[:, None], r.entropy[:, None], r.top_logp], -1).double() * w).sum()

    x.requires_grad_()
    got, = torch.autograd.grad(f(x), x)
    want = central_difference(lambda z: f(z).item(), x.detach())
    close(got, want, 10 * 2 ** -12 / 6 + 60 * E(19) * 2 ** 6)


# ---------------------------------------------------------------------------
# distill_topk: the definition
# ---------------------------------------------------------------------------
def distill_want(logits, ids, scores, tail, T=1.0):
    """(loss, T dL/dx / T, tolerance of each before the type's rounding), float64."""
    V, K = logits.shape[-1], ids.shape[-1]
    lead = logits.shape[:-1]
    lp = log_p(logits, T).reshape(-1, V)
    ids, c = ids.reshape(-1, K).long(), scores.to(F64).reshape(-1, K)
    loss, grad = torch.zeros(lp.shape[0], dtype=F64, device=DEV), torch.zeros_like(lp)
    tol_l, tol_g = torch.zeros_like(loss), torch.zeros_like(loss)
    for r in range(lp.shape[0]):
        ok = (ids[r] >= 0) & (ids[r] < V)
        i, cr, p = ids[r][ok], c[r][ok], lp[r].exp()
        if not bool((cr > -INF).any()):
            continue
        q = torch.softmax(cr, 0) if tail == "renorm" else cr.exp()
        on = torch.zeros(V, dtype=F64, device=DEV).index_add_(0, i, q)
        listed = torch.zeros(V, dtype=torch.bool, device=DEV)
        listed[i] = True
        lq = q.log()
        terms = torch.where(q > 0, q * (lq - lp[r][i]), 0.0)
        loss[r] = terms.sum()
        Q, share = q.sum(), 0.0
        tol_l[r] = (E(V) + K * U) * torch.where(q > 0, q * (4 + lq.abs() + lp[r][i].abs()), 0.0).sum()
        tol_g[r] = E(V) * (1 + q.sum())
        if tail == "bucket":
            rest = 1 - q.sum()
            if rest >= 2.0 ** -20 and not bool(listed.all()):
                pr = p[~listed].sum()
                loss[r] += rest * (rest.log() - pr.log())
                off = (K + 8) * U  # what the rest, one less a sum of K float32 terms, is off
                tol_l[r] += off * (2 + (rest / pr).log().abs()) + rest * E(V) * 4
                if pr > 0:
                    share = rest / pr
                    tol_g[r] += off + rest * E(V) * 4
                Q = Q + rest
        if lp[r].max() > -INF:
            grad[r] = p * (Q - torch.where(listed, 0.0, share)) - on
    return loss.view(lead), (grad / T).view(*lead, V), tol_l.view(lead), (tol_g / T).view(lead)[..., None]


def check_distill(logits, ids, scores, tail, T=1.0, grad=True):
    x = logits.detach().requires_grad_(grad)
    got = sf.distill_topk(x, ids, scores, temperature=T, tail=tail)
    loss, g, tol_l, tol_g = distill_want(logits, ids, scores, tail, T)
    assert got.dtype == torch.float32 and got.shape == logits.shape[:-1]
    close(got, loss, tol_l + U * loss.abs())
    if grad:
        up = randn(*loss.shape, seed=11)
        d, = torch.autograd.grad(got, x, up)
        want = g * up[..., None].double()
        assert d.dtype == logits.dtype and d.shape == logits.shape
        close(d, want, half_step(want, logits.dtype) + tol_g * up[..., None].abs().double())


def teacher_list(logits, K, T=1.0, noise=0.5, seed=12):
    x = logits.float() + randn(*logits.shape, seed=seed, scale=noise)
    r = sf.token_logprobs(x, top_k=K, temperature=T)
    return r.top_ids, r.top_logp


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", ["renorm", "bucket"])
@pytest.mark.parametrize("rows,V,K,T", [(1, 1, 1, 1.0), (2, 3, 2, 1.0), (4, 9, 9, 2.0), (7, 130, 128, 0.7), (33, 1000, 16, 2.0),
                                        (5, 4099, 1, 1.0), (3, 32003, 100, 1.0), (2, 131072, 64, 1.5),
                                        (1, 262147, 128, 1.0), (500, 2100, 7, 1.0)])
def test_distill(dtype, tail, rows, V, K, T):
    x = randn(rows, V, seed=V, scale=2.5, dtype=dtype)
    ids, scores = teacher_list(x, K, T)
    check_distill(x, ids, scores, tail, T)


@pytest.mark.parametrize("tail", ["renorm", "bucket"])
def test_distill_lists_with_gaps(tail):
    """Absent entries, an empty list, scores of -inf, one entry alone, an id
    listed twice, unsorted ids, the first and the last class."""
    V = 700
    x = randn(8, V, seed=1, scale=2.0)
    ids = torch.randint(0, V, (8, 6), generator=gen(2), device=DEV)
    ids[:, 0], ids[:, 1] = 0, V - 1
    scores = torch.log_softmax(randn(8, 9, seed=3), -1)[:, :6].contiguous()
    ids[0, 2:4] = -1
    ids[1] = -1
    scores[2] = -INF
    scores[3, 1:] = -INF
    ids[4, 1:] = -1
    ids[5] = torch.tensor([9, 9, 4, 9, 4, 1], device=DEV)
    ids[6] = torch.arange(6, device=DEV).flip(0)
    check_distill(x, ids, scores, tail)
    r = sf.distill_topk(x, ids, scores, tail=tail)
    assert r[1] == 0 and r[2] == 0


@pytest.mark.parametrize("tail", ["renorm", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_masked_students(tail, dtype):
    """Classes of the list without probability under the student (loss +inf where the
    teacher gives weight), none off the list, and the type's lowest value."""
    V = 300
    x = randn(5, V, seed=4, dtype=dtype)
    ids = torch.arange(8, device=DEV).repeat(5, 1) * 3
    scores = torch.log_softmax(randn(5, 20, seed=5), -1)[:, :8].contiguous()
    x[0, 3] = -INF
    x[1, 200:] = -INF
    x[2, 30:] = torch.finfo(dtype).min
    x[3, 6] = -INF
    scores[3, 2] = -INF  # weight 0 there: no term
    check_distill(x, ids, scores, tail)
    assert sf.distill_topk(x, ids, scores, tail=tail)[0] == INF


def test_distill_rest_of_a_confident_teacher():
    """A listed mass of one to the last bits: the rest below 2^-20 is none; a rest of
    10^-4 is told from the student's own mass off the list."""
    V = 2000
    x = randn(3, V, seed=6)
    x[:, :4] += 20.0
    ids = torch.arange(4, device=DEV).repeat(3, 1)
    p = torch.tensor([0.5, 0.25, 0.125, 0.125], device=DEV)
    scores = torch.stack([p, p * (1 - 1e-4), p * (1 - 3e-7)]).log()
    check_distill(x, ids, scores, "bucket")


def test_distill_scores_and_ids_of_other_types():
    x = randn(4, 500, seed=2)
    ids, scores = teacher_list(x, 8)
    for dt in (torch.bfloat16, torch.float16):
        check_distill(x, ids, scores.to(dt), "renorm")
        check_distill(x, ids.int(), scores.to(dt), "bucket")


def test_distill_id_outside_the_vocabulary_is_absent():
    x = randn(2, 60, seed=2)
    ids = torch.tensor([[5, 60, 7], [1, 2, -5]], device=DEV)
    scores = torch.log_softmax(randn(2, 5, seed=1), -1)[:, :3].contiguous()
    got = sf.distill_topk(x, ids, scores, tail="bucket")
    with pytest.raises(_lib.SparseFFNError, match="outside the vocabulary"):
        sf.check_status()
    gone = ids.clone()
    gone[0, 1] = gone[1, 2] = -1
    assert torch.equal(got, sf.distill_topk(x, gone, scores, tail="bucket"))


@pytest.mark.parametrize("tail", ["renorm", "bucket"])
def test_distill_gradient_against_differences(tail):
    x = randn(2, 17, seed=8)
    ids = torch.tensor([[3, 16, 5], [0, 1, 1]], device=DEV)
    scores = torch.log_softmax(randn(2, 9, seed=1), -1)[:, :3].contiguous()
    f = lambda z: sf.distill_topk(z, ids, scores, temperature=1.3, tail=tail).double().sum()  # noqa: E731
    x.requires_grad_()
    got, = torch.autograd.grad(f(x), x)
    want = central_difference(lambda z: f(z).item(), x.detach())
    close(got, want, 10 * 2 ** -12 / 6 + 60 * E(17) * 2 ** 6)


def test_distill_without_rows():
    e = torch.empty(0, 100, device=DEV, requires_grad=True)
    r = sf.distill_topk(e, torch.empty(0, 3, dtype=torch.long, device=DEV), torch.empty(0, 3, device=DEV))
    r.sum().backward()
    assert r.shape == (0,) and e.grad.shape == (0, 100)


# ---------------------------------------------------------------------------
# How they are run
# ---------------------------------------------------------------------------
def step(x, t, ids, scores):
    r = sf.token_logprobs(x, t, top_k=5)
    loss = sf.distill_topk(x, ids, scores, tail="bucket")
    g, = torch.autograd.grad([r.logp, r.entropy, loss], x, [torch.ones_like(loss)] * 3)
    return r.logp.detach(), r.top_ids, loss.detach(), g


def inputs(seed, rows=50, V=3001):
    x = randn(rows, V, seed=seed, scale=2.0, dtype=torch.bfloat16)
    ids, scores = teacher_list(x, 9)
    return x, torch.randint(0, V, (rows,), generator=gen(seed), device=DEV), ids, scores


def test_equal_inputs_give_equal_bits_on_any_stream():
    a = inputs(1)
    a[0].requires_grad_()
    want = step(*a)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:  # two calls at once
        with torch.cuda.stream(s):
            got.append(step(*a))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(g, want))


def test_captured_and_replayed_on_new_inputs():
    a, b = inputs(1), inputs(2)
    a[0].requires_grad_()
    step(*a)  # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*a)
    for src in (b, inputs(3)):
        with torch.no_grad():
            for dst, s in zip(a, src):
                dst.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        x = src[0].detach().requires_grad_()
        assert all(torch.equal(p, q) for p, q in zip(out, step(x, *src[1:])))


def test_offsets_beyond_32_bits():
    """45000 x 50304 logits, 2.26e9 elements: the last rows' values and gradients.
    (Not the bits of a small call: few rows are shared out among more threads.)"""
    R, V = 45000, 50304
    x = torch.zeros(R, V, device=DEV, dtype=torch.bfloat16)
    tail = randn(3, V, seed=1, scale=2.0, dtype=torch.bfloat16)
    x[-3:] = tail
    t = torch.full((R,), -100, device=DEV)
    t[-3:] = torch.tensor([0, V - 1, 77], device=DEV)
    ids, scores = torch.full((R, 4), -1, device=DEV), torch.zeros(R, 4, device=DEV)
    ids[-3:], scores[-3:] = teacher_list(tail, 4)
    x.requires_grad_()
    got = step(x, t, ids, scores)
    one = torch.ones(3, device=DEV)
    logp, ent, top, _ = score_want(tail, t[-3:], 5, 1.0)
    loss, g, tol_l, tol_g = distill_want(tail, ids[-3:], scores[-3:], "bucket")
    close(got[0][-3:], logp, E(V) + 4 * U * logp.abs())
    assert torch.equal(got[1][-3:], top)
    close(got[2][-3:], loss, tol_l + U * loss.abs())
    g2, mag = score_grad_want(tail, t[-3:], top, 1.0, one, one, torch.zeros(3, 5, device=DEV))
    eps = torch.finfo(torch.bfloat16).eps  # each of the two gradients is rounded, then their sum
    close(got[3][-3:], g + g2, eps * (g.abs() + g2.abs()) * 1.01 + tol_g + E(V) * mag)
    # rows left out take the entropy's upstream too: nothing of it reaches them
    assert not bool(got[3][:-3].any())


def test_two_devices_argument_checks_need_no_second_device():
    x = randn(2, 10)
    with pytest.raises(ValueError, match="CUDA"):
        sf.token_logprobs(x, torch.zeros(2, dtype=torch.long))


def test_library_ops():
    ops = torch.ops.sparseffn
    x, t, ids, scores = inputs(4, rows=6, V=200)
    torch.library.opcheck(ops.token_logprobs.default, (x, t, 3, 1.5, -100),
                          test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(ops.distill_topk.default, (x, ids, scores, 1.0, "bucket"),
                          test_utils=("test_schema", "test_faketensor"))

    def f(x, t, ids, scores):
        r = sf.token_logprobs(x, t, top_k=3)
        return (sf.distill_topk(x, ids, scores) - r.logp + 0.1 * r.entropy).sum() + 0 * r.top_ids.sum()

    torch._dynamo.reset()
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    want, got = f(a, t, ids, scores), torch.compile(f, backend="aot_eager", fullgraph=True)(b, t, ids, scores)
    want.backward()
    got.backward()
    torch._dynamo.reset()
    assert torch.equal(want, got) and torch.equal(a.grad, b.grad)


def test_gradients_are_not_differentiable_again():
    x, t, ids, scores = inputs(5, rows=4, V=50)
    x.requires_grad_()
    for out in (sf.token_logprobs(x, t).logp, sf.distill_topk(x, ids, scores)):
        with pytest.raises(RuntimeError, match="not differentiable again"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_logits_changed_before_the_backward_are_refused():
    x, t, _, _ = inputs(5, rows=4, V=50)
    x.requires_grad_()
    y = x * 1
    out = sf.token_logprobs(y, t).logp.sum()
    with torch.no_grad():
        y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_ops_refuse_what_the_functions_refuse():
    ops = torch.ops.sparseffn
    x, t, ids, scores = inputs(5, rows=4, V=50)
    logp, ent, top, _, stats = ops.token_logprobs(x, t, 3, 1.0, -100)
    loss, kept = ops.distill_topk(x, ids, scores, 1.0, "bucket")
    bad = [lambda: ops.token_logprobs(x, t[:3], 3, 1.0, -100), lambda: ops.token_logprobs(x, t, 51, 1.0, -100),
           lambda: ops.token_logprobs_bwd(x, t, top, ent, stats[:2], logp, None, None, 1.0, -100),
           lambda: ops.token_logprobs_bwd(x, t, top[:, :2], ent, stats, None, None, logp[:, None].expand(4, 3)[:, :3][:2], 1.0, -100),
           lambda: ops.token_logprobs_bwd(x, t, top, ent, stats, logp.half(), None, None, 1.0, -100),
           lambda: ops.distill_topk(x, ids[:2], scores, 1.0, "bucket"),
           lambda: ops.distill_topk_bwd(x, ids, scores, kept[:, :2], loss, 1.0, "bucket"),
           lambda: ops.distill_topk_bwd(x, ids, scores, kept, loss[:1], 1.0, "bucket")]
    for f in bad:
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("rows", [3, 2000])
def test_ids_listed_twice_give_equal_bits(rows):
    """Whichever entry's thread comes first: the loss and its gradient are the same bits each time."""
    x = randn(rows, 5000, seed=1, scale=2.0, dtype=torch.bfloat16).requires_grad_()
    ids = torch.randint(0, 40, (rows, 100), generator=gen(2), device=DEV) * 120
    scores = torch.log_softmax(randn(rows, 120, seed=3), -1)[:, :100].contiguous()
    runs = []
    for _ in range(8):
        loss = sf.distill_topk(x, ids, scores, tail="bucket")
        runs.append((loss.detach(), torch.autograd.grad(loss.sum(), x)[0]))
    assert all(torch.equal(a, runs[0][0]) and torch.equal(b, runs[0][1]) for a, b in runs)
    check_distill(x[:3], ids[:3], scores[:3], "bucket")


@pytest.mark.parametrize("rows,V", [(3, 50000), (1300, 257)])
def test_calls_without_gradients_give_the_bits_of_calls_with(rows, V):
    x = randn(rows, V, seed=51, scale=2.0, dtype=torch.bfloat16)
    t = torch.randint(0, V, (rows,), generator=gen(52), device=DEV)
    ids, scores = teacher_list(randn(rows, V, seed=53, scale=2.0), 9)
    leaf = x.clone().requires_grad_()
    for call in (lambda x: sf.token_logprobs(x, t, top_k=7), lambda x: (sf.distill_topk(x, ids, scores, tail="bucket"),)):
        kept = call(leaf)
        with torch.no_grad():
            inside = call(leaf)
        for got in (call(x), inside):
            for a, b in zip(got, kept):
                assert not a.requires_grad and torch.equal(a, b)
