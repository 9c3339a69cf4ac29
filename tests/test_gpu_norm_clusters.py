"""GPU checks of residual_norm on rows that several blocks share (wider than
4096): neighbouring rows of very different size, so that a sum that belongs to
another row or came too late shows, over and over with equal bits."""
import pytest
import torch

import autoresearch2_b200 as sf
from test_gpu_norms import BF16, F32, check, close, params, randn, want_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def uneven(rows, D, seed, dtype):
    size = torch.tensor([1.0, 64.0, 0.125, 1024.0, 4.0], device=DEV).repeat(-(-rows // 5))[:rows, None]
    return (randn(rows, D, seed=seed) * size).to(dtype)


@pytest.mark.parametrize("xt,yt,D", [(BF16, BF16, 4104), (F32, BF16, 8192), (F32, F32, 8200), (BF16, BF16, 16384),
                                     (F32, F32, 9001)])
def test_uneven_neighbours(xt, yt, D):
    rows = 700
    pre, post, gate = params(D)
    check(uneven(rows, D, 1, xt), uneven(rows, D, 2, yt), pre, post, gate, True, 0.5)


@pytest.mark.parametrize("D", [4104, 8192, 16384])
def test_equal_bits_time_after_time(D):
    rows = 1500
    x, y = uneven(rows, D, 3, BF16), uneven(rows, D, 4, BF16)
    pre, post, gate = params(D)
    leaves = [t.requires_grad_() for t in (x, y, pre, post, gate)]
    dx, dh = uneven(rows, D, 5, BF16), uneven(rows, D, 6, BF16)

    def once():
        a, h = sf.residual_norm(x, y, pre, post, gate, True, 0.5)
        return [a, h, *torch.autograd.grad([a, h], leaves, [dx, dh])]

    first = once()
    assert all(bool(t.isfinite().all()) for t in first)
    for _ in range(20):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))
    sf.check_status()


@pytest.mark.parametrize("rows,D,xt,yt", [(3000, 16384, BF16, BF16), (4000, 8193, F32, F32), (5003, 12000, F32, BF16)])
def test_weight_gradients_of_many_rows(rows, D, xt, yt):
    """Rows wider than 8192 go to 32 clusters at most, so a thread adds up rows / 32 of
    them in float32 (fma: one rounding a term); the clusters' sums are joined in 64
    bits.  Beside the terms' own C u M (test_gpu_norms) that is (rows / 32 + 2) u M."""
    x, y = randn(rows, D, seed=1, dtype=xt), randn(rows, D, seed=2, dtype=yt)
    pre, post, gate = params(D)
    leaves = [t.requires_grad_() for t in (pre, post, gate)]
    dxn, dh = randn(rows, D, seed=3, dtype=xt), randn(rows, D, seed=4, dtype=yt)
    a, h = sf.residual_norm(x, y, pre, post, gate, True, 0.5)
    got = torch.autograd.grad([a, h], leaves, [dxn, dh])
    want = {name: [0.0, 0.0] for name in ("dpre", "dpost", "dgate")}
    for at in range(0, rows, 500):
        part = slice(at, at + 500)
        g = gate.detach().expand(min(500, rows - at), D)
        values = want_norm(x[part], y[part], pre, post, g, True, 0.5, 1e-6, dxn[part], dh[part])
        for name, sums in want.items():
            for i in range(2):
                sums[i] = sums[i] + values[name][i].sum(0)
    for g, name in zip(got, want):
        close(g, *want[name], extra=rows / 32 + 2)
    sf.check_status()
