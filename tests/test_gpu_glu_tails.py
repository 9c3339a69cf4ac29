"""GPU checks of the gated block's activations far down their tails, where the
results are tiny but still normal numbers of bfloat16: relative to their own size.

A block of one feature and weights of 1 computes x act(x), and its gradient by x is
act(x) + x act'(x) times dy (Wu as well being 1).  act and act' of SiLU are within
2^-21 max(|x|, 2) of themselves for x >= -91, 2^-14.5 at most there, and act' = s +
a (1 - s) by two more float32 roundings of values as large as |x| times itself, below
2^-16; the products' float32 roundings are below 2^-21.  The forward rounds h once
and y is h; the backward rounds dg and du and then their sum dx, of which du is
the smaller one by 1 / |x|."""
import pytest
import torch

import autoresearch2_b200 as sf

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64, BF16 = torch.float64, torch.bfloat16


def half(t):
    return torch.finfo(t).eps / 2 * (1 + 2 ** -8)


def points(T):
    """x in [-91, 12], thickest where e^x leaves float32's normal numbers."""
    a, b = torch.linspace(-91, -85, T - T // 2), torch.linspace(-85, 12, T // 2)
    return torch.cat([a, b]).to(BF16)[:, None].to(DEV)


@pytest.mark.parametrize("T", [12, 40, 64, 1537])
def test_silu_keeps_small_tails(T):
    x = points(T)
    one = torch.ones(1, 1, device=DEV, dtype=BF16)
    y = sf.gated_ffn(x, one, one, one, "silu").to(F64)
    x = x.to(F64)
    want = x * x / (1 + torch.exp(-x))
    assert ((y - want).abs() <= (half(BF16) + 2 ** -14) * want.abs()).all()


@pytest.mark.parametrize("T", [12, 40, 1537])
def test_gradients_keep_them_too(T):
    x = points(T).requires_grad_()
    one = torch.ones(1, 1, device=DEV, dtype=BF16)
    y = sf.gated_ffn(x, one, one, one, "silu")
    dx = torch.autograd.grad(y, x, torch.ones_like(y))[0].to(F64)
    x = x.detach().to(F64)
    s = 1 / (1 + torch.exp(-x))
    a, d = x * s, s + x * s * (1 - s)
    dg, du = x * d, a
    tol = half(BF16) * (dg + du).abs() + (half(BF16) + 2 ** -13) * (dg.abs() + du.abs())
    assert ((dx - dg - du).abs() <= tol).all()


def test_silu_far_out():
    """Beyond: zeros on the left, x on the right, infinities and NaN as float64 has them."""
    x = torch.tensor([-1e4, -200, -140, 100, 1e4, float("nan"), float("-inf"), float("inf")], dtype=BF16, device=DEV)
    one = torch.ones(1, 1, device=DEV, dtype=BF16)
    for T in (8, 40, 160):
        y = sf.gated_ffn(x.repeat(T // 8)[:, None], one, one, one, "silu")[:8, 0]
        assert (y[:3] == 0).all() and torch.equal(y[3:5], (x[3:5].to(F64) ** 2).to(BF16)) and torch.isnan(y[5:7]).all() and y[7] == float("inf")
