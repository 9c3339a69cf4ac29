"""GPU checks that infinities and NaN in one row change no other row's results: bit for
bit the ones of the same call with finite numbers in their place."""
import pytest
import torch

import autoresearch2_b200 as sf

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16
BAD = (2, 4)


def randn(*shape, seed=0, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * scale).to(dtype)


def spoiled(t):
    t = t.clone()
    t[BAD[0], 5], t[BAD[1], 1] = float("nan"), float("inf")
    return t


def rest(T):
    return [i for i in range(T) if i not in BAD]


@pytest.mark.parametrize("T", [6, 16, 20, 48, 64, 140, 300])
@pytest.mark.parametrize("D,F", [(64, 96), (101, 137), (520, 1000)])
def test_gated_ffn(T, D, F):
    x, Wg, Wu, W2, dy = (randn(*s, seed=i, scale=c) for i, (s, c) in enumerate(
        [((T, D), 1), ((F, D), D ** -0.5), ((F, D), D ** -0.5), ((D, F), F ** -0.5), ((T, D), 1)]))
    y, bad = sf.gated_ffn(x, Wg, Wu, W2), sf.gated_ffn(spoiled(x), Wg, Wu, W2)
    assert torch.isfinite(y).all() and torch.equal(bad[rest(T)], y[rest(T)])
    assert torch.isnan(bad[BAD[0]]).all() and not torch.isfinite(bad[BAD[1]]).all()
    for checkpoint in (None, "fp8"):
        def dx(x, dy):
            x = x.detach().requires_grad_()
            return torch.autograd.grad(sf.gated_ffn(x, Wg, Wu, W2, checkpoint=checkpoint), x, dy)[0]

        want = dx(x, dy)
        assert torch.isfinite(want).all()
        for got in (dx(spoiled(x), dy), dx(x, spoiled(dy))):
            assert torch.equal(got[rest(T)], want[rest(T)]) and torch.isnan(got[BAD[0]]).any()
    sf.check_status()


@pytest.mark.parametrize("T", [6, 16, 20, 64, 140])
@pytest.mark.parametrize("K,N", [(64, 96), (101, 137), (1030, 600)])
def test_linear_and_8_bit_product(T, K, N):
    x, W, dy = randn(T, K), randn(N, K, seed=1, scale=K ** -0.5), randn(T, N, seed=2)
    w8 = sf.fp8_pack(W)
    for f in (lambda x: sf.ckpt_linear(x, W), lambda x: sf.fp8_matmul(x, w8), lambda x: sf.fp8_pack(x).to_dense()):
        y, bad = f(x), f(spoiled(x))
        assert torch.isfinite(y).all() and torch.equal(bad[rest(T)], y[rest(T)]) and torch.isnan(bad[BAD[0]]).any()
    x.requires_grad_()
    want, got = (torch.autograd.grad(sf.ckpt_linear(x, W), x, d)[0] for d in (dy, spoiled(dy)))
    assert torch.isfinite(want).all() and torch.equal(got[rest(T)], want[rest(T)]) and torch.isnan(got[BAD[0]]).all()
    sf.check_status()


@pytest.mark.parametrize("T", [20, 140])
def test_columns_of_weights(T):
    """Likewise for the weights' gradients: a spoiled feature of x or output gradient keeps to
    its own columns and rows of them, and a spoiled weight row to its own outputs."""
    K, N = 101, 137
    x, W, dy = randn(T, K), randn(N, K, seed=1, scale=K ** -0.5).requires_grad_(), randn(T, N, seed=2)
    want = torch.autograd.grad(sf.ckpt_linear(x, W), W, dy)[0]
    bad = dy.clone()
    bad[3, 7] = float("nan")
    got = torch.autograd.grad(sf.ckpt_linear(x, W), W, bad)[0]
    rows = [i for i in range(N) if i != 7]
    assert torch.equal(got[rows], want[rows]) and torch.isnan(got[7]).all()
    with torch.no_grad():
        V = W.clone()
        V[9, 3] = float("nan")
        y, z = sf.ckpt_linear(x, W), sf.ckpt_linear(x, V)
        cols = [i for i in range(N) if i != 9]
        assert torch.equal(z[:, cols], y[:, cols]) and torch.isnan(z[:, 9]).all()
    sf.check_status()
