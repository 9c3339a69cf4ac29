"""GPU checks of gated_ffn against its definition in float64: the forward, what
it keeps, and every gradient from what was kept.

Tolerances.  u = finfo.eps / 2 is half a step of the type.  A product's sum of K
terms errs by at most s(K) S, s(K) = (K / 16 + 64) 2^-23, S the sum of its terms'
magnitudes (tensor cores add at least 16 products a step in float32 and lose at
most 2^-23 of S a step; the rest is for joins of parts).  act and act' are
computed within 2^-18 of max(|g|, 1)^2 (at most two dozen float32 roundings of
values of that size, exp's argument among them, whose rounding grows with |g|).
So with Eg = s(D) Sg and Eu = s(D) Su

    |h - ref| <= E_h = |u| (L Eg + 2^-18 max(|g|, 1)^2) + |act| Eu,   L = max |act'| nearby
    y: u |y| + |W2| (u |h| + E_h) + s(F) S

and, given g and u as kept (checked apart: half a step, and Eg, Eu),

    dh: E_dh = s(D) S;  dg: u |dg| + |u act'| E_dh + 2^-18 |dh u| max(|g|, 1)^2
    du, h alike; the gradients' products carry these, times the other
    factor's magnitudes, and their own s(K) S and rounding."""
import pytest
import torch

import autoresearch2_b200 as sf
from autoresearch2_b200 import glu
from test_gpu_fp8 import want_blocks

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16
ACTS = ["silu", "gelu", "relu", "relu2"]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def act(g, name):
    """(act, act') in float64."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if name == "gelu":
        c = 0.5 * torch.erfc(-g / 2 ** 0.5)
        return g * c, c + g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    r = g.clamp_min(0)
    return (r, (g > 0).to(F64)) if name == "relu" else (r * r, 2 * r)


def s(K):
    return (K / 16 + 64) * 2 ** -23


def half(t):
    return torch.finfo(t).eps / 2 * (1 + 2 ** -8)


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps


def check(name, got, want, tol):
    assert got.shape == want.shape, name
    err = (got.detach().to(F64) - want).abs()
    tol = tol + half(got.dtype) * want.abs() + tiny(got.dtype)
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.3g} of the tolerance"


def unpacked(values, tiles, dtype):
    return sf.fp8_unpack(sf.Fp8Tensor(values, tiles), dtype)


def inputs(T, D, F, dtype, seed=0):
    x, dy = randn(T, D, seed=seed, dtype=dtype), randn(T, D, seed=seed + 1, dtype=dtype)
    Wg, Wu = (randn(F, D, seed=seed + 2 + i, scale=D ** -0.5, dtype=dtype) for i in range(2))
    return x, Wg, Wu, randn(D, F, seed=seed + 4, scale=F ** -0.5, dtype=dtype), dy


def forward_reference(x, Wg, Wu, W2, name):
    """y and its tolerance; g, u with theirs."""
    x, Wg, Wu, W2 = (t.detach().to(F64) for t in (x, Wg, Wu, W2))
    D, F = x.shape[1], Wg.shape[0]
    g, u = x @ Wg.T, x @ Wu.T
    Eg, Eu = s(D) * (x.abs() @ Wg.abs().T), s(D) * (x.abs() @ Wu.abs().T)
    a, _ = act(g, name)
    L = 2 * (g.abs() + Eg) if name == "relu2" else torch.full_like(g, 1.13)
    h = a * u
    Eh = u.abs() * (L * Eg + 2 ** -18 * g.abs().clamp_min(1).square()) + a.abs() * Eu
    return h @ W2.T, h, Eh, W2, g, Eg, u, Eu, F


def check_forward(y, x, Wg, Wu, W2, name):
    want, h, Eh, W2, *_, F = forward_reference(x, Wg, Wu, W2, name)
    dt = y.dtype
    check("y", y, want, (half(dt) * h.abs() + Eh + tiny(dt)) @ W2.abs().T + s(F) * (h.abs() @ W2.abs().T))


def check_backward(grads, dy, x, Wg, Wu, W2, g, u, name):
    """grads (dx, dWg, dWu, dW2) from x, g, u as kept."""
    dt = dy.dtype
    dy, x, Wg, Wu, W2, g, u = (t.detach().to(F64) for t in (dy, x, Wg, Wu, W2, g, u))
    T, D, F = x.shape[0], x.shape[1], g.shape[1]
    a, d = act(g, name)
    dh = dy @ W2
    Edh = s(D) * (dy.abs() @ W2.abs())
    f = 2 ** -18 * g.abs().clamp_min(1).square()
    dg, du, h = dh * u * d, dh * a, a * u
    Edg = half(dt) * dg.abs() + (u * d).abs() * Edh + f * (dh * u).abs() + tiny(dt)
    Edu = half(dt) * du.abs() + a.abs() * Edh + f * dh.abs() + tiny(dt)
    Eh = half(dt) * h.abs() + f * u.abs() + tiny(dt)
    A = lambda t: t.abs()  # noqa: E731
    dx, dWg, dWu, dW2 = grads
    check("dW2", dW2, dy.T @ h, A(dy).T @ Eh + s(T) * (A(dy).T @ A(h)))
    check("dWg", dWg, dg.T @ x, Edg.T @ A(x) + s(T) * (A(dg).T @ A(x)))
    check("dWu", dWu, du.T @ x, Edu.T @ A(x) + s(T) * (A(du).T @ A(x)))
    check("dx", dx, dg @ Wg + du @ Wu, Edg @ A(Wg) + Edu @ A(Wu) + s(2 * F) * (A(dg) @ A(Wg) + A(du) @ A(Wu)))


SIZES = [(1, 64, 64), (3, 8, 40), (5, 129, 65), (16, 768, 256), (32, 96, 1001), (33, 64, 96), (64, 130, 300), (128, 128, 128),
         (129, 264, 129), (300, 768, 515), (513, 96, 1024), (40, 1, 1), (1000, 200, 333)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,D,F", SIZES)
def test_forward(T, D, F, dtype):
    x, Wg, Wu, W2, _ = inputs(T, D, F, dtype)
    for name in ACTS if T in (5, 33, 64, 129) else ("silu",):
        y = sf.gated_ffn(x, Wg, Wu, W2, name)
        check_forward(y, x, Wg, Wu, W2, name)
        assert torch.equal(y, sf.gated_ffn(x, Wg, Wu, W2, name))
    sf.check_status()


@pytest.mark.parametrize("T,D,F", [(1, 3000, 5003), (8, 600, 2500), (16, 2600, 4096), (27, 2500, 7001), (32, 515, 9000),
                                   (20, 256, 20480), (48, 2048, 8192), (24, 8192, 1000), (47, 5120, 640), (49, 640, 1024), (64, 2048, 8192), (61, 8192, 1000),
                                   (63, 264, 20480), (65, 640, 1024)])
def test_forward_of_few_rows_and_long_weights(T, D, F):
    """Several groups of weight rows a multiprocessor, in both projections; many
    calls under way at once."""
    x, Wg, Wu, W2, _ = inputs(T, D, F, BF16)
    ys = [sf.gated_ffn(x, Wg, Wu, W2) for _ in range(20)]
    check_forward(ys[0], x, Wg, Wu, W2, "silu")
    assert all(torch.equal(ys[0], y) for y in ys[1:])
    sf.check_status()


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,D,F", SIZES)
def test_training(T, D, F, dtype, checkpoint):
    x, Wg, Wu, W2, dy = inputs(T, D, F, dtype, seed=20)
    leaves = [t.requires_grad_() for t in (x, Wg, Wu, W2)]
    for name in ACTS if T in (33, 129) else ("silu",):
        y = sf.gated_ffn(x, Wg, Wu, W2, name, checkpoint=checkpoint)
        grads = torch.autograd.grad(y, leaves, dy)
        check_forward(y.detach(), x, Wg, Wu, W2, name)
        with torch.no_grad():
            _, g, u, gt, ut, xv, xt = glu._forward(x, Wg, Wu, W2, glu.ACTIVATIONS[name], glu.KEEP[checkpoint])
        _, _, _, _, wg, Eg, wu, Eu, _ = forward_reference(x, Wg, Wu, W2, name)
        if checkpoint is None:
            check("g", g, wg, Eg)
            check("u", u, wu, Eu)
            kept = x.detach()
        else:
            kept = unpacked(xv, xt, F32)
            assert torch.equal(kept.to(F64), want_blocks(x.detach())[0])
            kept = unpacked(xv, xt, dtype)
            for v, t, w, E in ((g, gt, wg, Eg), (u, ut, wu, Eu)):
                got = unpacked(v, t, F32).to(F64)
                # half a step of e4m3 of the value, or half the smallest of the block's scale (448 -> 2^-9:
                # 2^-10 / 224 of the block's largest at most)
                top = torch.nn.functional.pad(w.abs() + E, (0, -F % 128)).view(T, -1, 128).amax(-1)
                floor = (top * 2 ** -10 / 224).repeat_interleave(128, 1)[:, :F]
                assert ((got - w).abs() <= torch.maximum(w.abs() * 2 ** -4, floor) * (1 + 2 ** -8) + 2 * E).all()
            g, u = unpacked(g, gt, F32), unpacked(u, ut, F32)
        check_backward(grads, dy, kept, Wg, Wu, W2, g, u, name)
        again = torch.autograd.grad(sf.gated_ffn(x, Wg, Wu, W2, name, checkpoint=checkpoint), leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))
    sf.check_status()


@pytest.mark.parametrize("name", ACTS)
def test_gradient_against_differences(name):
    """Directional derivatives of sum(y * dy), by central differences of the
    float64 definition, against the kernels' gradients along random directions."""
    T, D, F = 70, 96, 200
    x, Wg, Wu, W2, dy = inputs(T, D, F, BF16, seed=40)
    leaves = [t.requires_grad_() for t in (x, Wg, Wu, W2)]
    grads = torch.autograd.grad(sf.gated_ffn(x, Wg, Wu, W2, name), leaves, dy)
    at = [t.detach().to(F64) for t in leaves]

    def f(x, Wg, Wu, W2):
        return ((act(x @ Wg.T, name)[0] * (x @ Wu.T)) @ W2.T * dy.to(F64)).sum()

    for i, gr in enumerate(grads):
        v = randn(*gr.shape, seed=50 + i).to(F64)
        eps = 1e-5
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + eps * v, at[i] - eps * v
        diff = (f(*up) - f(*down)) / (2 * eps)
        # Each gradient element is a sum whose factors were rounded at most four
        # times, 2^-9 each; against the root of the sum of squares those add up as
        # independent errors, eight standard deviations of them here, and relu's
        # kink moves by g's rounding.
        tol = 8 * 4 * 2 ** -9 * (gr.to(F64) * v).norm() * 2
        assert (diff - (gr.to(F64) * v).sum()).abs() <= tol, (name, i)


def test_partial_gradients_leading_dimensions_and_none_kept():
    x, Wg, Wu, W2, dy = inputs(90, 64, 80, BF16)
    x, dy = x.view(3, 30, 64), dy.view(3, 30, 64)
    leaves = [x, Wg, Wu, W2]
    for checkpoint in (None, "fp8"):
        want = torch.autograd.grad(sf.gated_ffn(*(t.requires_grad_() for t in leaves), checkpoint=checkpoint), leaves, dy)
        assert want[0].shape == x.shape
        for i in range(4):
            only = [t if j == i else t.detach() for j, t in enumerate(leaves)]
            got = torch.autograd.grad(sf.gated_ffn(*only, checkpoint=checkpoint), only[i], dy)[0]
            assert torch.equal(got, want[i])
    with torch.no_grad():
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        y = sf.gated_ffn(x, Wg, Wu, W2)
        assert torch.cuda.memory_allocated() - base <= 2 * y.numel() + 1024


def test_no_rows():
    x, Wg, Wu, W2, dy = inputs(0, 64, 80, BF16)
    leaves = [t.requires_grad_() for t in (x, Wg, Wu, W2)]
    for checkpoint in (None, "fp8"):
        y = sf.gated_ffn(x, Wg, Wu, W2, checkpoint=checkpoint)
        grads = torch.autograd.grad(y, leaves, dy)
        assert y.shape == (0, 64) and not any(g.any() for g in grads)


@pytest.mark.parametrize("T", [1, 9])
def test_few_unaligned_rows_with_aligned_weights(T):
    big, (_, Wg, Wu, W2, _) = randn(T, 100, seed=1, dtype=BF16), inputs(1, 96, 200, BF16)
    x = big[:, 3:99]
    assert torch.equal(sf.gated_ffn(x, Wg, Wu, W2), sf.gated_ffn(x.contiguous(), Wg, Wu, W2))
    assert torch.equal(sf.ckpt_linear(x, Wg), sf.ckpt_linear(x.contiguous(), Wg))
    W = randn(200, 99, seed=2, dtype=BF16)[:, 3:]
    assert torch.equal(sf.ckpt_linear(x, W), sf.ckpt_linear(x.contiguous(), W.contiguous()))


@pytest.mark.parametrize("T", [4, 150])
def test_strided_operands(T):
    big = randn(2 * T, 200, seed=1, dtype=BF16)
    W = randn(300, 300, seed=2, scale=0.1, dtype=BF16)
    x, Wg, Wu, W2 = big[::2, 3:99], W[:130, 1:97], W[:96, :130].T, W[:96, 9:139]
    got = sf.gated_ffn(x, Wg, Wu, W2)
    assert torch.equal(got, sf.gated_ffn(*(t.contiguous() for t in (x, Wg, Wu, W2))))
    leaves = [t.detach().requires_grad_() for t in (x, Wg, Wu, W2)]
    cont = [t.detach().contiguous().requires_grad_() for t in (x, Wg, Wu, W2)]
    dy = randn(96, T, seed=3, dtype=BF16).T
    for a, b in zip(torch.autograd.grad(sf.gated_ffn(*leaves, checkpoint="fp8"), leaves, dy),
                    torch.autograd.grad(sf.gated_ffn(*cont, checkpoint="fp8"), cont, dy.contiguous())):
        assert torch.equal(a, b)


def test_infinities_and_nan_stay_in_their_rows():
    for T in (6, 20, 140):
        x, Wg, Wu, W2, dy = inputs(T, 64, 96, BF16)
        x[2, 5] = float("nan")
        x[4, 1] = float("inf")
        y = sf.gated_ffn(x, Wg, Wu, W2)
        assert torch.isnan(y[2]).all() and torch.isnan(y[4]).any()
        rest = [i for i in range(T) if i not in (2, 4)]
        assert torch.equal(y[rest], sf.gated_ffn(x[rest], Wg, Wu, W2)) or torch.isfinite(y[rest]).all()
    leaves = [t.requires_grad_() for t in (x, Wg, Wu, W2)]
    for checkpoint in (None, "fp8"):
        dx = torch.autograd.grad(sf.gated_ffn(x, Wg, Wu, W2, checkpoint=checkpoint), x, dy)[0]
        assert torch.isnan(dx[2]).any() and torch.isfinite(dx[rest]).all()


@pytest.mark.parametrize("T", [12, 40, 1537])
def test_gelu_keeps_small_tails(T):
    """x gelu(x) alone, one weight of 1 each: Phi is within 2^-16 of itself for |x| <= 12
    (2.7e-6 for |x| < 5, its exponent's rounding beyond), the products' float32 roundings
    below 2^-21, h is rounded once and y is h."""
    x = torch.linspace(-12, 12, T, device=DEV).to(BF16)[:, None]
    one = torch.ones(1, 1, device=DEV, dtype=BF16)
    y = sf.gated_ffn(x, one, one, one, "gelu").to(F64)
    x = x.to(F64)
    want = x * x * 0.5 * torch.erfc(-x / 2 ** 0.5)
    assert ((y - want).abs() <= (half(BF16) + 2 ** -15) * want.abs()).all()
