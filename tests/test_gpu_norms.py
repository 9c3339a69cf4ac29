"""GPU checks of residual_norm against its definition in float64 (forward and
every gradient), at widths from one to 16384 elements, odd sizes, strides and
every pair of types, and of its gradient against central differences.

Tolerances.  u = 2^-24 is half a float32 step.  A sum over a row adds at most
32 terms in a thread, then a tree of 5 and up to 16 warps: r1 and r2 are within
40 u, a row mean within 60 u of the mean of magnitudes.  Each elementwise term
has under 20 roundings and carries those of r1, r2 and the means.  So before
the output's own rounding (finfo.eps / 2 of the value, or half its smallest
subnormal) an element is within

    C u M,   C = 256,

M the sum of the magnitudes of its terms (written beside each value below).  A
weight gradient adds N such products: within (C + N / 64 + 64) u of the sum of
their magnitudes (at most N / 64 rows in a register, then 32 partial sums, then
their tree) -- N / 64 bounds the rows of one block for the grids used here."""
import pytest
import torch

import autoresearch2_b200 as sf

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
C = 256
F64 = torch.float64
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
PAIRS = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, scale=1.0, base=0.0, dtype=F32):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale + base).to(dtype)


def close(got, want, mag, extra=0.0):
    assert got.shape == want.shape, (got.shape, want.shape)
    fi = torch.finfo(got.dtype)
    tol = want.abs() * (fi.eps / 2) * (1 + 2 ** -10) + fi.smallest_normal * fi.eps / 2 + (C + extra) * U * mag
    err = (got.detach().to(F64) - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.3g} of the tolerance"


def want_norm(x, y, pre, post, gate, post_norm, scale, eps, dxn=None, dh=None):
    """{name: (value, magnitude)} in float64; gate already [rows, D] or None."""
    d = lambda t: t.detach().to(F64) if t is not None else None  # noqa: E731
    x, y, pre, post, gate = map(d, (x, y, pre, post, gate))
    D = x.shape[-1]
    one = torch.ones(1, D, dtype=F64, device=DEV)
    pre_, post_, gate_ = (one if t is None else t for t in (pre, post, gate))
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    out = {}
    if y is None:
        z, mz = x, x.abs()
    else:
        r1 = (mean(y * y) + eps).rsqrt() if post_norm else torch.ones_like(y[..., :1])
        yh = y * r1
        u = yh * post_
        z, mz = scale * x + gate_ * u, (scale * x).abs() + (gate_ * u).abs()
        out["x_new"] = z, mz
    r2 = (mean(z * z) + eps).rsqrt()
    zh, mzh = z * r2, mz * r2
    out["h"] = zh * pre_, mzh * pre_.abs()
    if dh is None and dxn is None:
        return out
    dh = torch.zeros_like(x) if dh is None else d(dh)
    dxn = torch.zeros_like(x) if dxn is None else d(dxn)
    t = dh * pre_
    e = dxn + r2 * (t - zh * mean(t * zh))
    me = dxn.abs() + r2 * (t.abs() + mzh * mean(t.abs() * mzh))
    out["dx"] = (scale * e, abs(scale) * me) if y is not None else (e, me)
    rows = x.reshape(-1, D).shape[0]
    out["dpre"] = (dh * zh).reshape(rows, D), (dh.abs() * mzh).reshape(rows, D)
    if y is not None:
        out["dgate"] = (e * u).reshape(rows, D), (me * u.abs()).reshape(rows, D)
        du, mdu = gate_ * e, gate_.abs() * me
        out["dpost"] = (du * yh).reshape(rows, D), (mdu * yh.abs()).reshape(rows, D)
        v, mv = du * post_, mdu * post_.abs()
        if post_norm:
            out["dy"] = r1 * (v - yh * mean(v * yh)), r1 * (mv + yh.abs() * mean(mv * yh.abs()))
        else:
            out["dy"] = v, mv
    return out


def check(x, y, pre=None, post=None, gate=None, post_norm=False, scale=1.0, eps=1e-6, out_dtype=None, use=(True, True)):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, y, pre, post, gate)]
    x_new, h = sf.residual_norm(*leaves, post_norm=post_norm, residual_scale=scale, eps=eps, out_dtype=out_dtype)
    D = x.shape[-1]
    rows = x.numel() // D
    G = gate.numel() // D if gate is not None else 1
    g = gate.reshape(G, 1, D).expand(G, rows // G, D).reshape(x.shape) if gate is not None else None
    assert h.dtype == (out_dtype or (y if y is not None else x).dtype) and x_new.dtype == x.dtype
    dxn = randn(*x.shape, seed=21, dtype=x.dtype) if use[0] and y is not None else None
    dh = randn(*x.shape, seed=22, dtype=h.dtype) if use[1] else None
    want = want_norm(x, y, pre, post, g, post_norm, scale, eps, dxn, dh)
    close(h, *want["h"])
    if y is not None:
        close(x_new, *want["x_new"])
    else:
        assert x_new is leaves[0]
    outs = [(o, d) for o, d in ((x_new, dxn), (h, dh)) if d is not None]
    names = [(n, t) for n, t in zip(("dx", "dy", "dpre", "dpost", "dgate"), leaves) if t is not None]
    grads = torch.autograd.grad([o for o, _ in outs], [t for _, t in names], [d for _, d in outs])
    for (name, t), got in zip(names, grads):
        assert got.dtype == t.dtype and got.shape == t.shape, name
        value, mag = want[name]
        extra = 0.0
        if name in ("dpre", "dpost"):
            value, mag, extra = value.sum(0), mag.sum(0), rows / 64 + 64
        elif name == "dgate":
            value, mag = (v.view(G, rows // G, D).sum(1).view(t.shape) for v in (value, mag))
            extra = rows / 64 + 64
        close(got, value, mag, extra)
    a, b = sf.residual_norm(x, y, pre, post, gate, post_norm, scale, eps, out_dtype)  # without gradients
    assert torch.equal(b, h) and torch.equal(a, x_new)


def params(D, seed=0, dtype=F32):
    return [randn(D, seed=seed + i, scale=0.2, base=1.0, dtype=dtype) for i in range(3)]


@pytest.mark.parametrize("xt,yt", PAIRS)
@pytest.mark.parametrize("rows,D", [(1, 8), (2, 64), (7, 128), (3, 40), (3001, 64), (2999, 128), (1026, 120), (12345, 16)])
def test_narrow_rows(xt, yt, rows, D):
    """Several rows to a warp, the last of them behind the end."""
    x, y = randn(rows, D, seed=5, scale=2.0, dtype=xt), randn(rows, D, seed=6, dtype=yt)
    pre, post, gate = params(D)
    x[rows // 2] = 0
    check(x, y, pre, post, gate, post_norm=True, scale=0.5)
    check(x, None, pre, out_dtype=yt)
    if rows % 3 == 0:  # a gate row for each third
        check(x, y, pre, post, randn(3, D, seed=8), post_norm=True)


@pytest.mark.parametrize("xt,yt", PAIRS)
@pytest.mark.parametrize("rows,D", [(1, 1), (2, 7), (3, 8), (5, 31), (1, 64), (40, 100), (3000, 256), (7, 257), (33, 768),
                                    (2, 1001), (700, 1024), (5, 2056), (9, 4096), (3, 4097), (2, 5000), (310, 8192),
                                    (2, 8200), (3, 12345), (400, 16384), (1, 16383)])
def test_everything_on(xt, yt, rows, D):
    pre, post, gate = params(D)
    check(randn(rows, D, seed=1, scale=2.0, dtype=xt), randn(rows, D, seed=2, dtype=yt), pre, post, gate, True, 0.7)


@pytest.mark.parametrize("xt,yt", PAIRS)
@pytest.mark.parametrize("D", [48, 333, 4608])
def test_parts_left_out(xt, yt, D):
    """No weights, no gate, no norm after the block, no block at all; one of the two upstreams alone."""
    x, y = randn(37, D, seed=1, dtype=xt), randn(37, D, seed=2, dtype=yt)
    pre, post, gate = params(D)
    check(x, y)
    check(x, y, post_norm=True)
    check(x, y, pre, None, None, False, 0.5)
    check(x, y, None, post, None, True)
    check(x, y, None, None, gate, False)
    check(x, y, pre, post, gate, True, use=(True, False))
    check(x, y, pre, post, gate, True, use=(False, True))
    check(x, None, pre)
    check(x, None, None, out_dtype=yt)


@pytest.mark.parametrize("wt", [F32, BF16, F16])
@pytest.mark.parametrize("D", [320, 1003, 6144])
def test_weights_of_any_type(wt, D):
    pre, post, gate = params(D, dtype=wt)
    check(randn(65, D, seed=1, dtype=BF16), randn(65, D, seed=2, dtype=BF16), pre, post, gate, True)


@pytest.mark.parametrize("D", [64, 999, 4160, 8193])
@pytest.mark.parametrize("rows,G", [(6, 2), (6, 6), (4000, 5), (4000, 1000), (1300, 1), (4001, 4001)])
def test_gates_for_runs_of_rows(D, rows, G):
    pre, post, _ = params(D)
    check(randn(rows, D, seed=1), randn(rows, D, seed=2, dtype=BF16), pre, post,
          randn(G, D, seed=3, dtype=BF16), True, 0.9)


def test_gates_shaped_as_the_stream():
    x, y = randn(3, 4, 5, 96, seed=1), randn(3, 4, 5, 96, seed=2)
    for shape in ((3, 1, 1, 96), (3, 4, 1, 96), (3, 4, 5, 96), (1, 1, 1, 96), (96,), (12, 96)):
        check(x, y, gate=randn(*shape, seed=4), post_norm=True)


@pytest.mark.parametrize("D", [96, 97])
def test_strided_rows(D):
    """Rows of a wider tensor, shifted off 16 bytes, expanded, transposed, three dimensions."""
    big = randn(20, 4, 2 * D + 9, seed=1, scale=2.0, dtype=BF16)
    y = randn(20, 4, D, seed=2, dtype=BF16)
    pre, post, gate = params(D)
    for x in (big[..., :D], big[..., 1:D + 1], big[..., 8:D + 8], big[:, :1, :D].expand(20, 4, D),
              big[..., :D].transpose(0, 1).contiguous().transpose(0, 1), big[..., ::2][..., :D]):
        check(x, y, pre, post, gate, True)
        check(y, x, pre, post, gate, True)
    check(big[:, 0, :D], y[:1, 0].expand(20, D), pre, post, gate, True)
    pre1 = torch.cat([pre, pre])[1:D + 1]  # a weight off its 16-byte boundary
    check(y, y, pre1, post, gate, True)


def test_zero_rows_of_the_stream_and_zero_values():
    D = 128
    pre, post, gate = params(D)
    x = torch.empty(0, D, device=DEV, requires_grad=True)
    w = pre.clone().requires_grad_()
    a, h = sf.residual_norm(x, torch.empty(0, D, device=DEV), w, post, gate, True)
    (a.sum() + h.sum()).backward()
    assert a.shape == h.shape == (0, D) and x.grad.shape == (0, D) and not w.grad.any()
    x, y = randn(4, D, seed=1), randn(4, D, seed=2)
    x[0] = 0
    y[0] = 0
    y[1] = 0
    check(x, y, pre, post, gate, True, eps=1e-5)
    check(x * 0, None, pre, eps=1e-5)


def test_gradient_against_differences():
    """Central differences of the kernel's forward at step h = 2^-5: its error is
    h^2 / 6 of a third derivative (below 60 for these unit-sized rows and upstreams)
    plus the forward's rounding, C u times the sum of upstream magnitudes, over h."""
    D, R = 6, 2
    base = [randn(R, D, seed=1), randn(R, D, seed=2), *params(D)]
    w = [randn(R, D, seed=5).double(), randn(R, D, seed=6).double()]

    def f(ts):
        a, h = sf.residual_norm(*ts, post_norm=True, residual_scale=0.8)
        return (a.double() * w[0]).sum() + (h.double() * w[1]).sum()

    leaves = [t.clone().requires_grad_() for t in base]
    grads = torch.autograd.grad(f(leaves), leaves)
    eps = 2 ** -5
    for n, (t, g) in enumerate(zip(base, grads)):
        for i in range(t.numel()):
            hi, lo = ([b.clone() for b in base] for _ in range(2))
            hi[n].view(-1)[i] += eps
            lo[n].view(-1)[i] -= eps
            d = (f(hi) - f(lo)) / (hi[n].view(-1)[i].double() - lo[n].view(-1)[i].double())
            assert abs(float(d - g.view(-1)[i])) <= 60 * eps ** 2 / 6 + C * U * 100 / eps


def test_equal_inputs_give_equal_bits_captured_and_on_other_streams():
    D, R = 768, 2500
    x, y = randn(R, D, seed=1, dtype=BF16), randn(R, D, seed=2, dtype=BF16)
    leaves = [t.requires_grad_() for t in (x, y, *params(D))]
    d = [randn(R, D, seed=4, dtype=BF16), randn(R, D, seed=5, dtype=BF16)]

    def step():
        out = sf.residual_norm(*leaves, post_norm=True)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, d))

    want = step()
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    for g in got + [out]:
        assert all(torch.equal(p, q) for p, q in zip(g, want))
    with torch.no_grad():
        for t in leaves[:2]:
            t.mul_(-0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_offsets_beyond_32_bits():
    """140000 x 16384 elements, 2.29e9: the last rows equal a small call's."""
    R, D = 140000, 16384
    x = torch.zeros(R, D, device=DEV, dtype=BF16)
    x[-2:] = randn(2, D, seed=1, dtype=BF16)
    pre, _, gate = params(D)
    x.requires_grad_()
    a, h = sf.residual_norm(x, x.detach(), pre, None, gate, True)
    small = x.detach()[-2:].clone().requires_grad_()
    a2, h2 = sf.residual_norm(small, small.detach(), pre, None, gate, True)
    assert torch.equal(a[-2:], a2) and torch.equal(h[-2:], h2)
    g, = torch.autograd.grad(h, x, torch.ones(1, 1, device=DEV, dtype=BF16).expand(R, D).contiguous())
    g2, = torch.autograd.grad(h2, small, torch.ones_like(h2))
    assert torch.equal(g[-2:], g2)


def test_library_op():
    D = 200
    x, y = randn(30, D, seed=1, dtype=BF16), randn(30, D, seed=2, dtype=BF16)
    pre, post, gate = params(D)
    torch.library.opcheck(torch.ops.sparseffn.residual_norm.default,
                          (x, y, pre, post, gate, 1, True, 0.5, 1e-6, BF16), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.sparseffn.residual_norm.default,
                          (x, None, None, None, None, 1, False, 1.0, 1e-6, BF16),
                          test_utils=("test_schema", "test_faketensor"))

    def f(x, y, pre, post, gate):
        a, h = sf.residual_norm(x, y, pre, post, gate, True, 0.5)
        return (a.float() * 2 + h.float().square()).sum()

    torch._dynamo.reset()
    one = [t.clone().requires_grad_() for t in (x, y, pre, post, gate)]
    two = [t.clone().requires_grad_() for t in (x, y, pre, post, gate)]
    f(*one).backward()
    torch.compile(f, backend="aot_eager", fullgraph=True)(*two).backward()
    torch._dynamo.reset()
    assert all(torch.equal(p.grad, q.grad) for p, q in zip(one, two))


def test_gradients_are_not_differentiable_again():
    x = randn(3, 16, seed=1).requires_grad_()
    _, h = sf.residual_norm(x, x)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        torch.autograd.grad(h.sum(), x, create_graph=True)


def test_ops_refuse_what_the_function_refuses():
    op, bwd = torch.ops.sparseffn.residual_norm, torch.ops.sparseffn.residual_norm_bwd
    D = 64
    x, y, gate = randn(6, D, seed=1), randn(6, D, seed=2), randn(2, D, seed=3)
    _, _, stats = op(x, y, None, None, gate, 2, False, 1.0, 1e-6, F32)
    rest = (False, 1.0, F32)
    bad = [lambda: op(x, y, None, None, gate, 4, False, 1.0, 1e-6, F32), lambda: op(x, y, None, None, gate, 3, False, 1.0, 1e-6, F32),
           lambda: op(x, y[:5], None, None, None, 1, False, 1.0, 1e-6, F32), lambda: op(x, y, gate[0, :9], None, None, 1, False, 1.0, 1e-6, F32),
           lambda: op(x, y, None, None, None, 0, False, 1.0, 1e-6, F32),
           lambda: bwd(x, y, None, None, gate, 3, *rest, stats, x, y, [True] * 5),
           lambda: bwd(x, y, None, None, gate, 2, *rest, stats[:4], x, y, [True] * 5),
           lambda: bwd(x, y, None, None, gate, 2, *rest, stats, x[:5], y, [True] * 5),
           lambda: bwd(x, y, None, None, gate, 2, *rest, stats, x, y.half(), [True] * 5)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
