"""GPU checks of the 8-bit block format, its product and the linear layer that
keeps its input in it, against their definitions in float64.

Tolerances.  The format has none: values and exponents are equal, bit for bit.
A product's result is rounded once (half a step, finfo.eps / 2 of it, or half its
smallest subnormal).  Its sum of K terms is added on tensor cores in float32:
each step adds at least 16 products and loses at most 2^-23 of the sum of
magnitudes S (truncation of the sum, and of the products as they are aligned),
and so do the up to 64 additions that join warps, parts and blocks:

    |err| <= eps / 2 |C| + (K / 16 + 64) 2^-23 S."""
import pytest
import torch

import autoresearch2_b200 as sf
from autoresearch2_b200 import fp8

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def want_blocks(x):
    """(dequantised float64, exponents) of the format's definition, in float64;
    a NaN stands for infinities and NaN."""
    x = x.reshape(-1, x.shape[-1]).to(F64)
    rows, width = x.shape
    nb = -(-width // 128)
    p = torch.nn.functional.pad(x, (0, nb * 128 - width)).view(rows, nb, 128)
    fin = torch.where(torch.isfinite(p), p.abs(), torch.zeros_like(p)).amax(-1)
    # smallest e with amax <= 448 * 2^e, by trying every one
    e = torch.full((rows, nb), -118, device=x.device, dtype=torch.int32)
    for k in range(-118, 121):
        e = torch.where(fin > 448.0 * 2.0 ** k, torch.full_like(e, k + 1), e)
    e = torch.where(fin == 0, torch.zeros_like(e), e)
    s = torch.exp2(e.to(F64))[..., None]
    y = torch.where(torch.isfinite(p), p, torch.full_like(p, float("nan"))) / s
    top = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30)))
    top = top - (y.abs() < torch.exp2(top)).to(F64)  # log2 may have rounded up across a power
    step = torch.exp2(top.clamp_min(-6) - 3)
    return (torch.round(y / step) * step * s).view(rows, nb * 128)[:, :width], e


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, nan=0.0), torch.nan_to_num(b, nan=0.0))


def close_sum(got, a, b):
    """got against a [M, K] b [N, K]^T in float64, by the bound above."""
    want, mag = a @ b.T, a.abs() @ b.abs().T
    fi = torch.finfo(got.dtype)
    tol = want.abs() * (fi.eps / 2) * (1 + 2 ** -9) + fi.smallest_normal * fi.eps / 2 + (a.shape[1] / 16 + 64) * 2 ** -23 * mag
    err = (got.to(F64) - want).abs()
    assert got.shape == want.shape
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.3g} of the tolerance"


# ---------------------------------------------------------------------------
# Pack, unpack
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 16), (5, 127), (2, 3, 128), (33, 129), (129, 640), (257, 1001), (300, 2048)])
def test_pack_is_the_definition(shape, dtype):
    x = randn(*shape, seed=sum(shape), dtype=dtype)
    x = x * torch.exp2(torch.randint(-12, 12, (*shape[:-1], 1), generator=gen(1), device=DEV).float()).to(dtype)
    q = sf.fp8_pack(x)
    want, e = want_blocks(x)
    assert q.shape == x.shape and torch.equal(q.exponents, e)
    assert same(sf.fp8_unpack(q, F32).view(-1, shape[-1]).to(F64), want)
    for out in (F32, BF16):  # exact
        assert same(q.to_dense(out).to(F64), want.view(shape))
    assert torch.equal(q.to_dense(F16), want.view(shape).to(F16))


def test_pack_of_odd_blocks():
    """Zeros, subnormals, powers of two and their neighbours at the scale's
    border, infinities and NaN, the largest values of each type."""
    x = torch.zeros(16, 256, device=DEV)
    x[1] = -0.0
    x[2, :4] = torch.tensor([448.0, 1e-9, -448.0, 2.0 ** -9], device=DEV)
    x[3, 5] = torch.nextafter(torch.tensor(448.0), torch.tensor(INF)).item()
    x[4] = 1e-44
    x[5] = randn(256, seed=2) * 1e-40
    x[6, :3] = torch.tensor([INF, -INF, float("nan")], device=DEV)
    x[6, 3:8] = 1.0
    x[7, :128] = INF
    x[8] = torch.finfo(F32).max
    x[9] = -torch.finfo(F32).max
    x[10, 0] = 2.0 ** -130
    x[11] = torch.arange(256, device=DEV) * 2.0 ** -12  # ties of the subnormal steps
    x[12] = 1 + torch.arange(256, device=DEV) / 128.0
    x[13, 0] = 3.4e38
    x[13, 1] = 1e-38
    x[14, 200] = 1e-30
    q = sf.fp8_pack(x)
    want, e = want_blocks(x)
    assert torch.equal(q.exponents, e)
    got = q.to_dense(F32).to(F64)
    top = torch.finfo(F32).max
    assert same(got, want.clamp(-top, top))
    assert int(q.exponents.min()) == -118 and int(q.exponents.max()) == 120
    for dtype in (BF16, F16):
        top = torch.finfo(dtype).max
        y = torch.full((2, 128), top, device=DEV, dtype=dtype)
        y[1] = -top
        got = sf.fp8_pack(y).to_dense(dtype)
        want = want_blocks(y)[0]
        assert torch.equal(got.to(F64), want.clamp(-top, top).to(dtype).to(F64)) and torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pack_takes_any_strides(dtype):
    base = randn(40, 700, seed=3, dtype=dtype)
    for x in (base[:, 3:390], base[::2, :384], base.T, base[:, ::2], base[:1].expand(7, 700), base.view(4, 10, 700)[:, 1:9],
              base[:, 5:6], base[5]):
        q = sf.fp8_pack(x)
        want, e = want_blocks(x.contiguous())
        assert q.shape == x.shape and torch.equal(q.exponents, e)
        assert torch.equal(q.to_dense(F32).to(F64).view(want.shape), want)


def test_pack_of_no_rows():
    q = sf.fp8_pack(torch.empty(0, 64, device=DEV))
    assert q.shape == (0, 64) and sf.fp8_unpack(q).shape == (0, 64)
    w = sf.fp8_pack(randn(40, 64))
    assert sf.fp8_matmul(q, w).shape == (0, 40)
    assert sf.fp8_matmul(sf.fp8_pack(randn(3, 64)), sf.fp8_pack(randn(0, 64))).shape == (3, 0)


# ---------------------------------------------------------------------------
# The product
# ---------------------------------------------------------------------------
SIZES = [(1, 64, 64), (1, 1000, 4096), (8, 48, 16), (9, 130, 1001), (16, 256, 640), (17, 33, 129), (32, 300, 2048),
         (33, 64, 64), (64, 100, 130), (128, 128, 128), (129, 257, 513), (200, 1000, 1333), (256, 256, 512), (300, 515, 4096),
         (777, 1001, 96), (1, 1, 1), (40, 1, 7), (513, 768, 16384), (1, 5003, 3000), (16, 4800, 1100),
         (10, 9001, 700),  # these three: several groups of rows a multiprocessor
         (40, 300, 14336), (300, 257, 9000), (17, 1001, 2049),  # in parts of K
         (20, 20000, 300), (24, 2048, 8192), (37, 4096, 5120), (48, 640, 8200), (49, 640, 8200), (64, 2048, 8192), (57, 20000, 300), (65, 640, 8200), (9, 8200, 4100)]  # up to 64 rows


@pytest.mark.parametrize("out", [BF16, F16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K, out):
    a = randn(M, K, seed=M, dtype=BF16) * torch.exp2(torch.randint(-3, 4, (M, 1), generator=gen(5), device=DEV)).to(BF16)
    b = randn(N, K, seed=N + 1, scale=K ** -0.5)
    b[:, ::7] *= 16  # scales that differ from block to block
    qa, qb = sf.fp8_pack(a), sf.fp8_pack(b)
    got = sf.fp8_matmul(qa, qb, out_dtype=out)
    assert got.dtype == out
    close_sum(got, qa.to_dense(F32).to(F64), qb.to_dense(F32).to(F64))
    assert torch.equal(got, sf.fp8_matmul(qa, qb, out_dtype=out))
    assert torch.equal(got, sf.fp8_matmul(a, qb, out_dtype=out))  # packed within the call
    sf.check_status()


@pytest.mark.parametrize("M", [4, 20, 300])
def test_product_picks_each_blocks_scale(M):
    """One element a block: every (row, block) scale of both operands is told apart."""
    K, N = 1280, 270
    a, b = torch.zeros(M, K, device=DEV), torch.zeros(N, K, device=DEV)
    for k in range(K // 128):
        a[:, 128 * k + 5] = torch.exp2(torch.randint(-8, 9, (M,), generator=gen(k), device=DEV).float()) * 1.5
        b[:, 128 * k + 5] = torch.exp2(torch.randint(-8, 9, (N,), generator=gen(90 + k), device=DEV).float())
    got = sf.fp8_matmul(sf.fp8_pack(a), sf.fp8_pack(b))
    close_sum(got, a.to(F64), b.to(F64))


@pytest.mark.parametrize("M", [2, 20, 140])
def test_product_of_far_scales(M):
    """Exponents whose sum leaves the scales' own range, NaN rows."""
    a, b = randn(M, 256, seed=8), randn(130, 256, seed=9)
    a *= 2.0 ** -100
    b *= 2.0 ** 110
    a[1, 3] = float("nan")
    b[7, 200] = INF
    qa, qb = sf.fp8_pack(a), sf.fp8_pack(b)
    got = sf.fp8_matmul(qa, qb)
    da, db = qa.to_dense(F32).to(F64), qb.to_dense(F32).to(F64)
    assert torch.isnan(got[1]).all() and torch.isnan(got[:, 7]).all()
    keep_m, keep_n = [i for i in range(M) if i != 1], [i for i in range(130) if i != 7]
    close_sum(got[keep_m][:, keep_n], da[keep_m], db[keep_n])


def test_product_shapes_and_types():
    w = sf.fp8_pack(randn(48, 64, seed=1))
    x = randn(2, 5, 64, seed=2, dtype=F16)
    y = sf.fp8_matmul(x, w)
    assert y.shape == (2, 5, 48) and y.dtype == F16
    assert sf.fp8_matmul(sf.fp8_pack(x), w).dtype == BF16
    assert sf.fp8_matmul(x.float(), w).dtype == BF16
    assert sf.fp8_matmul(x[0, 0], w).shape == (48,)
    assert torch.equal(sf.fp8_matmul(x[0, 0], w), y[0, 0])


@pytest.mark.parametrize("M", [2, 40])
def test_misaligned_blocks_are_refused(M):
    b = sf.fp8_pack(randn(64, 64))
    q = sf.fp8_pack(randn(M, 64))
    t = torch.zeros(q.scale_tiles.numel() + 2, dtype=torch.uint8, device=DEV)[2:].view(q.scale_tiles.shape)
    v = torch.zeros(M * 80 + 1, dtype=torch.uint8, device=DEV)[1:].view(fp8.E4M3).view(M, 80)[:, :64]
    with pytest.raises(sf._lib.SparseFFNError, match="misaligned"):
        sf.fp8_matmul(sf.Fp8Tensor(q.values, t), b)
    with pytest.raises(ValueError, match="start on 16 bytes"):
        sf.fp8_matmul(sf.Fp8Tensor(v, q.scale_tiles), b)
    with pytest.raises(sf._lib.SparseFFNError, match="misaligned"):
        sf.fp8_unpack(sf.Fp8Tensor(v, q.scale_tiles))


def test_product_beside_others_rows():
    """Nothing is written past the result, with rows that are not 16 bytes apart."""
    from autoresearch2_b200 import _lib
    for M in (5, 20, 70):
        N, K = 77, 200
        qa, qb = sf.fp8_pack(randn(M, K, seed=4)), sf.fp8_pack(randn(N, K, seed=5))
        big = torch.full((M + 2, N + 3), 7.0, device=DEV, dtype=BF16)
        args = [qa.values.data_ptr(), 208, qa.scale_tiles.data_ptr(), qb.values.data_ptr(), 208, qb.scale_tiles.data_ptr(), M,
                N, K, big[1:, 1:].data_ptr(), 1, N + 3]
        if M > fp8.FEW_ROWS:
            args += [None, 0]
        _lib.call("sffn_few_rows_fp8" if M <= fp8.FEW_ROWS else "sffn_fp8_mm", *args,
                  _lib.status_word(big.device).data_ptr(), _lib.stream_handle(big.device))
        inner = torch.zeros_like(big, dtype=torch.bool)
        inner[1:M + 1, 1:N + 1] = True
        assert (big[~inner] == 7.0).all()
        assert torch.equal(big[inner].view(M, N), sf.fp8_matmul(qa, qb))


# ---------------------------------------------------------------------------
# The linear layer
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,N,K", [(1, 64, 64), (7, 33, 65), (32, 128, 256), (33, 48, 1001), (300, 515, 130), (1024, 200, 96),
                                   (2000, 1, 3), (257, 256, 2048), (20, 2048, 8192), (48, 19001, 72), (47, 1024, 1000), (17, 1, 3)])
def test_linear(T, N, K, dtype):
    x = randn(T, K, seed=1, dtype=dtype).requires_grad_()
    W = randn(N, K, seed=2, scale=K ** -0.5, dtype=dtype).requires_grad_()
    dy = randn(T, N, seed=3, dtype=dtype)
    y = sf.ckpt_linear(x, W)
    dx, dW = torch.autograd.grad(y, [x, W], dy)
    xd, Wd, dyd = x.detach().to(F64), W.detach().to(F64), dy.to(F64)
    kept = want_blocks(x.detach())[0].to(dtype).to(F64)  # float16: its own rounding of subnormals
    close_sum(y.detach(), xd, Wd)
    close_sum(dx, dyd, Wd.T)
    close_sum(dW, dyd.T, kept.T)
    with torch.no_grad():
        assert torch.equal(sf.ckpt_linear(x, W), y)
    sf.check_status()


def test_linear_gradient_against_differences():
    """The directional derivative of sum(y * dy) along W, by central differences of
    the definition at the kept x (the product is linear: they are exact)."""
    x, W, dy = randn(200, 130, seed=1, dtype=BF16), randn(70, 130, seed=2, dtype=BF16).requires_grad_(), randn(200, 70, seed=3, dtype=BF16)
    dW = torch.autograd.grad(sf.ckpt_linear(x, W), W, dy)[0].to(F64)
    kept, v = want_blocks(x)[0], randn(70, 130, seed=4).to(F64)
    f = lambda w: ((kept @ w.T) * dy.to(F64)).sum()  # noqa: E731
    diff = (f(W.detach().to(F64) + 0.5 * v) - f(W.detach().to(F64) - 0.5 * v))
    # each element of dW is off by 2^-9 of itself, its sum by the bound above
    tol = ((2 ** -9 * dW.abs() + 80 * 2 ** -23 * (dy.to(F64).abs().T @ kept.abs())) * v.abs()).sum()
    assert (diff - (dW * v).sum()).abs() <= tol


def test_linear_keeps_half():
    """What lives between forward and backward: x in 8 bits (and the weight)."""
    x, W = randn(4096, 1024, seed=1, dtype=BF16), randn(64, 1024, seed=2, dtype=BF16).requires_grad_()
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    y = sf.ckpt_linear(x.clone(), W)
    kept = torch.cuda.memory_allocated() - base - y.numel() * 2
    assert kept <= 4096 * 1024 * (1 + 1 / 128) + 4096, kept
    y.sum().backward()
    assert W.grad.shape == W.shape


def test_linear_partial_gradients_and_leading_dimensions():
    x, W = randn(2, 50, 96, seed=1, dtype=BF16), randn(40, 96, seed=2, dtype=BF16)
    dy = randn(2, 50, 40, seed=3, dtype=BF16)
    both = torch.autograd.grad(sf.ckpt_linear(x.requires_grad_(), W.requires_grad_()), [x, W], dy)
    only_x = torch.autograd.grad(sf.ckpt_linear(x, W.detach()), x, dy)[0]
    only_W = torch.autograd.grad(sf.ckpt_linear(x.detach(), W), W, dy)[0]
    assert torch.equal(both[0], only_x) and torch.equal(both[1], only_W) and only_x.shape == x.shape
    shared = torch.autograd.grad(sf.ckpt_linear(x.detach(), W), W, dy[:, :1].expand(2, 50, 40))[0]
    assert torch.equal(shared, torch.autograd.grad(sf.ckpt_linear(x.detach(), W), W, dy[:, :1].expand(2, 50, 40).contiguous())[0])
    empty = randn(0, 96, dtype=BF16).requires_grad_()
    gx, gW = torch.autograd.grad(sf.ckpt_linear(empty, W), [empty, W], randn(0, 40, dtype=BF16))
    assert gx.shape == (0, 96) and not gW.any()


def test_linear_of_strided_operands():
    xs, Ws = randn(130, 300, seed=1, dtype=BF16), randn(300, 90, seed=2, dtype=BF16)
    for x, W in ((xs[:, 4:100], Ws[:96].T), (xs[::2, :96], Ws[::3, :][:90].T[:, :90].contiguous()[:, :1].expand(90, 96)),
                 (xs.T[:130, :96], Ws[3:99, 1:].T)):
        assert torch.equal(sf.ckpt_linear(x, W), sf.ckpt_linear(x.contiguous(), W.contiguous()))
