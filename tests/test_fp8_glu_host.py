"""CPU checks of the 8-bit blocks and the gated block: what the functions, the
ops and the C entry points refuse before any device call, the shapes and
strides torch.compile traces with, workspace and launch accounting."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import autoresearch2_b200 as sf
from autoresearch2_b200 import _lib, fp8, glu, gpt

vp = ctypes.c_void_p
P = vp(1 << 20)  # never dereferenced: the calls below fail their host checks
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ops = torch.ops.sparseffn


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cuda(*shape, dtype=BF16, **kw):
    return torch.empty(*shape, device="cuda", dtype=dtype, **kw)


def blocks(rows, width, device="cuda"):
    return sf.Fp8Tensor(torch.empty(rows, -(-width // 16) * 16, device=device, dtype=fp8.E4M3)[:, :width],
                        torch.empty(fp8._tile_shape(rows, width), device=device, dtype=torch.uint8))


def refused(error, match, f, *args, **kw):
    with pytest.raises(error, match=match):
        f(*args, **kw)


# ---------------------------------------------------------------------------
# Python
# ---------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    x, W = torch.randn(3, 32).bfloat16(), torch.randn(8, 32).bfloat16()
    refused(ValueError, "CUDA tensors only", sf.fp8_pack, x)
    refused(ValueError, "CUDA tensors only", sf.fp8_unpack, blocks(3, 32, "cpu"))
    refused(ValueError, "CUDA tensors only", sf.fp8_matmul, blocks(3, 32, "cpu"), blocks(8, 32, "cpu"))
    refused(ValueError, "CUDA tensors only", sf.fp8_matmul, x, blocks(8, 32, "cpu"))
    refused(ValueError, "CUDA tensors only", sf.ckpt_linear, x, W)
    refused(ValueError, "CUDA tensors only", sf.gated_ffn, x, W, W, W.T)
    refused(ValueError, "CUDA tensors only", ops.fp8_pack, x)
    refused(ValueError, "CUDA tensors only", ops.ckpt_linear, x, W, True)
    refused(ValueError, "CUDA tensors only", ops.gated_ffn, x, W, W, W.T, 2, 1)


def test_pack_and_unpack_refusals():
    with FakeTensorMode():
        refused(TypeError, "unsupported dtype", sf.fp8_pack, cuda(3, 32, dtype=torch.float64))
        refused(TypeError, "unsupported dtype", sf.fp8_pack, cuda(3, 32, dtype=torch.int8))
        refused(ValueError, "width >= 1", sf.fp8_pack, cuda(3, 0))
        refused(ValueError, "width >= 1", sf.fp8_pack, cuda(()))
        refused(RuntimeError, "no gradient", sf.fp8_pack, cuda(3, 32, requires_grad=True))
        refused(TypeError, "unsupported dtype", sf.fp8_unpack, blocks(3, 32), torch.int8)


def test_what_an_fp8_tensor_takes():
    v, t = torch.empty(5, 48, dtype=fp8.E4M3), torch.empty(fp8._tile_shape(5, 40), dtype=torch.uint8)
    q = sf.Fp8Tensor(v[:, :40], t)
    assert q.shape == (5, 40) and sf.Fp8Tensor(v[:, :40], t, (1, 5, 40)).shape == (1, 5, 40)
    assert q.vram_size() == 5 * 48 + 512 and "Fp8Tensor" in repr(q)
    for values, tiles, shape, match in (
            (v.view(torch.uint8)[:, :40], t, None, "float8_e4m3fn"), (v[0], t, None, "float8_e4m3fn"),
            (v[:, :0], t, None, "float8_e4m3fn"),
            (torch.empty(5, 40, dtype=fp8.E4M3), t, None, "16 bytes apart"),
            (torch.empty(48, 5, dtype=fp8.E4M3).T[:, :40], t, None, "dense rows"),
            (torch.empty(1, 40, dtype=fp8.E4M3).expand(5, 40), t, None, "16 bytes apart"),
            (v[:, :40], t[:0], None, "scale_tiles"), (v[:, :40], t.float(), None, "scale_tiles"),
            (v[:, :40], t.transpose(2, 3), None, "scale_tiles"),
            (v[:, :40], torch.empty(t.shape, dtype=torch.uint8, device="meta"), None, "scale_tiles are on"),
            (v[:, :40], t, (5, 8, 5), "not 5 rows of 40"), (v[:, :40], t, (4, 40), "not 5 rows of 40"), (v[:, :40], t, (), "not 5 rows")):
        refused(ValueError, match, sf.Fp8Tensor, values, tiles, shape)


def test_exponents_by_row_and_block():
    rows, width = 300, 1100
    nb = 9
    e = torch.arange(rows * nb).view(rows, nb) % 200
    byte = torch.zeros(384, 12, dtype=torch.uint8)
    byte[:rows, :nb] = e.to(torch.uint8)
    tiles = torch.zeros(3, 3, 32, 4, 4, dtype=torch.uint8)
    for r in range(384):
        for k in range(12):
            tiles[r // 128, k // 4, r % 32, r % 128 // 32, k % 4] = byte[r, k]
    q = sf.Fp8Tensor(torch.empty(rows, 1104, dtype=fp8.E4M3)[:, :width], tiles)
    assert torch.equal(q.exponents, e.int() - 127)


def test_product_refusals():
    with FakeTensorMode():
        a, b = blocks(3, 64), blocks(8, 64)
        refused(TypeError, "b must be an Fp8Tensor", sf.fp8_matmul, a, cuda(8, 64))
        b3 = sf.Fp8Tensor(b.values, b.scale_tiles, (1, 8, 64))
        refused(TypeError, "b must be an Fp8Tensor", sf.fp8_matmul, a, b3)
        refused(ValueError, "rows of 64, b of 80", sf.fp8_matmul, a, blocks(8, 80))
        refused(ValueError, "rows of 63, b of 64", sf.fp8_matmul, cuda(3, 63), b)
        refused(TypeError, "out_dtype", sf.fp8_matmul, a, b, F32)
        refused(RuntimeError, "no gradient", sf.fp8_matmul, cuda(3, 64, requires_grad=True), b)
        refused(TypeError, "unsupported dtype", sf.fp8_matmul, cuda(3, 64, dtype=torch.int32), b)


def test_linear_refusals():
    with FakeTensorMode():
        f = sf.ckpt_linear
        refused(TypeError, "unsupported dtype", f, cuda(3, 32, dtype=F32), cuda(8, 32, dtype=F32))
        refused(TypeError, "W is torch.float16", f, cuda(3, 32), cuda(8, 32, dtype=F16))
        refused(ValueError, r"W must be \(8, 32\)", f, cuda(3, 32), cuda(8, 33))
        refused(ValueError, "W must be", f, cuda(3, 32), cuda(32))
        refused(ValueError, "W must be", f, cuda(3, 32), cuda(0, 32))
        refused(ValueError, "width >= 1", f, cuda(3, 0), cuda(8, 0))
        refused(ValueError, "width >= 1", f, cuda(()), cuda(8, 1))
        refused(ValueError, "CUDA tensors only", f, cuda(3, 32), torch.empty(8, 32, dtype=BF16, device="meta"))


def test_gated_refusals():
    with FakeTensorMode():
        f = sf.gated_ffn
        x, Wg, W2 = cuda(3, 32), cuda(80, 32), cuda(32, 80)
        refused(ValueError, "activation must be one of", f, x, Wg, Wg, W2, "tanh")
        refused(ValueError, "checkpoint must be", f, x, Wg, Wg, W2, checkpoint="int8")
        refused(TypeError, "unsupported dtype", f, x.float(), Wg.float(), Wg.float(), W2.float())
        refused(TypeError, "Wu is torch.float16", f, x, Wg, Wg.half(), W2)
        refused(ValueError, r"Wu must be \(80, 32\)", f, x, Wg, cuda(81, 32), W2)
        refused(ValueError, r"W2 must be \(32, 80\)", f, x, Wg, Wg, cuda(80, 32))
        refused(ValueError, "Wg must be", f, x, cuda(80, 31), Wg, W2)
        refused(ValueError, "Wg must be", f, x, cuda(80), Wg, W2)
        refused(ValueError, "CUDA tensors only", f, x, Wg, Wg, torch.empty(32, 80, dtype=BF16, device="meta"))


def test_backward_ops_refuse_what_no_forward_keeps():
    def rows(T, F, ld, **kw):
        return torch.empty(T, ld, dtype=BF16, **kw)[:, :F]

    dy, q = torch.empty(3, 32, dtype=BF16), blocks(3, 80, "cpu")
    g = rows(3, 76, 80)
    ok = (dy, dy, 76, g, g, None, None, None, None)
    glu._check_kept(*ok)
    for i, bad in ((1, dy[:2]), (1, dy.half()), (3, rows(3, 75, 80)), (3, rows(3, 76, 88)), (4, g.half()), (3, torch.empty(3, 76, dtype=BF16)),
                   (4, rows(3, 76, 80, device="meta"))):
        refused(ValueError, "as the forward kept", glu._check_kept, *ok[:i], bad, *ok[i + 1:])
    x8 = blocks(3, 32, "cpu")
    ok = (dy, None, 80, q.values, q.values, q.scale_tiles, q.scale_tiles, x8.values, x8.scale_tiles)
    glu._check_kept(*ok)
    for i, bad in ((3, blocks(3, 96, "cpu").values), (7, q.values), (5, q.scale_tiles[:0]), (8, x8.scale_tiles.float())):
        refused(ValueError, "as the forward kept|scale_tiles", glu._check_kept, *ok[:i], bad, *ok[i + 1:])


def test_gpt_config_refusals():
    c = dict(n_layer=1, n_head=2, n_embd=32, ffn_hidden=64, vocab=64, seq_len=8)
    refused(ValueError, "gated must be one of", gpt.GPT, gpt.GPTConfig(**c, gated="tanh"), device="cpu")
    refused(ValueError, "ckpt8 goes with gated", gpt.GPT, gpt.GPTConfig(**c, ckpt8=True), device="cpu")
    m = gpt.GPT(gpt.GPTConfig(**c, gated="silu"), sparse=False, device="cpu", dtype=F32)
    idx = torch.zeros(2, 8, dtype=torch.long)
    assert m(idx).shape == (2, 8, 64)
    m(idx, idx).backward()
    assert all(p.grad is not None for p in m.blocks.parameters())
    refused(ValueError, "without gradients", m, idx, weights=[{}])
    with torch.no_grad():
        refused(ValueError, "one dict a block", m, idx, weights=[{}, {}])
    assert gpt.flops_per_token(gpt.GPTConfig(**c, gated="silu")) - gpt.flops_per_token(gpt.GPTConfig(**c)) == 6 * 32 * 64


# ---------------------------------------------------------------------------
# Tracing
# ---------------------------------------------------------------------------
def test_fake_kernels():
    with FakeTensorMode():
        x, W = cuda(2, 65, 100), cuda(48, 100)
        v, t = ops.fp8_pack(x)
        assert v.shape == (130, 100) and v.stride() == (112, 1) and v.dtype == fp8.E4M3 and t.shape == (2, 1, 32, 4, 4)
        assert ops.fp8_unpack(v, t, [2, 65, 100], F16).shape == (2, 65, 100)
        wv, wt = ops.fp8_pack(W)
        y = ops.fp8_matmul(v, t, wv, wt, F16)
        assert y.shape == (130, 48) and y.dtype == F16
        y, v, t = ops.ckpt_linear(x, W, True)
        assert y.shape == (2, 65, 48) and v.shape == (130, 100) and t.dtype == torch.uint8
        assert [s.numel() for s in ops.ckpt_linear(x, W, False)[1:]] == [0, 0]
        dx, dW = ops.ckpt_linear_bwd(y, W, v, t, [2, 65, 100], True, True)
        assert dx.shape == x.shape and dW.shape == W.shape
        Wg, W2 = cuda(75, 100), cuda(100, 75)
        for keep in (0, 1, 2):
            y, g, u, gt, ut, xv, xt = ops.gated_ffn(x, Wg, Wg, W2, 2, keep)
            assert y.shape == x.shape
            if keep == 1:
                assert g.shape == (130, 75) and g.stride() == (80, 1) and u.dtype == BF16
            if keep == 2:
                assert g.stride() == (80, 1) and g.dtype == fp8.E4M3 and xv.stride() == (112, 1)
            if keep:
                grads = ops.gated_ffn_bwd(y, x if keep == 1 else None, Wg, Wg, W2, g, u, gt, ut, xv, xt, 2, [True] * 4)
                assert [tuple(a.shape) for a in grads] == [(2, 65, 100), (75, 100), (75, 100), (100, 75)]


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_compile_traces_without_a_graph_break(checkpoint):
    from torch._dynamo.backends.common import aot_autograd
    graphs = []

    def record(gm, example_inputs):
        graphs.append(gm.code)
        return gm

    def block(x, W, Wg, Wu, W2):
        return ops.gated_ffn(ops.ckpt_linear(x, W, True)[0], Wg, Wu, W2, 2, glu.KEEP[checkpoint])[0].float().square().sum()

    torch._dynamo.reset()
    f = torch.compile(block, backend=aot_autograd(fw_compiler=record, bw_compiler=record), fullgraph=True)
    args = [torch.empty(*s, device="meta", dtype=BF16, requires_grad=True) for s in ((64, 32), (48, 32), (96, 48), (96, 48), (48, 96))]
    f(*args).backward()
    fw, bw = graphs
    assert fw.count("sparseffn.gated_ffn") == 1 and fw.count("sparseffn.ckpt_linear") == 1
    assert bw.count("sparseffn.gated_ffn_bwd") == 1 and bw.count("sparseffn.ckpt_linear_bwd") == 1
    assert all(a.grad is not None and a.grad.shape == a.shape for a in args)
    torch._dynamo.reset()


# ---------------------------------------------------------------------------
# C entry points
# ---------------------------------------------------------------------------
def rc(f, ok, **change):
    a = list(ok)
    for k, v in change.items():
        a[int(k[1:])] = v
    return f(*a)


ODD = vp((1 << 20) + 2)  # 2 bytes off
BIG = 1 << 40


def test_pack_entry(lib):
    ok = [P, 1, 10, 40, 40, P, 48, P, None]
    f = lib.sffn_fp8_pack
    assert rc(f, ok, _1=3) == 2 and rc(f, ok, _2=-1) == 1 and rc(f, ok, _3=-1) == 1 and rc(f, ok, _2=0) == 0 and rc(f, ok, _3=0) == 0
    assert rc(f, ok, _0=None) == 1 and rc(f, ok, _5=None) == 1 and rc(f, ok, _7=None) == 1
    assert rc(f, ok, _4=39) == 1 and rc(f, ok, _6=32) == 1
    assert rc(f, ok, _6=56) == 3 and rc(f, ok, _5=ODD) == 3 and rc(f, ok, _0=vp((1 << 20) + 1)) == 3 and rc(f, ok, _0=ODD, _1=0) == 3
    ok = [P, 48, P, 10, 40, 1, P, 40, None]
    f = lib.sffn_fp8_unpack
    assert rc(f, ok, _5=-1) == 2 and rc(f, ok, _3=-1) == 1 and rc(f, ok, _3=0) == 0
    assert rc(f, ok, _0=None) == 1 and rc(f, ok, _2=None) == 1 and rc(f, ok, _6=None) == 1 and rc(f, ok, _7=39) == 1 and rc(f, ok, _1=32) == 1
    assert rc(f, ok, _0=ODD) == 3 and rc(f, ok, _1=41) == 3


def test_product_entries(lib):
    for f, few in ((lib.sffn_fp8_mm, False), (lib.sffn_few_rows_fp8, True)):
        ok = [P, 48, P, P, 48, P, 100, 8, 40, P, 1, 8, None, 0, P, None]
        if few:
            ok[6:] = [10, 8, 40, P, 1, 8, P, None]
            assert rc(f, ok, _6=65) == 1
        assert rc(f, ok, _10=0) == 2 and rc(f, ok, _6=-1) == 1 and rc(f, ok, _8=0) == 1 and rc(f, ok, _6=0) == 0 and rc(f, ok, _7=0) == 0
        for i in (0, 2, 3, 5, 9, len(ok) - 2):
            assert rc(f, ok, **{f"_{i}": None}) == 1
        assert rc(f, ok, _1=32) == 1 and rc(f, ok, _4=32) == 1 and rc(f, ok, _11=7) == 1
        assert rc(f, ok, _1=56) == 3 and rc(f, ok, _0=ODD) == 3 and rc(f, ok, _3=ODD) == 3 and rc(f, ok, _9=vp((1 << 20) + 1)) == 3
        assert rc(f, ok, _2=ODD) == 3 and rc(f, ok, _5=ODD) == 3
        assert rc(f, ok, _7=BIG, _11=BIG) == 8
    f, ok = lib.sffn_fp8_mm, [P, 16384, P, P, 16384, P, 100, 512, 16384, P, 1, 512, P, 1 << 30, P, None]
    assert rc(f, ok, _6=BIG) == 8 and rc(f, ok, _12=None) == 4 and rc(f, ok, _13=100) == 4 and rc(f, ok, _12=ODD) == 3
    w = lib.sffn_fp8_mm_workspace_bytes
    assert w(16384, 8192, 4096) == 0 and w(0, 8, 8) == 0 and w(100, 512, 16384) % (100 * 512 * 4) == 0 and w(100, 512, 16384)
    f, ok = lib.sffn_fp8_linear, [P, 1, 40, P, 48, P, 100, 8, 40, P, 1, 8, P, 1 << 20, P, None]
    assert lib.sffn_fp8_linear_workspace_bytes(100, 8, 40) == 100 * 48 + (-100 * 48) % 256 + 512
    assert rc(f, ok, _1=3) == 2 and rc(f, ok, _6=0) == 1 and rc(f, ok, _0=None) == 1 and rc(f, ok, _12=None) == 4 and rc(f, ok, _13=100) == 4
    assert rc(f, ok, _12=ODD) == 3


def test_gemm_entry(lib):
    ok = [1, P, 40, 0, P, 40, 0, None, 0, None, 0, 0, 100, 64, 40, P, 64, None, 0, P, None]
    f = lib.sffn_gemm16
    assert rc(f, ok, _0=0) == 2 and rc(f, ok, _12=-1) == 1 and rc(f, ok, _14=0) == 1 and rc(f, ok, _11=-1) == 1 and rc(f, ok, _12=0) == 0
    for i in (1, 4, 15, 19):
        assert rc(f, ok, **{f"_{i}": None}) == 1
    assert rc(f, ok, _2=32) == 1 and rc(f, ok, _5=32) == 1 and rc(f, ok, _16=63) == 1 and rc(f, ok, _3=1, _2=96) == 1
    assert rc(f, ok, _11=8) == 1 and rc(f, ok, _11=8, _7=P, _8=8, _9=P, _10=0) == 1
    assert rc(f, ok, _2=44) == 3 and rc(f, ok, _1=ODD) == 3 and rc(f, ok, _15=vp((1 << 20) + 1)) == 3 and rc(f, ok, _17=ODD, _18=99) == 3
    assert rc(f, ok, _11=8, _7=ODD, _8=8, _9=P, _10=8) == 3 and rc(f, ok, _12=BIG) == 8


def test_gated_entries(lib):
    up = [1, 2, P, 32, P, 32, P, 32, 100, 32, 76, P, 80, 1, P, P, 80, None, None, P, None]
    f = lib.sffn_glu_up
    assert rc(f, up, _0=0) == 2 and rc(f, up, _1=4) == 1 and rc(f, up, _13=3) == 1 and rc(f, up, _9=0) == 1 and rc(f, up, _8=0) == 0
    for i in (2, 4, 6, 11, 14, 15, 19):
        assert rc(f, up, **{f"_{i}": None}) == 1
    assert rc(f, up, _13=2) == 1 and rc(f, up, _16=75) == 1 and rc(f, up, _12=75) == 1 and rc(f, up, _3=24) == 1
    assert rc(f, up, _16=76) == 3 and rc(f, up, _13=2, _17=P, _18=P, _16=88) == 3 and rc(f, up, _14=ODD) == 3 and rc(f, up, _12=84) == 3
    assert rc(f, up, _4=ODD) == 3 and rc(f, up, _8=BIG) == 8
    dg = [1, 2, P, 32, P, 80, 100, 32, 76, 1, P, P, 80, None, None, P, P, 160, P, 80, P, None]
    f = lib.sffn_glu_dgrad
    assert rc(f, dg, _9=0) == 1 and rc(f, dg, _0=0) == 2 and rc(f, dg, _6=0) == 0 and rc(f, dg, _9=2) == 1
    for i in (2, 4, 10, 11, 15, 16, 18, 20):
        assert rc(f, dg, **{f"_{i}": None}) == 1
    assert rc(f, dg, _5=72) == 1 and rc(f, dg, _17=72) == 1 and rc(f, dg, _19=72) == 1 and rc(f, dg, _19=84) == 3 and rc(f, dg, _16=ODD) == 3


def test_few_row_entries(lib):
    mm = [1, P, 40, P, 40, 10, 64, 40, P, 64, P, None]
    f = lib.sffn_few_rows_mm
    assert rc(f, mm, _0=0) == 2 and rc(f, mm, _5=65) == 1 and rc(f, mm, _7=0) == 1 and rc(f, mm, _5=0) == 0 and rc(f, mm, _6=0) == 0
    for i in (1, 3, 8, 10):
        assert rc(f, mm, **{f"_{i}": None}) == 1
    assert rc(f, mm, _2=39) == 1 and rc(f, mm, _4=39) == 1 and rc(f, mm, _9=63) == 1 and rc(f, mm, _1=vp((1 << 20) + 1)) == 3
    # more than 16 rows: only on 16 bytes
    assert rc(f, mm, _5=17, _2=41) == 3 and rc(f, mm, _5=17, _4=44) == 3 and rc(f, mm, _5=64, _3=vp((1 << 20) + 8)) == 3
    f = lib.sffn_few_rows_ffn
    b = [1, 2, P, 40, P, 40, P, 40, P, 64, 10, 40, 64, P, 64, P, 40, P, None]
    assert rc(f, b, _0=0) == 2 and rc(f, b, _1=-1) == 1 and rc(f, b, _13=None) == 1 and rc(f, b, _10=65) == 1 and rc(f, b, _10=0) == 0 and rc(f, b, _5=39) == 1
    for i in (3, 5, 7, 9, 14):
        assert rc(f, b, _10=17, **{f"_{i}": 68}) == 3, i


def test_pad_entry(lib):
    f = lib.sffn_pad_rows16
    d = (ctypes.c_int64 * 6)(1 << 20, 3, 5, 5, 1 << 21, 8)
    assert f(0, None, None) == 0 and f(1, None, None) == 1 and f(5, ctypes.addressof(d), None) == 1
    for i, v, want in ((1, -1, 1), (2, -1, 1), (5, 4, 1), (0, 0, 1), (4, 0, 1), (5, 12, 3), (4, (1 << 21) + 8, 3), (0, (1 << 20) + 1, 3), (1, 0, 0)):
        c = (ctypes.c_int64 * 6)(*d)
        c[i] = v
        assert f(1, ctypes.addressof(c), None) == want, (i, v)


def test_workspace_and_launches(lib):
    w = lib.sffn_gemm16_workspace_bytes
    assert w(16384, 4096, 4096, 0) == 0 and w(0, 8, 8, 0) == 0 and w(8, 8, -1, 0) == 0
    n = w(768, 2001, 32768, 0)
    assert n and n % (768 * 2004 * 4) == 0  # float32 parts, rows of a multiple of 4
    assert w(768, 2001, 16384, 16384) == n
    a = [None] * 21
    assert _lib._launches("sffn_gemm16", a) == 1
    a[18] = n
    b = [None] * 6 + [100, 512, 16384] + [None] * 7
    assert _lib._launches("sffn_fp8_mm", b) == 1 and _lib._launches("sffn_fp8_linear", b) == 3
    b[6], b[12] = 16, 1
    assert _lib._launches("sffn_fp8_mm", b) == 2 and _lib._launches("sffn_fp8_linear", b) == 2
    assert _lib._launches("sffn_gemm16", a) == 2 and _lib._launches("sffn_few_rows_ffn", []) == 2


def test_launches_of_the_blocks():
    f = _lib._launches
    linear = lambda T, N, K, odd=0, keep=1: f("sffn_ckpt_linear", [1, 1, K, 1, K, odd, T, N, K, 1, keep, 1, 1, 0, 1, 0])  # noqa: E731
    assert linear(8, 64, 64) == 2 and linear(8, 64, 64, 1) == 3 and linear(8, 64, 64, 3, None) == 1 and linear(4096, 4096, 64) == 2 and linear(4096, 4096, 63, 1) == 3
    bwd = lambda T, N, K, dx, dW, odd=0: f("sffn_ckpt_linear_bwd", [1, 1, N, 1, K, odd, 1, K, 1, T, N, K, dx, dW, 1, 0, 1, 0])  # noqa: E731
    assert bwd(4096, 4096, 4096, 1, 1) == 3 and bwd(4096, 4096, 4096, None, 1, 2) == 2 and bwd(4096, 4096, 4096, 1, None, 2) == 2
    assert bwd(32768, 768, 768, 1, 1) == 4  # the weight gradient in parts, joined
    up = lambda keep, T, odd=0: f("sffn_gated_ffn", [1, 2, keep, 1, 64, 1, 64, 1, 64, 1, 64, odd, T, 64, 64])  # noqa: E731
    assert up(0, 8) == 2 and up(0, 8, 9) == 3 and up(0, 8, 3) == 2 and up(0, 64) == 2 and up(1, 8) == 2 and up(2, 8) == 3 and up(2, 64, 1) == 4 and up(1, 8, 8) == 2
    T, D, F = 4096, 4096, 4096
    down = lambda keep, steps, dx, dwg, dwu, dw2, odd=0: f("sffn_gated_ffn_bwd", [  # noqa: E731
        1, 2, keep, steps, 1, D, 1, D, 1, D, 1, D, 1, F, odd, 1, 1, 1, 1, 1, 1, T, D, F, dx, dwg, dwu, dw2, 1, 0, 1, 0])
    assert down(1, 15, 1, 16, 16 + F * D * 2, 1) == 4 and down(2, 15, 1, 16, 16 + F * D * 2, 1) == 5
    assert down(1, 15, 1, 16, 32, 1, 16) == 6 and down(1, 1, 1, 16, 32, 1) == 1 and down(1, 6, 1, None, None, 1) == 1


def test_block_entries(lib):
    w = lib.sffn_ckpt_linear_workspace_bytes
    assert w(0, 0, 0, 64, 64, 64) == 0 and w(0, 3, 0, 8, 64, 64) == 0 and w(0, 1, 0, 64, 64, 63) == 64 * 64 * 2
    assert w(1, 0, 1, 64, 64, 64) == 0 and w(1, 0, 2, 64, 64, 63) >= 64 * 64 * 2 and w(0, 0, 0, 0, 64, 64) == 0
    ok = [1, P, 64, P, 64, 0, 100, 64, 64, P, P, P, None, 0, P, None]
    f = lib.sffn_ckpt_linear
    assert rc(f, ok, _0=0) == 2 and rc(f, ok, _6=0) == 1 and rc(f, ok, _1=None) == 1 and rc(f, ok, _14=None) == 1
    assert rc(f, ok, _5=1) == 4 and rc(f, ok, _5=1, _12=P, _13=100) == 4 and rc(f, ok, _5=1, _12=ODD, _13=1 << 20) == 3
    ok = [1, P, 64, P, 64, 0, P, 64, P, 100, 64, 64, P, P, P, 1 << 20, P, None]
    f = lib.sffn_ckpt_linear_bwd
    assert rc(f, ok, _0=0) == 2 and rc(f, ok, _9=0) == 1 and rc(f, ok, _14=None) == 4 and rc(f, ok, _15=100) == 4 and rc(f, ok, _1=None) == 1
    w = lib.sffn_gated_ffn_workspace_bytes
    assert w(0, 0, 0, 0, 64, 64, 64) == 64 * 64 * 2 and w(1, 1, 0, 15, 4096, 4096, 4096) == 3 * 4096 * 4096 * 2
    assert w(1, 2, 0, 15, 4096, 4096, 4096) == 4 * 4096 * 4096 * 2 and w(0, 1, 0, 0, 64, 0, 64) == 0
    ok = [1, 2, 1, P, 64, P, 64, P, 64, P, 64, 0, 100, 64, 64, P, P, P, None, None, None, None, P, 1 << 20, P, None]
    f = lib.sffn_gated_ffn
    assert rc(f, ok, _0=0) == 2 and rc(f, ok, _2=3) == 1 and rc(f, ok, _12=0) == 1 and rc(f, ok, _22=None) == 4 and rc(f, ok, _23=8) == 4
    ok = [1, 2, 1, 15, P, 64, P, 64, P, 64, P, 64, P, 64, 0, P, P, None, None, None, None, 100, 64, 64, P, P, P, P, P, 1 << 24, P, None]
    f = lib.sffn_gated_ffn_bwd
    assert rc(f, ok, _0=0) == 2 and rc(f, ok, _2=0) == 1 and rc(f, ok, _21=0) == 1 and rc(f, ok, _28=None) == 4 and rc(f, ok, _29=8) == 4
