"""CPU checks of token_logprobs, distill_topk and residual_norm: what the
Python functions and the C entry points refuse before any device call, the
shapes torch.compile traces with, and the launch accounting."""
import ctypes
import threading

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import autoresearch2_b200 as sf
from autoresearch2_b200 import _lib, logits, norms

vp, i64, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float
P = vp(1 << 20)  # never dereferenced: the calls below fail their host checks
INF = float("inf")


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cuda(*shape, dtype=torch.float32, **kw):
    return torch.empty(*shape, device="cuda", dtype=dtype, **kw)


def refused(error, match, f, *args, **kw):
    with pytest.raises(error, match=match):
        f(*args, **kw)


def test_cpu_tensors_are_refused():
    x, t = torch.randn(3, 10), torch.zeros(3, dtype=torch.long)
    refused(ValueError, "CUDA tensors only", sf.token_logprobs, x, t)
    refused(ValueError, "CUDA tensors only", sf.distill_topk, x, t[:, None], torch.zeros(3, 1))
    refused(ValueError, "CUDA tensors only", sf.residual_norm, x, x)


def test_token_logprobs_refusals():
    with FakeTensorMode():
        x, t = cuda(3, 10), cuda(3, dtype=torch.long)
        f = sf.token_logprobs
        refused(TypeError, "unsupported dtype", f, cuda(3, 10, dtype=torch.float64), t)
        refused(TypeError, "int64 or int32", f, x, cuda(3))
        refused(TypeError, "int64 or int32", f, x, cuda(3, dtype=torch.int16))
        refused(ValueError, "shape", f, x, cuda(4, dtype=torch.long))
        refused(ValueError, "shape", f, x, cuda(3, 1, dtype=torch.long))
        refused(ValueError, "V >= 1", f, cuda(3, 0), t)
        refused(ValueError, "V >= 1", f, cuda(()), t)
        refused(ValueError, "CUDA tensors only", f, x, torch.zeros(3, dtype=torch.long, device="meta"))
        for k in (-1, 11, 2.0, True):
            refused(ValueError, "top_k", f, x, t, top_k=k)
        refused(ValueError, "top_k", f, cuda(3, 1000), t, top_k=129)
        for temperature in (0, -1.0, INF, float("nan"), 1e-320, 2e-39, 1e-31, 1e31, "1"):
            refused(ValueError, "temperature", f, x, t, temperature=temperature)


def test_distill_topk_refusals():
    with FakeTensorMode():
        x, ids, c = cuda(3, 200), cuda(3, 4, dtype=torch.long), cuda(3, 4)
        f = sf.distill_topk
        refused(ValueError, "tail", f, x, ids, c, tail="none")
        refused(ValueError, "1 <= K <= 128", f, x, cuda(3, 0, dtype=torch.long), cuda(3, 0))
        refused(ValueError, "1 <= K <= 128", f, x, cuda(3, 129, dtype=torch.long), cuda(3, 129))
        refused(ValueError, "1 <= K <= 128", f, x, None, c)
        refused(TypeError, "int64 or int32", f, x, c, c)
        refused(ValueError, "shape", f, x, cuda(2, 4, dtype=torch.long), c)
        refused(ValueError, "shape", f, x, ids, cuda(3, 5))
        refused(TypeError, "unsupported dtype", f, x, ids, cuda(3, 4, dtype=torch.float64))
        refused(ValueError, "temperature", f, x, ids, c, temperature=0.0)
        refused(ValueError, "detach", f, x, ids, cuda(3, 4, requires_grad=True))


def test_residual_norm_refusals():
    with FakeTensorMode():
        f = sf.residual_norm
        bf = torch.bfloat16
        x, w = cuda(6, 8), cuda(8)
        refused(ValueError, "1 <= D <= 16384", f, cuda(2, 16385))
        refused(ValueError, "1 <= D <= 16384", f, cuda(2, 0))
        refused(ValueError, "1 <= D <= 16384", f, cuda(()))
        refused(TypeError, "unsupported dtype", f, cuda(2, 8, dtype=torch.float64))
        refused(TypeError, "x is", f, cuda(6, 8, dtype=bf), cuda(6, 8))
        refused(TypeError, "x is", f, cuda(6, 8, dtype=bf), cuda(6, 8, dtype=torch.float16))
        refused(TypeError, "out_dtype", f, x, x, out_dtype=bf)
        refused(TypeError, "x is", f, x, out_dtype=torch.int32)
        refused(ValueError, "x's shape", f, x, cuda(5, 8))
        refused(ValueError, "pre_weight", f, x, x, cuda(9))
        refused(ValueError, "post_weight", f, x, x, w, cuda(1, 8), post_norm=True)
        refused(ValueError, "post_norm=True", f, x, x, w, w)
        refused(ValueError, "go with a block output", f, x, None, w, residual_scale=0.5)
        refused(ValueError, "go with a block output", f, x, gate=w)
        for eps in (0.0, -1e-6, INF, float("nan"), 1e-40):
            refused(ValueError, "eps", f, x, x, eps=eps)
        for scale in (INF, -1e39, float("nan")):
            refused(ValueError, "residual_scale", f, x, x, residual_scale=scale)
        refused(ValueError, "evenly", f, x, x, gate=cuda(4, 8))
        refused(ValueError, "last dimension", f, x, x, gate=cuda(6, 1))
        y = cuda(2, 3, 8)
        for shape in ((1, 3, 8), (3, 1, 8), (2, 2, 8), (1, 2, 3, 8)):
            refused(ValueError, "leading dimensions", f, y, y, gate=cuda(*shape))
        refused(ValueError, "evenly", f, y, y, gate=cuda(4, 8))
        refused(ValueError, "CUDA tensors only", f, x, x, torch.empty(8, device="meta"))


def test_row_maps():
    """How leading dimensions become rows: the strides handed to the kernels."""
    base = torch.empty(4, 6, 30)
    rows = lambda t: logits._rows(t)[1:]  # noqa: E731
    assert rows(base) == (24, 24, 0, 30)
    assert rows(torch.empty(5)) == (1, 1, 0, 5)
    assert rows(base[..., :20]) == (24, 24, 0, 30)
    assert rows(base[:, 1:]) == (20, 5, 180, 30)
    assert rows(base[:, 2]) == (4, 4, 0, 180)
    assert rows(base[0, 0]) == (1, 1, 0, 30) and rows(base[0, 0, :7]) == (1, 1, 0, 7)
    assert rows(base.transpose(0, 1)) == (24, 4, 30, 180)
    assert rows(base[:1].expand(4, 6, 30)) == (24, 6, 0, 30)
    assert rows(base.transpose(1, 2)) == (120, 120, 0, 6)  # copied
    assert rows(torch.empty(2, 3, 4, 50)[:, :2, 1:, :7]) == (12, 12, 0, 7)  # three strides: copied
    assert rows(torch.empty(0, 5)) == (0, 0, 0, 5) and rows(torch.empty(3, 0, 9)[..., :5])[0] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_lie_as_their_logits(dtype):
    base = torch.empty(8, 1000, dtype=dtype)
    for x in (base, base[:, :777], base[:, 3:700], base[:, :998], base[0], base[:1, 1:]):
        x, rows, _, _, step = logits._rows(x)
        grad, ld = logits._grad_like(x, rows, step)
        assert grad.shape == x.shape and (rows == 1 or grad.stride(0) == ld)
        for r in range(rows):
            a, b = (t.data_ptr() + r * s * t.element_size() for t, s in ((x, step), (grad, ld)))
            assert a % 16 == b % 16


def test_fake_kernels():
    ops = torch.ops.sparseffn
    with FakeTensorMode():
        x = cuda(2, 5, 300, dtype=torch.bfloat16)
        logp, ent, ids, top, stats = ops.token_logprobs(x, cuda(2, 5, dtype=torch.long), 7, 1.0, -100)
        assert logp.shape == ent.shape == (2, 5) and ids.shape == top.shape == (2, 5, 7) and stats.shape == (2, 5, 2)
        assert ids.dtype == torch.int64 and logp.dtype == torch.float32
        assert ops.token_logprobs(x, None, 0, 1.0, -100)[0].shape == (0,)
        loss, stats = ops.distill_topk(x, ids, top, 1.0, "renorm")
        assert loss.shape == (2, 5) and stats.shape == (2, 5, 4)
        a, h, stats = ops.residual_norm(cuda(4, 8), cuda(4, 8, dtype=torch.bfloat16), None, None, None, 1, False, 1.0,
                                        1e-6, torch.bfloat16)
        assert a.dtype == torch.float32 and h.dtype == torch.bfloat16 and stats.shape == (4, 2)
        assert ops.residual_norm(cuda(4, 8), None, None, None, None, 1, False, 1.0, 1e-6,
                                 torch.float32)[0].shape == (0,)


def test_c_scores_refusals(lib):
    ok = [P, 0, 4, 100, 4, 0, 100, P, 8, -100, 5, 1.0, P, P, P, P, P, P, None]

    def rc(**changes):
        a = list(ok)
        for k, v in changes.items():
            a[int(k[1:])] = v
        return lib.sffn_token_logprobs(*a)

    assert rc(_1=3) == 2 and rc(_2=-1) == 1 and rc(_3=0) == 1 and rc(_4=0) == 1 and rc(_5=-1) == 1
    assert rc(_0=None) == 1 and rc(_0=vp(2)) == 3 and rc(_0=vp(3), _1=1) == 3
    assert rc(_8=2) == 1 and rc(_10=-1) == 1 and rc(_10=101) == 1 and rc(_3=1000, _10=129) == 8
    for t in (0.0, -1.0, INF, float("nan"), 3e30):
        assert rc(_11=t) == 1
    for i in (12, 13, 15, 16, 17):
        assert rc(**{f"_{i}": None}) == 1
    assert rc(_3=1 << 31) == 8 and rc(_2=1 << 32) == 8
    assert rc(_2=0, _0=None) == 0  # no rows: nothing to do
    for i, off in ((7, 4), (12, 2), (13, 2), (14, 2), (15, 4), (16, 2), (17, 1)):
        assert rc(**{f"_{i}": vp((1 << 20) + off)}) == 3

    ok = [P, 0, 4, 100, 4, 0, 100, P, 8, -100, P, 5, 1.0, P, P, P, P, P, P, 100, None]

    def rc(**changes):
        a = list(ok)
        for k, v in changes.items():
            a[int(k[1:])] = v
        return lib.sffn_token_logprobs_bwd(*a)

    assert rc(_1=5) == 2 and rc(_19=99) == 1 and rc(_18=vp(2)) == 3 and rc(_10=None) == 1 and rc(_11=200) == 1
    for i in (13, 14, 18):
        assert rc(**{f"_{i}": None}) == 1


def test_c_distill_refusals(lib):
    ok = [P, 1, 4, 100, 4, 0, 100, P, 8, P, 0, 5, 1, 1.0, P, P, P, None]

    def rc(f, base, **changes):
        a = list(base)
        for k, v in changes.items():
            a[int(k[1:])] = v
        return f(*a)

    f = lib.sffn_distill_topk
    assert rc(f, ok, _1=7) == 2 and rc(f, ok, _10=7) == 2 and rc(f, ok, _8=1) == 1 and rc(f, ok, _11=0) == 1
    assert rc(f, ok, _11=129) == 8 and rc(f, ok, _12=2) == 1 and rc(f, ok, _3=1 << 24, _6=1 << 24) == 8
    for i in (7, 9, 14, 16):
        assert rc(f, ok, **{f"_{i}": None}) == 1
    ok = [P, 1, 4, 100, 4, 0, 100, P, 8, P, 0, 5, 1, 1.0, P, P, P, 100, None]
    f = lib.sffn_distill_topk_bwd
    assert rc(f, ok, _17=50) == 1 and rc(f, ok, _16=vp(1)) == 3 and rc(f, ok, _12=-1) == 1
    for i in (7, 9, 14, 15, 16):
        assert rc(f, ok, **{f"_{i}": None}) == 1


def test_c_norm_refusals(lib):
    ok = [P, 0, 64, P, 1, 64, 10, 64, P, 0, P, 0, P, 0, 5, 1, 1.0, 1e-6, P, P, P, P, None]

    def rc(f, base, **changes):
        a = list(base)
        for k, v in changes.items():
            a[int(k[1:])] = v
        return f(*a)

    f = lib.sffn_residual_norm
    assert rc(f, ok, _1=1, _4=2) == 2 and rc(f, ok, _1=1, _4=0) == 2 and rc(f, ok, _9=4) == 2
    assert rc(f, ok, _6=-1) == 1 and rc(f, ok, _7=0) == 1 and rc(f, ok, _7=16385) == 8 and rc(f, ok, _14=0) == 1
    assert rc(f, ok, _3=None) == 1 and rc(f, ok, _15=0) == 1 and rc(f, ok, _17=0.0) == 1
    assert rc(f, ok, _0=None) == 1 and rc(f, ok, _18=None) == 1 and rc(f, ok, _19=None) == 1 and rc(f, ok, _21=None) == 1
    assert rc(f, ok, _6=0) == 0
    for i, off in ((0, 2), (3, 1), (8, 2), (10, 2), (12, 2), (18, 2), (19, 1), (20, 4)):
        assert rc(f, ok, **{f"_{i}": vp((1 << 20) + off)}) == 3
    b = [P, 0, 64, P, 1, 64, 10, 64, P, 0, P, 0, P, 0, 5, 1, 1.0, P, P, P, P, P, P, P, P, P, 1 << 20, P, None]
    f = lib.sffn_residual_norm_bwd
    need = lib.sffn_residual_norm_bwd_workspace_bytes(10, 64, 5)
    assert rc(f, b, _26=need - 1) == 4 and rc(f, b, _25=None) == 3 and rc(f, b, _25=vp(8)) == 3
    assert rc(f, b, _8=None) == 1 and rc(f, b, _10=None) == 1 and rc(f, b, _12=None) == 1 and rc(f, b, _17=None) == 1
    assert lib.sffn_residual_norm_bwd_workspace_bytes(0, 64, 5) == 0
    assert lib.sffn_residual_norm_bwd_workspace_bytes(10, 64, 0) < need


def test_launches_of_the_norm_backward():
    base = [None] * 29
    assert _lib._launches("sffn_residual_norm_bwd", base) == 1
    assert _lib._launches("sffn_residual_norm_bwd", base[:23] + [vp(16)] + base[24:]) == 2
    assert _lib._launches("sffn_residual_norm_bwd", base[:23] + [vp(0)] + base[24:]) == 1


def test_gate_groups():
    x = torch.empty(4, 6, 8)
    for shape, groups in (((8,), 1), ((1, 8), 1), ((3, 8), 3), ((4, 1, 8), 4), ((4, 6, 8), 24), ((1, 1, 8), 1)):
        assert norms._gate_groups(torch.empty(*shape), x) == groups


def test_a_thread_is_bound_once_and_to_no_other_device(monkeypatch):
    calls = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "set_device", calls.append)
    for index, want in ((0, []), (1, [torch.device("cuda", 1)])):
        monkeypatch.setattr(_lib, "_thread", threading.local())
        for _ in range(3):
            _lib.bind_thread(torch.device("cuda", index))
        assert calls == want
