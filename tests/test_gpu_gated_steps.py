"""GPU checks of the gated block's backward as it is made of steps: the weights'
gradients as one product or two, wherever their buffers lie."""
import pytest
import torch

import autoresearch2_b200 as sf
from autoresearch2_b200 import _lib, glu

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16


def randn(*shape, seed=0, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * scale).to(dtype)


def inputs(T, D, F, dtype=BF16):
    return [randn(*s, seed=i, scale=s[1] ** -0.5 if i else 1.0, dtype=dtype) for i, s in enumerate([(T, D), (F, D), (F, D), (D, F)])], \
        randn(T, D, seed=9, dtype=dtype)


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("T,D,F", [(300, 96, 37), (777, 1001, 1357), (130, 64, 200)])
def test_buffers_that_lie_as_for_one_product(monkeypatch, T, D, F, checkpoint):
    """Two gradients at the distance of the joint buffer, other data between and behind
    them: it stays as it is, and the gradients are those of the op, which
    computes them apart."""
    (x, Wg, Wu, W2), dy = inputs(T, D, F)
    keep = glu.KEEP[checkpoint]
    with torch.no_grad():
        _, *kept = glu._forward(x, Wg, Wu, W2, 2, keep)
        kept_x = x if keep == 1 else None
        want = glu._backward(dy, kept_x, Wg, Wu, W2, *kept, 2, [True] * 4, apart=True)
        ld = (F + 7) // 8 * 8
        buf = torch.full((2 * ld + 32, D), 77.0, device=DEV, dtype=BF16)
        dWg, dWu = buf[:F], buf[ld:ld + F]

        def call(name, *a):
            a = list(a)
            for flags in (0, glu.APART):
                a[3] = a[3] & 15 | flags
                a[25], a[26] = dWg.data_ptr(), dWu.data_ptr()
                buf.fill_(77.0)
                _lib.call(name, *a)
                assert (buf[F:ld] == 77).all() and (buf[ld + F:] == 77).all()
                if flags or F % 8:  # as two products
                    assert torch.equal(dWg, want[1]) and torch.equal(dWu, want[2])

        monkeypatch.setattr(glu, "call", call)
        glu._backward(dy, kept_x, Wg, Wu, W2, *kept, 2, [True] * 4, apart=True)
    sf.check_status()


class Comm(sf.parallel.GradAllReduce):
    """Keeps a copy of each gradient as it is when it is submitted."""

    def __init__(self):
        super().__init__()
        self.seen = []

    def submit(self, t):
        self.seen.append((t, t.clone()))
        return t


def with_and_without_a_communicator(f, leaves, dy):
    want = torch.autograd.grad(f(*leaves), leaves, dy)
    comm = Comm()
    with comm.attached():
        got = torch.autograd.grad(f(*leaves), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    return got, comm.seen


SIZES = [(160, 96, 200), (777, 1001, 1357), (40, 64, 37), (1, 21, 8), (33, 101, 96)]


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,D,F", SIZES)
def test_gated_ffn_with_a_communicator(T, D, F, dtype, checkpoint):
    """Step by step instead of in one call, all gradients wanted: the same ones, each final
    when it is handed on (dW2 first, then dWg and dWu)."""
    leaves, dy = inputs(T, D, F, dtype)
    leaves = [t.requires_grad_() for t in leaves]
    got, seen = with_and_without_a_communicator(lambda *a: sf.gated_ffn(*a, checkpoint=checkpoint), leaves, dy)
    assert [t.data_ptr() for t, _ in seen] == [got[i].data_ptr() for i in (3, 1, 2)]
    for (t, then), i in zip(seen, (3, 1, 2)):
        assert torch.equal(then, got[i])
    sf.check_status()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,N", SIZES)
def test_ckpt_linear_with_a_communicator(T, K, N, dtype):
    leaves = [randn(T, K, seed=1, dtype=dtype).requires_grad_(), randn(N, K, seed=2, scale=K ** -0.5, dtype=dtype).requires_grad_()]
    got, seen = with_and_without_a_communicator(sf.ckpt_linear, leaves, randn(T, N, seed=3, dtype=dtype))
    ((t, then),) = seen
    assert t.data_ptr() == got[1].data_ptr() and torch.equal(then, got[1])
    sf.check_status()
