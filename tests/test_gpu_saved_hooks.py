"""GPU checks of the gated block and ckpt_linear under saved-tensor hooks: what
is moved away between forward and backward (save_on_cpu) or copied comes back
dense, and the gradients are those of the plain call, bit for bit."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

import autoresearch2_b200 as sf
from autoresearch2_b200 import glu

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16
HOOKS = {"save_on_cpu": lambda: save_on_cpu(), "save_on_cpu pinned": lambda: save_on_cpu(pin_memory=True),
         "clone": lambda: saved_tensors_hooks(lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format)),
         "other strides": lambda: saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone())}


def randn(*shape, seed=0, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * scale).to(dtype)


def gated_inputs(T, D, F, dtype):
    shapes = [(T, D), (F, D), (F, D), (D, F)]
    return [randn(*s, seed=i, scale=s[1] ** -0.5 if i else 1.0, dtype=dtype).requires_grad_() for i, s in enumerate(shapes)], \
        randn(T, D, seed=9, dtype=dtype)


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,D,F", [(777, 1001, 1357), (130, 96, 200), (1, 21, 37), (65, 1, 1)])
def test_gated_ffn(T, D, F, dtype, checkpoint, hook):
    leaves, dy = gated_inputs(T, D, F, dtype)
    want = torch.autograd.grad(sf.gated_ffn(*leaves, checkpoint=checkpoint), leaves, dy)
    with HOOKS[hook]():
        y = sf.gated_ffn(*leaves, checkpoint=checkpoint)
    got = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sf.check_status()


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_gated_ffn_op(checkpoint):
    """The torch.library op's own autograd formula."""
    leaves, dy = gated_inputs(77, 101, 137, BF16)
    want = torch.autograd.grad(sf.gated_ffn(*leaves, checkpoint=checkpoint), leaves, dy)
    with HOOKS["clone"]():
        y = torch.ops.sparseffn.gated_ffn(*leaves, glu.ACTIVATIONS["silu"], glu.KEEP[checkpoint])[0]
    got = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sf.check_status()


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("hook", ["save_on_cpu", "clone"])
def test_compiled(checkpoint, hook):
    leaves, _ = gated_inputs(77, 101, 137, BF16)
    leaves.append(randn(37, 101, seed=5).requires_grad_())
    dy = randn(77, 37, seed=9)

    def f(x, Wg, Wu, W2, W):
        return sf.ckpt_linear(sf.gated_ffn(x, Wg, Wu, W2, checkpoint=checkpoint), W)

    want = torch.autograd.grad(f(*leaves), leaves, dy)
    torch._dynamo.reset()
    compiled = torch.compile(f, backend="aot_eager", fullgraph=True)
    with HOOKS[hook]():
        y = compiled(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))
    torch._dynamo.reset()
    sf.check_status()


def test_activation_checkpointing():
    """torch.utils.checkpoint recomputes the forward; twice through the same graph."""
    from torch.utils.checkpoint import checkpoint
    leaves, dy = gated_inputs(77, 101, 137, BF16)
    want = torch.autograd.grad(sf.gated_ffn(*leaves, checkpoint="fp8"), leaves, dy)
    y = checkpoint(lambda *a: sf.gated_ffn(*a, checkpoint="fp8"), *leaves, use_reentrant=False)
    for _ in range(2):
        got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    sf.check_status()


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_what_a_hook_must_not_return(checkpoint):
    leaves, dy = gated_inputs(77, 101, 137, BF16)
    for bad in (lambda t: t[:-1], lambda t: t.float(), lambda t: t.cpu()):
        with saved_tensors_hooks(lambda t: t, bad):
            y = sf.gated_ffn(*leaves, checkpoint=checkpoint)
        with pytest.raises((TypeError, ValueError)):
            torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,N", [(1499, 1001, 515), (130, 96, 200), (1, 21, 37), (65, 1, 1)])
def test_ckpt_linear(T, K, N, dtype, hook):
    x, W = randn(T, K, seed=1, dtype=dtype).requires_grad_(), randn(N, K, seed=2, scale=K ** -0.5, dtype=dtype).requires_grad_()
    dy = randn(T, N, seed=3, dtype=dtype)
    want = torch.autograd.grad(sf.ckpt_linear(x, W), [x, W], dy)
    ys = []
    with HOOKS[hook]():
        ys += [sf.ckpt_linear(x, W), torch.ops.sparseffn.ckpt_linear(x, W, True)[0], sf.ckpt_linear(x, W.detach())]
    for y in ys[:2]:
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, [x, W], dy), want))
    assert torch.equal(torch.autograd.grad(ys[2], x, dy)[0], want[0])
    sf.check_status()


def test_what_a_hook_must_not_return_to_ckpt_linear():
    x, W, dy = randn(77, 101).requires_grad_(), randn(37, 101, seed=1).requires_grad_(), randn(77, 37, seed=2)
    for bad in (lambda t: t[:-1], lambda t: t.float(), lambda t: t.cpu()):
        with saved_tensors_hooks(lambda t: t, bad):
            y = sf.ckpt_linear(x, W)
        with pytest.raises((TypeError, ValueError)):
            torch.autograd.grad(y, [x, W], dy)
