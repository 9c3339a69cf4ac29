"""GPU checks of what a target outside the vocabulary does to gradients: its log
probability is NaN and has none; the row's entropy and alternatives keep theirs;
a training step goes on with finite gradients and the status word set."""
import pytest
import torch

import autoresearch2_b200 as sf
from autoresearch2_b200 import _lib, gpt

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bad", [50, -1, 2 ** 40])
def test_the_rest_of_the_row_keeps_its_gradient(bad):
    x = torch.randn(4, 50, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).requires_grad_()
    t = torch.tensor([3, bad, 4, 5], device=DEV)
    r = sf.token_logprobs(x, t, top_k=3)
    g, = torch.autograd.grad(r.logp.sum() + 2 * r.entropy.sum() + r.top_logp.sum(), x)
    alone = sf.token_logprobs(x, None, top_k=3)
    want, = torch.autograd.grad(2 * alone.entropy.sum() + alone.top_logp.sum(), x)
    assert torch.equal(g[1], want[1]) and bool(g.isfinite().all())
    with pytest.raises(_lib.SparseFFNError, match="outside the vocabulary"):
        sf.check_status()


def test_a_step_with_a_bad_target():
    cfg = gpt.GPTConfig(n_layer=1, n_head=2, n_embd=64, ffn_hidden=256, vocab=128, seq_len=16)
    student, teacher = (gpt.GPT(cfg, sparse=False, device=DEV, seed=s) for s in (0, 1))
    idx, tgt = gpt.synthetic_batch(cfg, 2, DEV)
    tgt[0, 3] = 128
    step = gpt.DistillStep(student, teacher, idx, tgt, top_k=8, hard_weight=0.5)
    loss = step.loss()
    loss.backward()
    assert bool(loss.detach().isnan()) and all(bool(p.grad.isfinite().all()) for p in student.parameters())
    with pytest.raises(_lib.SparseFFNError, match="outside the vocabulary"):
        sf.check_status()
