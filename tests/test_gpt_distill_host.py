"""CPU checks of the GPT harness's options: the sandwich blocks and the
distillation step run on the CUDA library alone and say so, and the default
configuration has neither's parameters."""
import pytest
import torch

from autoresearch2_b200 import gpt

SMALL = dict(n_layer=2, n_head=4, n_embd=64, ffn_hidden=256, vocab=128, seq_len=16)


def model(**kw):
    return gpt.GPT(gpt.GPTConfig(**SMALL, **kw), sparse=False, device="cpu", dtype=torch.float32)


def test_sandwich_parameters():
    plain, sandwich = model(), model(sandwich=True)
    names = {n for n, _ in sandwich.named_parameters()} - {n for n, _ in plain.named_parameters()}
    assert len(names) == 2 * 6 + 1 and all(p.dtype == torch.float32 for p in sandwich.parameters())
    assert torch.equal(sandwich.blocks[0].mlp_gate, torch.full((64,), 0.5)) and bool((sandwich.norm_out == 1).all())
    assert not any("gate" in n for n, _ in plain.named_parameters())


def test_options_need_cuda():
    idx, tgt = gpt.synthetic_batch(gpt.GPTConfig(**SMALL), 2, "cpu")
    with pytest.raises(ValueError, match="CUDA tensors only"):
        model(sandwich=True)(idx, tgt)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        model().score(idx, tgt)


def test_hard_weight_needs_targets():
    with pytest.raises(ValueError, match="hard_weight"):
        gpt.DistillStep(model(), model(), None, None, hard_weight=0.5)
