"""CPU check of the GPT harness without blocks (its embeddings alone)."""
import pytest
import torch

from autoresearch2_b200 import gpt


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("gated", [None, "silu"])
def test_a_model_of_no_layers(sparse, gated):
    cfg = gpt.GPTConfig(n_layer=0, n_head=2, n_embd=32, ffn_hidden=64, vocab=64, seq_len=8, gated=gated)
    m = gpt.GPT(cfg, sparse=sparse, device="cpu", dtype=torch.float32)
    idx = torch.zeros(2, 8, dtype=torch.long)
    m(idx, idx).backward()
    assert m(idx).shape == (2, 8, 64) and m.wte.grad.any()
    with torch.no_grad():
        assert torch.equal(m(idx, weights=m.packed_weights()), m(idx))
