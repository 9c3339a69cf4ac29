"""CPU checks, with the C calls left out, that token_logprobs, distill_topk and
residual_norm refuse forward-mode tangents instead of dropping them, and that a
forward-mode level alone changes nothing."""
import pytest
import torch
from torch.autograd import forward_ad

import autoresearch2_b200 as sf
from autoresearch2_b200 import _lib, logits, norms


@pytest.fixture(autouse=True)
def on_the_host(monkeypatch):
    word = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "status_word", lambda device: word)
    for module in (logits, norms):
        monkeypatch.setattr(module, "call", lambda *a: 0)
        monkeypatch.setattr(module, "stream_handle", lambda device: 0)


X, T = torch.randn(3, 10), torch.zeros(3, dtype=torch.long)
IDS, SCORES = torch.zeros(3, 2, dtype=torch.long), torch.zeros(3, 2)
W = torch.ones(10)
CALLS = {
    "token_logprobs": lambda t: sf.token_logprobs(t, T, top_k=2),
    "token_logprobs without targets": lambda t: sf.token_logprobs(t),
    "distill_topk": lambda t: sf.distill_topk(t, IDS, SCORES),
    "distill_topk, scores": lambda t: sf.distill_topk(X, IDS, t[:, :2]),
    "residual_norm": lambda t: sf.residual_norm(t, X, post_norm=True),
    "residual_norm, y": lambda t: sf.residual_norm(X, t),
    "residual_norm, first": lambda t: sf.residual_norm(t),
    "residual_norm, weight": lambda t: sf.residual_norm(X, X, t[0]),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_refused(name, grad):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = forward_ad.make_dual(X, torch.ones_like(X))
        with pytest.raises(RuntimeError, match="forward.mode AD"):
            CALLS[name](dual)
        CALLS[name](X)


@pytest.mark.parametrize("name", CALLS)
def test_func_jvp_is_refused(name):
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: CALLS[name](t)[0], (X,), (torch.ones_like(X),))


def test_no_level_and_no_gradient_pass_autograd_by():
    assert not _lib.tracked(X, None)
    leaf = X.clone().requires_grad_()
    assert _lib.tracked(None, leaf)
    with torch.no_grad():
        assert not _lib.tracked(leaf)
