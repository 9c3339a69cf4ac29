"""CPU checks of what the backward ops refuse of the forward's statistics: a
tensor of another device or type never reaches a kernel."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from autoresearch2_b200 import logits, norms

F32 = torch.float32


def test_norm_backward_refuses_foreign_statistics():
    with FakeTensorMode():
        x = torch.empty(6, 64, device="cuda")
        ok = torch.empty(6, 2, device="cuda")
        norms._check_backward(x, x, x, x, ok, F32)
        for stats in (torch.empty(6, 2), torch.empty(6, 2, device="meta"), ok.double(), torch.empty(6, 3, device="cuda"),
                      torch.empty(2, 6, device="cuda").t()):
            with pytest.raises(ValueError, match="stats are the forward's"):
                norms._check_backward(x, x, x, x, stats, F32)


def test_logits_backwards_refuse_foreign_statistics():
    with FakeTensorMode():
        ok = torch.empty(6, 4, device="cuda")
        logits._check_kept("stats", ok, (6, 4), ok.device)
        for stats in (torch.empty(6, 4), ok.half(), torch.empty(6, 2, device="cuda")):
            with pytest.raises(ValueError, match="stats must be"):
                logits._check_kept("stats", stats, (6, 4), ok.device)
