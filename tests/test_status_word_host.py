"""CPU check of the status word when two threads ask for a device's first one at
once: there is one, which both get.  A second would leave the first thread's
kernels an address that the allocator gives away."""
import threading

import torch

from autoresearch2_b200 import _lib


def test_one_word_for_two_first_callers(monkeypatch):
    both = threading.Barrier(2)
    zeros = torch.zeros

    def made_at_once(*size, dtype=None, device=None):
        both.wait(timeout=30)
        return zeros(*size, dtype=dtype)

    monkeypatch.setattr(_lib, "_status", {})
    monkeypatch.setattr(torch, "zeros", made_at_once)
    got = [None, None]

    def ask(i):
        got[i] = _lib.status_word(torch.device("cuda", 0))

    threads = [threading.Thread(target=ask, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got[0] is not None and got[0] is got[1] is _lib._status[0]
    assert _lib.status_word(torch.device("cuda", 0)) is got[0]
