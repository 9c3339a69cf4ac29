"""GPU checks of two host threads that call the same operator with different
sizes at once: a launch's shared memory limit belongs to the kernel and device,
so one call must not take from the other what it needs."""
import threading

import pytest
import torch

import autoresearch2_b200 as sf
from autoresearch2_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def randn(*shape, seed=0, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def at_once(calls, times):
    """Each call in a thread of its own, `times` times; its outputs must stay those of the first time."""
    wanted = [call() for call in calls]
    torch.cuda.synchronize()
    start, errors = threading.Barrier(len(calls)), []

    def work(call, want):
        try:
            start.wait()
            for _ in range(times):
                got = call()
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        except Exception as e:  # noqa: BLE001  (reported by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(calls, wanted)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


def test_norms_of_two_sizes():
    def of(rows, D, seed):
        x, y = randn(rows, D, seed=seed).requires_grad_(), randn(rows, D, seed=seed + 1)
        up = randn(rows, D, seed=seed + 2)

        def call():
            a, h = sf.residual_norm(x, y, post_norm=True)
            return a, h, *torch.autograd.grad([a, h], x, [up, up])
        return call

    at_once([of(8000, 768, 1), of(600, 768, 4), of(3000, 1536, 7)], 400)


def test_lists_of_two_vocabularies():
    base = randn(1200, 400000, seed=1)
    ids = torch.randint(0, 300000, (1200, 4), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    scores = torch.full((1200, 4), -2.0, device=DEV)

    def of(V):
        return lambda: (sf.distill_topk(base[:, :V], ids, scores, tail="bucket"),)

    at_once([of(400000), of(300000)], 300)


def launched_at_once(calls, times):
    """Each call of a C entry in a thread of its own, which does nothing else: no return code but 0."""
    start, codes = threading.Barrier(len(calls)), [[] for _ in calls]

    def work(call, mine):
        start.wait()
        for _ in range(times):
            rc = call()
            if rc:
                mine.append(rc)

    threads = [threading.Thread(target=work, args=a) for a in zip(calls, codes)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not any(codes), [(len(c), c[:1]) for c in codes]


def test_entry_of_the_norm_from_two_threads():
    """Few rows of 4096 columns take 192 KB of shared memory, of 768 columns 36 KB, in one kernel."""
    lib, status = _lib.load(), _lib.status_word(torch.device(DEV, torch.cuda.current_device()))

    def of(D):
        x, y, a, h = (randn(4, D, seed=i) for i in range(4))
        return lambda: lib.sffn_residual_norm(x.data_ptr(), 1, D, y.data_ptr(), 1, D, 4, D, None, 0, None, 0, None, 0,
                                              1, 0, 1.0, 1e-6, a.data_ptr(), h.data_ptr(), None, status.data_ptr(), None)

    launched_at_once([of(4096), of(768)], 40000)


def test_entry_of_the_lists_from_two_threads():
    """The bit lists of 400000 classes take 55 KB, of 300000 40 KB.  Lists without
    entries: the kernel ends before it reads a logit."""
    lib, status = _lib.load(), _lib.status_word(torch.device(DEV, torch.cuda.current_device()))
    rows, most = 600, 400000
    x = torch.zeros(rows, most, device=DEV, dtype=BF16)
    ids = torch.full((rows, 1), -1, device=DEV)
    scores, loss = torch.zeros(rows, 1, device=DEV), torch.empty(rows, device=DEV)

    def of(V):
        return lambda: lib.sffn_distill_topk(x.data_ptr(), 1, rows, V, rows, 0, most, ids.data_ptr(), 8,
                                             scores.data_ptr(), 0, 1, 1, 1.0, loss.data_ptr(), None, status.data_ptr(),
                                             None)

    launched_at_once([of(most), of(300000)], 40000)
