"""CPU checks of what the backward of the gated block and of ckpt_linear hands to
the library when saved-tensor hooks (save_on_cpu and the like) gave back copies
of what the forward kept, which are dense: the rows that the library's kernels
will read are those that were kept.  No kernel runs here: the C call is
replaced by one that looks at its arguments."""
import ctypes

import pytest
import torch

import autoresearch2_b200 as sf
from autoresearch2_b200 import _lib, fp8, glu

BF16, F16 = torch.bfloat16, torch.float16


def fill(*shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def values(rows, width, seed):
    """e4m3 rows as a forward keeps them: padded to 16 bytes."""
    out = fp8._empty_values(rows, width, "cpu")
    out.copy_(fill(rows, width, seed=seed).float().to(fp8.E4M3))
    return out


def tiles(rows, width, seed):
    t = fp8._empty_tiles(rows, width, "cpu")
    return t.copy_(torch.randint(100, 150, t.shape, generator=torch.Generator().manual_seed(seed)))


def moved(t):
    """A dense copy, as a hook returns one.  (In a larger buffer, so that what is read past
    its end here is memory of this test.)"""
    n = t.numel()
    buf = torch.zeros(2 * n + 4096, dtype=t.dtype)
    return buf[:n].view(t.shape).copy_(t)


def read(address, rows, width, ld, like):
    """[rows, width] at an address, rows ld elements apart."""
    es = like.element_size()
    raw = ctypes.string_at(address, ((rows - 1) * ld + width) * es)
    flat = torch.frombuffer(bytearray(raw), dtype=torch.uint8)
    return torch.stack([flat[r * ld * es:r * ld * es + width * es] for r in range(rows)])


def as_bytes(t):
    return t.contiguous().view(torch.uint8).view(t.shape[0], -1)


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(_lib, "require_cuda", lambda *ts: None)
    monkeypatch.setattr(_lib, "bind_thread", lambda dev: None)
    monkeypatch.setattr(_lib, "once_differentiable", lambda name: None)
    monkeypatch.setattr(_lib, "status_word", lambda dev: torch.zeros(1, dtype=torch.int32))
    for module in (fp8, glu):
        monkeypatch.setattr(module, "stream_handle", lambda dev: 0)
    return seen


def gated_step(monkeypatch, seen, T, D, F, dtype, keep, hook):
    """One step with a forward that keeps known tensors; the arguments of the C call go to
    `seen` together with what it would read.  Returns what was kept."""
    if keep == 1:
        kept = [fp8._empty_rows(fill(1, 1, seed=0, dtype=dtype), T, F, 8).copy_(fill(T, F, seed=s, dtype=dtype)) for s in (1, 2)] + [None] * 4
    else:
        kept = [values(T, F, 1), values(T, F, 2), tiles(T, F, 3), tiles(T, F, 4), values(T, D, 5), tiles(T, D, 6)]
    monkeypatch.setattr(glu, "_forward", lambda x, *a: (torch.zeros_like(x), *kept))

    def call(name, *a):
        assert name == "sffn_gated_ffn_bwd"
        up = lambda n, m: (n + m - 1) // m * m  # noqa: E731
        x, ldx, odd, (g, u, gt, ut, xv, xt) = a[6], a[7], a[14], a[15:21]
        got = []
        for p, w in ((g, F), (u, F)):
            assert p % 16 == 0
            got.append(read(p, T, w, up(w, 8 if keep == 1 else 16), kept[0]))
        if keep == 2:
            assert xv % 16 == 0
            got.append(read(xv, T, D, up(D, 16), kept[4]))
            got += [torch.frombuffer(bytearray(ctypes.string_at(p, t.numel())), dtype=torch.uint8).view(t.shape)
                    for p, t in ((gt, kept[2]), (ut, kept[3]), (xt, kept[5]))]
        else:
            assert (T == 1 or ldx % 8 == 0) and x % 16 == 0 or odd & 16
            got.append(read(x, T, D, ldx, fill(1, 1, seed=0, dtype=dtype)))
        seen.append(got)

    monkeypatch.setattr(glu, "call", call)
    ts = [fill(T, D, seed=10, dtype=dtype), fill(F, D, seed=11, dtype=dtype), fill(F, D, seed=12, dtype=dtype), fill(D, F, seed=13, dtype=dtype)]
    leaves = [t.requires_grad_() for t in ts]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook):
        y = glu._GatedFFN.apply(*leaves, 2, keep)
    y.backward(fill(T, D, seed=14, dtype=dtype))
    return kept, ts[0].detach()


@pytest.mark.parametrize("hook", [moved, lambda t: t], ids=["moved", "kept"])
@pytest.mark.parametrize("keep", [1, 2])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,D,F", [(7, 21, 37), (1, 21, 37), (5, 32, 48), (9, 1, 1), (130, 24, 520)])
def test_gated_ffn_reads_what_was_kept(monkeypatch, calls, T, D, F, dtype, keep, hook):
    (kept, x) = gated_step(monkeypatch, calls, T, D, F, dtype, keep, hook)
    (got,) = calls
    want = [as_bytes(kept[0]), as_bytes(kept[1])]
    want += [as_bytes(kept[4]), kept[2], kept[3], kept[5]] if keep == 2 else [as_bytes(x)]
    assert len(got) == len(want)
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i


@pytest.mark.parametrize("keep", [1, 2])
def test_gated_ffn_refuses_what_was_not_kept(monkeypatch, calls, keep):
    """A hook that returns another type, shape or device."""
    def other_type(t):
        return t.float() if t.dtype in (BF16, fp8.E4M3) else t.int()

    for bad in (other_type, lambda t: t[:-1], lambda t: t.to("meta")):
        with pytest.raises((TypeError, ValueError)):
            gated_step(monkeypatch, calls, 7, 21, 37, BF16, keep, bad)
    for i in range(4 if keep == 1 else 9):  # each one alone
        count = [0]

        def one(t):
            count[0] += 1
            return t[:-1] if count[0] == i + 1 else t

        with pytest.raises((TypeError, ValueError)):
            gated_step(monkeypatch, calls, 7, 21, 37, BF16, keep, one)
    assert not calls


def linear_step(monkeypatch, seen, T, K, N, dtype, hook):
    kept = [values(T, K, 1), tiles(T, K, 2)]
    monkeypatch.setattr(fp8, "_linear_forward", lambda x, W, keep: (torch.zeros(T, N, dtype=dtype), *kept))

    def call(name, *a):
        assert name == "sffn_ckpt_linear_bwd"
        W, ldw, v, ldv, t = a[3], a[4], a[6], a[7], a[8]
        assert v % 16 == 0 and ldv % 16 == 0
        seen.append([read(v, T, K, ldv, kept[0]), torch.frombuffer(bytearray(ctypes.string_at(t, kept[1].numel())), dtype=torch.uint8).view(kept[1].shape),
                     read(W, N, K, ldw, fill(1, 1, seed=0, dtype=dtype))])

    monkeypatch.setattr(fp8, "call", call)
    x, W = (fill(*s, seed=i, dtype=dtype).requires_grad_() for i, s in enumerate([(T, K), (N, K)]))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook):
        y = fp8._CkptLinear.apply(x, W)
    y.backward(fill(T, N, seed=14, dtype=dtype))
    return as_bytes(kept[0]), kept[1], as_bytes(W.detach())


@pytest.mark.parametrize("hook", [moved, lambda t: t], ids=["moved", "kept"])
@pytest.mark.parametrize("T,K,N", [(7, 21, 37), (1, 21, 37), (5, 32, 48), (9, 1, 1), (130, 1001, 5)])
def test_ckpt_linear_reads_what_was_kept(monkeypatch, calls, T, K, N, hook):
    want = linear_step(monkeypatch, calls, T, K, N, F16, hook)
    (got,) = calls
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_ckpt_linear_refuses_what_was_not_kept(monkeypatch, calls):
    for bad in (lambda t: t.float(), lambda t: t[:-1], lambda t: t.to("meta")):
        for i in range(3):
            count = [0]

            def one(t):
                count[0] += 1
                return bad(t) if count[0] == i + 1 else t

            with pytest.raises((TypeError, ValueError)):
                linear_step(monkeypatch, calls, 7, 21, 37, BF16, one)
    assert not calls
