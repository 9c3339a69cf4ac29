"""CPU checks of how the gated block's backward chooses between one product and two for
the weights' gradients: on request, never by the places of buffers that have
rows of something else between or behind them."""
import ctypes

import pytest
import torch

from autoresearch2_b200 import _lib, fp8, glu

vp = ctypes.c_void_p
JOINT, APART = 16, 32


@pytest.mark.parametrize("D", [8, 1001, 4096])
@pytest.mark.parametrize("F", [1, 37, 1357, 2048])
def test_launches(D, F):
    T, ld = 4096, (F + 7) // 8 * 8
    dwg = 1 << 20

    def down(steps, dwu):
        return _lib._launches("sffn_gated_ffn_bwd", [1, 2, 1, steps, 1, D, 1, D, 1, D, 1, D, 1, F, 0, 1, 1, 1, 1, 1, 1, T, D, F, 1, dwg, dwu, 1, 1, 0, 1, 0])

    two, one = 2 * _lib._gemm16(F, D, T), _lib._gemm16(2 * ld, D, T)
    right_behind = dwg + ld * D * 2
    assert down(4 | APART, right_behind) == two and down(4 | APART, dwg + 64) == two and down(4, dwg + 64) == two
    assert down(4 | JOINT, right_behind) == one
    assert down(4, right_behind) == (one if F % 8 == 0 else two)


def test_entry_refuses_a_joint_product_of_other_places():
    lib = _lib.load()
    F, D = 37, 64
    P = 1 << 20
    ok = [1, 2, 1, 15, P, 64, P, 64, P, 64, P, 64, P, 40, 0, P, P, None, None, None, None, 100, D, F, P, P, P + 40 * D * 2, P, P, 1 << 24, P, None]

    def rc(**change):
        a = list(ok)
        for k, v in change.items():
            a[int(k[1:])] = v
        return lib.sffn_gated_ffn_bwd(*[vp(v) if i in (4, 6, 8, 10, 12, 15, 16, 24, 25, 26, 27, 28, 30) else v for i, v in enumerate(a)])

    # (an output that is missing altogether is refused after this: 1 too, with no device call)
    assert rc(_3=15 | JOINT | APART) == 1 and rc(_3=15 | JOINT, _26=P + 37 * D * 2) == 1 and rc(_3=15 | JOINT, _26=None) == 1
    assert rc(_3=15 | JOINT, _25=None) == 1


def test_the_python_paths_say_which(monkeypatch):
    """The eager path asks for one product into one buffer, the op for two."""
    monkeypatch.setattr(_lib, "bind_thread", lambda dev: None)
    monkeypatch.setattr(_lib, "status_word", lambda dev: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(glu, "stream_handle", lambda dev: 0)
    seen = []
    monkeypatch.setattr(glu, "call", lambda name, *a: seen.append((a[3], a[25], a[26])))
    T, D, F = 5, 24, 37
    t = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    g = fp8._empty_rows(t(1, 1), T, F, 8)
    args = (t(T, D), t(T, D), t(F, D), t(F, D), t(D, F), g, g, None, None, None, None, 2)
    glu._backward(*args, [True] * 4)
    glu._backward(*args, [True] * 4, apart=True)
    glu._backward(*args, [True, True, False, True])
    assert seen[0][0] == 15 | JOINT and seen[0][2] == seen[0][1] + 40 * D * 2
    assert [s[0] for s in seen[1:]] == [15 | APART] * 2
