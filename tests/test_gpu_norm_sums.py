"""GPU checks of residual_norm's weight gradients where only the sums over rows
can err.

Rows of +-1 at a width that is a power of two have the mean square one, and an eps
of 2^-126 leaves it: xh is x itself, and each term dh xh of dpre a whole number.  A
block's sums stay below 2^24, where float32 is exact; the sum over all blocks does
not.  It is taken in 64 bits and rounded once, so dpre has to be the float32 next to
the whole number."""
import pytest
import torch

import autoresearch2_b200 as sf

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32 = torch.float32


@pytest.mark.parametrize("rows,D,most", [(30000, 1024, 1 << 15), (5000, 256, 1 << 16), (2500, 8192, 1 << 18), (20000, 64, 1 << 14)])
def test_sums_over_the_blocks_are_rounded_once(rows, D, most):
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.ones(rows, D, device=DEV)
    dh = torch.randint(0, most, (rows, D), generator=g, device=DEV)
    pre = torch.ones(D, device=DEV, requires_grad=True)
    stats = torch.ops.sparseffn.residual_norm(x, None, pre, None, None, 1, False, 1.0, 2.0 ** -126, F32)[2]
    assert bool((stats[:, 1] == 1).all())
    _, h = sf.residual_norm(x, pre_weight=pre, eps=2.0 ** -126)
    got, = torch.autograd.grad(h, pre, dh.to(F32))
    total = dh.sum(0)
    assert int(total.min()) > 1 << 24
    assert torch.equal(got, total.to(F32))


def test_gate_rows_and_post_weight_too():
    """One gate row for each of three runs of rows: dgate and dpost join other blocks."""
    rows, D = 30000, 1024
    g = torch.Generator(device=DEV).manual_seed(1)
    x, y = torch.zeros(rows, D, device=DEV), torch.ones(rows, D, device=DEV)
    up = torch.randint(0, 1 << 14, (rows, D), generator=g, device=DEV)
    post, gate = torch.ones(D, device=DEV, requires_grad=True), torch.ones(3, D, device=DEV, requires_grad=True)
    a, _ = sf.residual_norm(x, y, None, post, gate, True, eps=2.0 ** -126)
    dpost, dgate = torch.autograd.grad(a, [post, gate], up.to(F32))
    assert torch.equal(dpost, up.sum(0).to(F32))
    assert torch.equal(dgate, up.view(3, -1, D).sum(1).to(F32))
