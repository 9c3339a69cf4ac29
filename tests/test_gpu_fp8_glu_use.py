"""GPU checks of the 8-bit blocks and the gated block as programs use them
together: a chain of all of them, traced by torch.compile, captured into CUDA
graphs, on other streams, threads and devices, within the GPT harness."""
import threading

import pytest
import torch

import autoresearch2_b200 as sf
from autoresearch2_b200 import gpt

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def randn(*shape, seed=0, scale=1.0, dtype=BF16, device=DEV):
    return (torch.randn(*shape, generator=torch.Generator(device=device).manual_seed(seed), device=device) * scale).to(dtype)


def chain_inputs(T=160, D=96, F=200, device=DEV):
    x = randn(2, T // 2, D, seed=1, device=device)
    return [x, randn(D, D, seed=2, scale=0.1, device=device), randn(F, D, seed=3, scale=0.1, device=device),
            randn(F, D, seed=4, scale=0.1, device=device), randn(D, F, seed=5, scale=0.1, device=device)]


def chain(x, W, Wg, Wu, W2, checkpoint="fp8"):
    """A norm, a projection and a gated block, their residual adds."""
    x, h = sf.residual_norm(x)
    x, h = sf.residual_norm(x, sf.ckpt_linear(h, W), post_norm=True)
    return sf.residual_norm(x, sf.gated_ffn(h, Wg, Wu, W2, checkpoint=checkpoint), post_norm=True)[1]


def grads_of(f, args, dy):
    leaves = [a.detach().requires_grad_() for a in args]
    y = f(*leaves)
    return y, torch.autograd.grad(y, leaves, dy)


def test_a_chain_of_them_against_torch():
    """float64 torch, bfloat16 inputs: output and gradients within the 2e-2 of the
    largest magnitude that the package's bfloat16 blocks are held to; all gradients but
    the projection's weight's, the one that 8 bits enter here."""
    args = chain_inputs()
    dy = randn(*args[0].shape, seed=9)
    y, got = grads_of(lambda *a: chain(*a, checkpoint=None), args, dy)

    def reference(x, W, Wg, Wu, W2):
        rms = lambda t: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
        x = x + rms(rms(x) @ W.T)
        h = rms(x)
        return rms(x + rms((torch.nn.functional.silu(h @ Wg.T) * (h @ Wu.T)) @ W2.T))

    want_y, want = grads_of(reference, [a.to(F64) for a in args], dy.to(F64))
    for i, (a, b) in enumerate(zip([y, *got], [want_y, *want])):
        assert i == 2 or (a.to(F64) - b).abs().max() <= 2e-2 * b.abs().max(), i
    sf.check_status()


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_compiled(checkpoint):
    args = chain_inputs()
    dy = randn(*args[0].shape, seed=9)
    want_y, want = grads_of(lambda *a: chain(*a, checkpoint=checkpoint), args, dy)
    torch._dynamo.reset()
    f = torch.compile(lambda *a: chain(*a, checkpoint=checkpoint), backend="aot_eager", fullgraph=True)
    y, got = grads_of(f, args, dy)
    assert torch.equal(y, want_y) and all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        w = sf.fp8_pack(args[2])
        g = torch.compile(lambda x, v, t: torch.ops.sparseffn.fp8_unpack(v, t, [200, 96], F16).sum()
                          + torch.ops.sparseffn.fp8_matmul(*torch.ops.sparseffn.fp8_pack(x), v, t, BF16).sum(),
                          backend="aot_eager", fullgraph=True)
        x = args[0]
        assert torch.equal(g(x, w.values, w.scale_tiles), w.to_dense(F16).sum() + sf.fp8_matmul(x, w).sum())
        f = torch.compile(lambda x, few: (sf.fp8_matmul(x, w), sf.fp8_matmul(few, w), sf.fp8_unpack(sf.fp8_pack(x), F32)),
                          backend="aot_eager", fullgraph=True)
        few = randn(3, 96, seed=3)
        for a, b in zip(f(x, few), (sf.fp8_matmul(x, w), sf.fp8_matmul(few, w), sf.fp8_pack(x).to_dense(F32))):
            assert torch.equal(a, b)
    torch._dynamo.reset()


def test_captured_and_replayed():
    """Forward and backward in a CUDA graph, replayed on other inputs; two captures,
    replayed in turn.  (No eager graph of the same leaves may live meanwhile: autograd
    would join the capture to that graph's stream, whatever the operators.)"""
    args = chain_inputs()
    leaves = [a.detach().requires_grad_() for a in args]
    dy = randn(*args[0].shape, seed=9)
    w8 = sf.fp8_pack(args[2])
    few, narrow = [randn(3, 96, seed=11), *args[2:]], [randn(40, 96, seed=12), *args[2:]]

    def step():
        y = chain(*leaves)
        with torch.no_grad():
            out = (sf.gated_ffn(*few), sf.fp8_matmul(leaves[0], w8), sf.fp8_matmul(few[0], w8), sf.gated_ffn(*narrow),
                   sf.fp8_matmul(narrow[0], w8))
        return [y.detach(), *torch.autograd.grad(y, leaves, dy), *out]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for seed in (21, 22, 23):
        with torch.no_grad():
            leaves[0].copy_(randn(*args[0].shape, seed=seed))
            dy.copy_(randn(*args[0].shape, seed=seed + 50))
            few[0].copy_(randn(3, 96, seed=seed + 90))
            narrow[0].copy_(randn(40, 96, seed=seed + 91))
        want = [t.clone() for t in step()]
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), seed
    sf.check_status()


@pytest.mark.parametrize("T", [1, 12, 40, 64, 90])
def test_operands_rewritten_between_calls(T):
    """Calls under way one behind the other, every operand written anew before each:
    kernels that start while the one before ends read none of it too early."""
    D, F, n = 520, 3000, 12
    sets = [[randn(*s, seed=10 * i + j, scale=0.05 if j else 1.0) for j, s in enumerate([(T, D), (F, D), (F, D), (D, F)])] for i in range(n)]
    live = [t.clone() for t in sets[0]]

    def calls():
        q = sf.fp8_pack(live[1])
        return sf.gated_ffn(*live), sf.fp8_matmul(live[0], q), sf.ckpt_linear(live[0], live[1])

    wanted, got = [], []
    for wait in (True, False):
        for s in sets:
            for a, b in zip(live, s):
                a.copy_(b)
            (wanted if wait else got).append(calls())
            if wait:
                torch.cuda.synchronize()
    for w, g in zip(wanted, got):
        assert all(torch.equal(a, b) for a, b in zip(w, g))
    sf.check_status()


def test_on_another_stream_than_the_tensors():
    args = chain_inputs(T=600)
    dy = randn(*args[0].shape, seed=9)
    want_y, want = grads_of(chain, args, dy)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late = [a + 0 for a in args]  # on the side stream, after the sleep
        late_dy = dy + 0
        y, got = grads_of(chain, late, late_dy)
    side.synchronize()
    assert torch.equal(y, want_y) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_threads_with_different_sizes_at_once():
    def of(T, D, F, checkpoint, seed):
        x, W, Wg, Wu, W2 = chain_inputs(T, D, F)
        x = (x + seed).requires_grad_()
        w8 = sf.fp8_pack(Wg)

        def call():
            y = sf.gated_ffn(x, Wg, Wu, W2, checkpoint=checkpoint)
            with torch.no_grad():
                return (y.detach(), *torch.autograd.grad(y, x, x.detach()), sf.fp8_matmul(x, w8), sf.gated_ffn(x[0, :9], Wg, Wu, W2),
                        sf.gated_ffn(x[0, :30], Wg, Wu, W2), sf.fp8_matmul(x[0, :30], w8))
        return call

    calls = [of(200, 64, 96, None, 0), of(900, 264, 520, "fp8", 1), of(64, 1000, 130, "fp8", 2)]
    wanted = [c() for c in calls]
    torch.cuda.synchronize()
    start, errors = threading.Barrier(3), []

    def work(call, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(150):
                    got = call()
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))
        except Exception as e:  # noqa: BLE001  (reported by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(calls, wanted)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    sf.check_status()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_another_device_than_the_current_one():
    args = chain_inputs()
    dy = randn(*args[0].shape, seed=9)
    want_y, want = grads_of(chain, args, dy)
    y, got = grads_of(chain, [a.to("cuda:1") for a in args], dy.to("cuda:1"))
    assert torch.equal(y.cpu(), want_y.cpu()) and all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, want))
    assert torch.cuda.current_device() == 0


def test_what_is_refused_of_differentiation():
    args = [a.requires_grad_() for a in chain_inputs()]
    x, W, Wg, Wu, W2 = args
    for name, y, leaf in (("ckpt_linear", sf.ckpt_linear(x, W), W), ("gated_ffn", sf.gated_ffn(x, Wg, Wu, W2), Wg)):
        with pytest.raises(RuntimeError, match=f"{name} is not differentiable again"):
            torch.autograd.grad(y.float().sum(), leaf, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), x.detach())
        for f in (lambda: sf.ckpt_linear(dual, W), lambda: sf.gated_ffn(dual, Wg, Wu, W2), lambda: sf.fp8_pack(dual),
                  lambda: sf.fp8_matmul(dual, sf.Fp8Tensor(*sf.fp8._pack(Wg.detach())))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f()
    y = sf.gated_ffn(x, Wg, Wu, W2)
    with torch.no_grad():
        Wg += 1  # autograd's version counter sees the change
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_one_leaf_used_twice():
    """Wg as both projections, x as output gradient: gradients add up."""
    x, W, Wg, Wu, W2 = chain_inputs()
    Wg.requires_grad_()
    g = torch.autograd.grad(sf.gated_ffn(x, Wg, Wg, W2), Wg, x)[0]
    a, b = Wg.detach().requires_grad_(), Wg.detach().clone().requires_grad_()
    ga, gb = torch.autograd.grad(sf.gated_ffn(x, a, b, W2), [a, b], x)
    assert torch.equal(g, ga + gb)


def test_weight_gradients_reach_an_attached_communicator():
    seen = []

    class Comm(sf.parallel.GradAllReduce):
        def submit(self, t):
            seen.append(tuple(t.shape))
            return t

    args = [a.requires_grad_() for a in chain_inputs()]
    with Comm().attached():
        torch.autograd.grad(sf.gated_ffn(args[0], *args[2:], checkpoint="fp8"), args[2:], args[0].detach())
        torch.autograd.grad(sf.ckpt_linear(args[0], args[1]), args[1], args[0].detach())
    assert seen == [(96, 200), (200, 96), (200, 96), (96, 96)]


# ---------------------------------------------------------------------------
# The GPT harness
# ---------------------------------------------------------------------------
CFG = gpt.GPTConfig(n_layer=2, n_head=4, n_embd=256, ffn_hidden=704, vocab=1024, seq_len=128, gated="silu")


def loss_and_grads(cfg, sparse, idx, tgt):
    m = gpt.GPT(cfg, sparse=sparse, device=DEV)
    loss = m(idx, tgt)
    loss.backward()
    return float(loss.detach()), {n: p.grad for n, p in m.named_parameters()}


@pytest.mark.parametrize("sandwich", [False, True])
def test_gpt_with_gated_mlps(sandwich):
    """The library's gated MLPs against torch's, as the harness' sparse MLPs are held
    to the dense ones: 2e-2 of a gradient's largest magnitude."""
    cfg = gpt.GPTConfig(**{**CFG.__dict__, "sandwich": sandwich})
    idx, tgt = gpt.synthetic_batch(cfg, 4, DEV)
    ls, gs = loss_and_grads(cfg, True, idx, tgt)
    ld, gd = loss_and_grads(cfg, False, idx, tgt)
    sf.check_status()
    assert abs(ls - ld) <= 2e-2 * abs(ld)
    for name, w in gd.items():
        assert (gs[name].float() - w.float()).abs().max() <= 2e-2 * w.float().abs().max(), name


def test_gpt_with_8_bit_checkpoints(monkeypatch):
    """Every weight's gradient is the operators' own for the inputs and output gradients
    that the model gave them, bit for bit (what those are worth: the operators'
    tests), and the loss is the one without checkpoints."""
    calls = []

    def recorded(f):
        def call(x, *rest):
            y = f(x, *rest)
            entry = [f, x.detach(), rest, None]
            y.register_hook(lambda dy: entry.__setitem__(3, dy))
            calls.append(entry)
            return y
        return call

    cfg8 = gpt.GPTConfig(**{**CFG.__dict__, "ckpt8": True})
    idx, tgt = gpt.synthetic_batch(cfg8, 4, DEV)
    plain = gpt.GPT(CFG, device=DEV)(idx, tgt)
    monkeypatch.setattr(gpt, "ckpt_linear", recorded(sf.ckpt_linear))
    monkeypatch.setattr(gpt, "gated_ffn", recorded(sf.gated_ffn))
    m = gpt.GPT(cfg8, device=DEV)
    loss = m(idx, tgt)
    loss.backward()
    assert abs(float(loss.detach()) - float(plain.detach())) <= 2e-2 * float(plain.detach()) and len(calls) == 3 * CFG.n_layer
    for f, x, rest, dy in calls:
        weights = [t for t in rest if isinstance(t, torch.Tensor)]
        kind = [t for t in rest if not isinstance(t, torch.Tensor)]
        assert kind == ([] if f is sf.ckpt_linear else ["silu", "fp8"])
        own = [w.detach().requires_grad_() for w in weights]
        for w, g in zip(weights, torch.autograd.grad(f(x, *own, *kind), own, dy)):
            assert torch.equal(w.grad, g)
    sf.check_status()


def test_gpt_training_steps_and_packed_weights():
    for gated in ("silu", None):
        cfg = gpt.GPTConfig(**{**CFG.__dict__, "gated": gated, "ckpt8": gated is not None})
        idx, tgt = gpt.synthetic_batch(cfg, 4, DEV, seed=1)
        m = gpt.GPT(cfg, sparse=True, device=DEV)
        step = gpt.TrainStep(m, idx, tgt, lr=1e-3)
        for _ in range(3):
            assert torch.isfinite(step())
        w8 = m.packed_weights()
        full, packed = m.score(idx, tgt), m.score(idx, tgt, weights=w8)
        assert packed.logp.shape == full.logp.shape and torch.isfinite(packed.logp).all()
        with torch.no_grad():
            logits, l8 = m(idx).float(), m(idx, weights=w8).float()
        # each product's factors are rounded by 2^-4 at most, at random: far below the
        # logits' own size
        assert (l8 - logits).norm() <= 0.25 * logits.norm()
    sf.check_status()


def test_train_gpt_command(capsys):
    from autoresearch2_b200 import train_gpt
    argv = ["--layers=1", "--width=128", "--heads=2", "--hidden=352", "--vocab=512", "--seq=64", "--batch=2", "--steps=2", "--warmup=1"]
    assert train_gpt.main([*argv, "--gated=silu", "--ckpt8"]) == 0
    out = capsys.readouterr().out
    assert '"mlp": "gated_silu"' in out and '"ckpt8": true' in out


def test_offsets_beyond_32_bits():
    """Matrices of 2.2e9 elements: their last rows are those of a small call's definition."""
    from test_gpu_fp8 import close_sum
    from test_gpu_glu import act, check_forward, half, s as sums
    T, D, F, n = 66000, 64, 33000, 8
    x, Wg, Wu, W2 = (randn(*s, seed=i, scale=s[-1] ** -0.5 if i else 1.0) for i, s in enumerate([(T, D), (F, D), (F, D), (D, F)]))
    xd, Wgd, Wud, W2d = (t.to(F64) for t in (x[-n:], Wg, Wu, W2))
    a, d = act(xd @ Wgd.T, "silu")
    dh = xd @ W2d
    mag = (dh * (xd @ Wud.T) * d).abs() @ Wgd.abs() + (dh * a).abs() @ Wud.abs()
    big = torch.zeros(T, F, device=DEV, dtype=BF16)
    big[-n:] = randn(n, F, seed=7)
    q, part = sf.fp8_pack(big), sf.fp8_pack(big[-n:].clone())
    assert torch.equal(q.values[-n:].view(torch.uint8), part.values.view(torch.uint8)) and torch.equal(q.exponents[-n:], part.exponents)
    big.fill_(1.0)
    assert torch.equal(sf.fp8_unpack(q)[-n:], part.to_dense())
    del big
    y = sf.fp8_matmul(q, sf.fp8_pack(W2), out_dtype=BF16)  # a long a
    close_sum(y[-n:], part.to_dense(F32).to(F64), sf.fp8_pack(W2).to_dense(F32).to(F64))
    assert (y[:-n] == 0).all()
    del q, y
    wide = sf.fp8_matmul(sf.fp8_pack(x), sf.fp8_pack(Wg))  # a long result
    close_sum(wide[-n:], sf.fp8_pack(x[-n:].clone()).to_dense(F32).to(F64), sf.fp8_pack(Wg).to_dense(F32).to(F64))
    del wide
    leaf = x.clone().requires_grad_()
    for checkpoint in (None, "fp8"):
        y = sf.gated_ffn(leaf, Wg, Wu, W2, checkpoint=checkpoint)
        check_forward(y.detach()[-n:], x[-n:], Wg, Wu, W2, "silu")
        dx = torch.autograd.grad(y, leaf, x)[0]
        few = x[-n:].clone().requires_grad_()
        y = sf.gated_ffn(few, Wg, Wu, W2, checkpoint=checkpoint)
        want = torch.autograd.grad(y, few, x[-n:].clone())[0]
        # dg and du are equal bit for bit, dx's sums in another order, each rounded once; the
        # magnitudes within 1 + 2^-4 of the kept factors
        tol = 2 * (half(BF16) * want.to(F64).abs() + sums(2 * F) * 1.25 * mag)
        assert ((dx[-n:].to(F64) - want.to(F64)).abs() <= tol).all()
    sf.check_status()
