"""GPU checks of the GPT harness on token_logprobs, distill_topk and
residual_norm together: the sandwich model and its distillation loss against
the same model written out in float64 torch operations (logits, loss and every
gradient), scoring, the training steps and the command.

Tolerance of the float32 models (2-norm of the difference over the result's): a
stage (a product over at most 1024 terms, a norm, a softmax) is within 192 u of
its operands' magnitude, u = 2^-24, and a loss and its gradient pass about 40 of
them in each of the two layers, 2 x 40 x 192 u < 1e-3."""
import json
import math

import pytest
import torch
import torch.nn.functional as F

import autoresearch2_b200 as sf
from autoresearch2_b200 import gpt, train_gpt

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 1e-3
CFG = gpt.GPTConfig(n_layer=2, n_head=4, n_embd=192, ffn_hidden=640, vocab=997, seq_len=65, sandwich=True)


def plain_logits(w, cfg, idx):
    """The sandwich model's logits in torch operations, for weights w by name."""
    def rms(t):
        return t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()

    B, T = idx.shape
    d, nh = cfg.n_embd, cfg.n_head
    x = w["wte"][idx] + w["wpe"][:T]
    mask = torch.ones(T, T, dtype=torch.bool, device=idx.device).tril()
    for i in range(cfg.n_layer):
        p = {k[len(f"blocks.{i}."):]: v for k, v in w.items() if k.startswith(f"blocks.{i}.")}
        q, k, v = (t.view(B, T, nh, d // nh).transpose(1, 2) for t in ((rms(x) * p["attn_pre"]) @ p["qkv"].T).split(d, -1))
        a = (q @ k.transpose(-1, -2) / math.sqrt(d // nh)).masked_fill(~mask, -math.inf).softmax(-1) @ v
        y = a.transpose(1, 2).reshape(B, T, d) @ p["proj"].T
        x = x + p["attn_gate"] * rms(y) * p["attn_post"]
        y = torch.relu((rms(x) * p["mlp_pre"]) @ p["W1"].T).square() @ p["W2"].T
        x = x + p["mlp_gate"] * rms(y) * p["mlp_post"]
    return (rms(x) * w["norm_out"]) @ w["wte"].T


def weights64(model):
    return {n: p.detach().double().requires_grad_() for n, p in model.named_parameters()}


def jitter(model, seed):
    """Norm weights and gates off their initial ones."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if p.dim() == 1:
                p.add_(torch.randn(p.shape, generator=g, device=DEV) * 0.1)
    return model


def close(got, want, what):
    off = (got.double() - want).norm() / want.norm()
    assert float(off) <= TOL, (what, float(off))


def models():
    teacher = jitter(gpt.GPT(CFG, sparse=False, device=DEV, dtype=torch.float32, seed=1), 1).requires_grad_(False)
    student = jitter(gpt.GPT(CFG, sparse=False, device=DEV, dtype=torch.float32, seed=2), 2)
    with torch.no_grad():  # logits apart from one another
        teacher.wte.mul_(8)
        student.wte.mul_(6)
    idx, tgt = gpt.synthetic_batch(CFG, 3, DEV)
    tgt[0, :20] = -100
    return teacher, student, idx, tgt


def test_sandwich_model_against_its_definition():
    _, model, idx, tgt = models()
    w = weights64(model)
    want = plain_logits(w, CFG, idx)
    close(model(idx), want, "logits")
    loss = F.cross_entropy(want.view(-1, CFG.vocab), tgt.view(-1))
    grads = torch.autograd.grad(loss, list(w.values()))
    got = model(idx, tgt)
    close(got, loss, "loss")
    got.backward()
    for (n, p), g in zip(model.named_parameters(), grads):
        close(p.grad, g, n)


@pytest.mark.parametrize("tail,T,hard", [("bucket", 1.0, 0.0), ("renorm", 2.0, 0.5)])
def test_distillation_from_the_teachers_list(tail, T, hard):
    """Teacher forward, its list, student forward, loss and backward, as a training step runs them."""
    teacher, student, idx, tgt = models()
    K = 20
    step = gpt.DistillStep(student, teacher, idx, tgt, top_k=K, temperature=T, tail=tail, hard_weight=hard)
    got = step.loss()
    got.backward()
    listed = teacher.score(idx, tgt, top_k=K, temperature=T)  # the list itself is checked below
    w = weights64(student)
    z = plain_logits(w, CFG, idx)
    lp = torch.log_softmax(z / T, -1)
    live = tgt != -100
    ids, c = listed.top_ids[live], listed.top_logp[live].double()
    lp_live = lp[live]
    if tail == "renorm":
        c = torch.log_softmax(c, -1)
    q = c.exp()
    loss = (q * (c - lp_live.gather(-1, ids))).sum(-1)
    if tail == "bucket":
        rest = 1 - q.sum(-1)
        off = torch.log1p(-lp_live.exp().gather(-1, ids).sum(-1))
        loss = loss + rest * (rest.log() - off)
    loss = loss.sum() * T * T / live.sum()
    if hard:
        loss = loss + hard * F.cross_entropy(z.view(-1, CFG.vocab), tgt.view(-1))
    close(got, loss, "loss")
    for (n, p), g in zip(student.named_parameters(), torch.autograd.grad(loss, list(w.values()))):
        close(p.grad, g, n)
    before = [p.detach().clone() for p in student.parameters()]
    student.zero_grad(set_to_none=True)
    step()
    assert all(not torch.equal(p, b) for p, b in zip(student.parameters(), before))
    sf.check_status()


def test_score_is_of_the_models_logits():
    teacher, _, idx, tgt = models()
    r = teacher.score(idx, tgt, top_k=7, temperature=1.5)
    z = teacher(idx)
    lp = torch.log_softmax(z.double() / 1.5, -1)
    live = tgt != -100
    assert torch.equal(r.top_ids[live], torch.sort(z.float(), dim=-1, descending=True, stable=True)[1][..., :7][live])
    want = lp.gather(-1, tgt.clamp_min(0)[..., None])[..., 0]
    assert float((r.logp.double() - want)[live].abs().max()) <= 2 ** -24 * (64 + 150 + 4 * float(want.abs().max()))
    assert bool((r.logp[~live] == 0).all()) and not r.logp.requires_grad


@pytest.mark.parametrize("sandwich", [False, True])
def test_sparse_student_of_a_dense_teacher(sandwich):
    """bf16, the MLPs sparse over their arena: the student's logits match the dense
    MLPs' within the bf16 tolerance, and a step leaves the status word clear."""
    cfg = gpt.GPTConfig(n_layer=2, n_head=4, n_embd=256, ffn_hidden=1024, vocab=1024, seq_len=128, sandwich=sandwich)
    teacher = gpt.GPT(cfg, sparse=False, device=DEV, seed=1).requires_grad_(False)
    sparse, dense = (gpt.GPT(cfg, sparse=s, device=DEV, fill=1.0, seed=2) for s in (True, False))
    idx, tgt = gpt.synthetic_batch(cfg, 4, DEV)
    steps = [gpt.DistillStep(m, teacher, idx, tgt, top_k=16, hard_weight=0.1) for m in (sparse, dense)]
    losses = [s.loss() for s in steps]
    assert abs(float(losses[0]) - float(losses[1])) <= 2e-2 * abs(float(losses[1]))
    for loss in losses:
        loss.backward()
    for (n, p), q in zip(sparse.named_parameters(), dense.parameters()):
        err = (p.grad.float() - q.grad.float()).abs().max()
        assert float(err) <= 2e-2 * float(q.grad.float().abs().max()), n
    for s in steps:
        s()
    sf.check_status()


def test_default_model_is_the_one_without_options():
    """No parameter, and not a bit of the loss or a gradient, differs from the blocks written out."""
    cfg = gpt.GPTConfig(n_layer=2, n_head=4, n_embd=128, ffn_hidden=512, vocab=512, seq_len=64)
    m = gpt.GPT(cfg, sparse=False, device=DEV)
    assert {n.split(".")[-1] for n, _ in m.named_parameters()} == {"wte", "wpe", "qkv", "proj", "W1", "W2"}
    idx, tgt = gpt.synthetic_batch(cfg, 4, DEV)
    loss = m(idx, tgt)
    got = torch.autograd.grad(loss, list(m.parameters()))
    B, T, d = 4, 64, 128
    x = m.wte[idx] + m.wpe[:T]
    for b in m.blocks:
        q, k, v = (F.rms_norm(x, (d,)) @ b.qkv.T).split(d, dim=-1)
        q, k, v = (t.view(B, T, 4, d // 4).transpose(1, 2) for t in (q, k, v))
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        x = x + y.transpose(1, 2).reshape(B, T, d) @ b.proj.T
        h = F.rms_norm(x, (d,)).view(B * T, d)
        x = x + (torch.relu(h @ b.W1.T).square() @ b.W2.T).view(B, T, d)
    logits = F.rms_norm(x, (d,)) @ m.wte.T
    want = F.cross_entropy(logits.float().view(B * T, -1), tgt.view(-1))
    assert torch.equal(loss, want)
    assert all(torch.equal(p, q) for p, q in zip(got, torch.autograd.grad(want, list(m.parameters()))))


def test_command(capsys, monkeypatch):
    for k in ("WORLD_SIZE", "RANK", "LOCAL_RANK"):
        monkeypatch.delenv(k, raising=False)
    args = "--steps 1 --warmup 1 --batch 2 --layers 2 --width 128 --heads 4 --hidden 512 --vocab 512 --seq 64".split()
    for more, k in ((["--sandwich"], 0), (["--sandwich", "--distill", "8"], 8), (["--dense", "--distill", "8"], 8)):
        assert train_gpt.main(args + more) == 0
        out = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
        assert out["distill_top_k"] == k and out["sandwich"] == ("--sandwich" in more) and math.isfinite(out["loss"])
