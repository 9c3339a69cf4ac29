"""A GPT-style decoder whose MLPs are the sparse ReLU^2 FFN: the end-to-end
consumer of the hot path.  The reference has no GPT model; its nearest
harness is DeepFFN (old/lib_sparse/prepare.py:50-78).

    GPTConfig(n_layer=12, n_head=12, n_embd=768, ffn_hidden=3072, vocab=50304, seq_len=1024)
    GPT(cfg, sparse=True, device="cuda", dtype=torch.bfloat16)
    TrainStep(model, idx, targets, lr=3e-4)  one AdamW step per call, returns the loss tensor
    DistillStep(student, teacher, idx, targets, top_k=64)  the same on a teacher's top logits
    model.score(idx, targets, top_k=8)  TokenLogprobs: log probabilities, entropy, alternatives
    synthetic_batch(cfg, batch, device)      seeded uniform token ids and next-token targets

Blocks: x += attn(rms_norm(x)); x += mlp(rms_norm(x)); causal attention by
torch's scaled_dot_product_attention; learned positions; the token embedding
is tied to the output projection; weights ~ N(0, 0.02).  With sparse=True
every MLP runs FFNSpRelu2 over one vals arena shared by all layers and
rewound at each step (an arena of `fill` x the dense activation size of all
layers; 0.6 by default, for the ~50% zeros of ReLU at initialisation), so
the stack keeps only the compacted ReLU outputs between forward and
backward; sparse=False runs the same MLP as dense torch matmuls.  An arena
too small for a step's activations sets the library's status word (values
past the end are dropped): check_status() after a step reports it.

GPTConfig(sandwich=True) norms every block's output too and gates it:
x = x + gate * rms(block(rms(x) * w_pre)) * w_post, the last norm before the
output projection included; a block's norms, gate and residual add are one
call of residual_norm (CUDA only; eps 1e-6).  The weights, float32, start at
one, the gates at (2 * n_layer) ** -0.5.  score() and DistillStep run on token_logprobs and
distill_topk: a dense GPT teaches a sparse one, or any GPT a smaller one with
the same vocabulary.
"""
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import bitsparse as bs
from .ffn import FFNSpRelu2
from .logits import distill_topk, token_logprobs
from .norms import residual_norm

__all__ = ["GPTConfig", "GPT", "TrainStep", "DistillStep", "flops_per_token", "synthetic_batch", "mfu"]


@dataclass
class GPTConfig:
    n_layer: int = 12
    n_head: int = 12
    n_embd: int = 768
    ffn_hidden: int = 3072
    vocab: int = 50304
    seq_len: int = 1024
    sandwich: bool = False  # norms and gates after the blocks as well as norms before them


def flops_per_token(cfg: GPTConfig) -> float:
    """Training FLOPs per token: 6 x the matmul parameters (embedding tied to
    the output projection counted once, positions excluded) plus the
    attention scores and values, 12 x layers x width x sequence length."""
    d, L = cfg.n_embd, cfg.n_layer
    per_layer = 4 * d * d + 2 * d * cfg.ffn_hidden
    return 6 * (L * per_layer + d * cfg.vocab) + 12 * L * d * cfg.seq_len


class Block(nn.Module):
    def __init__(self, cfg, sparse, device, dtype):
        super().__init__()
        d, h = cfg.n_embd, cfg.ffn_hidden
        self.n_head = cfg.n_head
        self.qkv = nn.Parameter(torch.empty(3 * d, d, device=device, dtype=dtype))
        self.proj = nn.Parameter(torch.empty(d, d, device=device, dtype=dtype))
        self.W1 = nn.Parameter(torch.empty(h, d, device=device, dtype=dtype))
        self.W2 = nn.Parameter(torch.empty(d, h, device=device, dtype=dtype))
        self.sparse = sparse
        if cfg.sandwich:
            for name in ("attn_pre", "attn_post", "attn_gate", "mlp_pre", "mlp_post", "mlp_gate"):
                self.register_parameter(name, nn.Parameter(torch.empty(d, device=device, dtype=torch.float32)))

    def attention(self, h):
        B, T, d = h.shape
        q, k, v = (h @ self.qkv.T).split(d, dim=-1)
        q, k, v = (t.view(B, T, self.n_head, d // self.n_head).transpose(1, 2) for t in (q, k, v))
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return y.transpose(1, 2).reshape(B, T, d) @ self.proj.T

    def mlp(self, h, arena):
        B, T, d = h.shape
        h = h.view(B * T, d)
        if self.sparse:
            m = FFNSpRelu2.apply(h, self.W1, self.W2, arena)
        else:
            m = torch.relu(h @ self.W1.T).square() @ self.W2.T
        return m.view(B, T, d)

    def forward(self, x, arena):
        d = x.shape[-1]
        x = x + self.attention(F.rms_norm(x, (d,)))
        return x + self.mlp(F.rms_norm(x, (d,)), arena)

    def sandwich_forward(self, x, h, arena, next_pre):
        """(x, h) after the block, h the norm for what follows (weights next_pre)."""
        x, h = residual_norm(x, self.attention(h), self.mlp_pre, self.attn_post, self.attn_gate, post_norm=True)
        return residual_norm(x, self.mlp(h, arena), next_pre, self.mlp_post, self.mlp_gate, post_norm=True)


class GPT(nn.Module):
    def __init__(self, cfg: GPTConfig, sparse=True, device="cuda", dtype=torch.bfloat16, fill=0.6, seed=0):
        super().__init__()
        self.cfg, self.sparse, self.fill = cfg, sparse, fill
        self.wte = nn.Parameter(torch.empty(cfg.vocab, cfg.n_embd, device=device, dtype=dtype))
        self.wpe = nn.Parameter(torch.empty(cfg.seq_len, cfg.n_embd, device=device, dtype=dtype))
        self.blocks = nn.ModuleList(Block(cfg, sparse, device, dtype) for _ in range(cfg.n_layer))
        g = torch.Generator(device=device).manual_seed(seed)
        with torch.no_grad():
            for p in self.parameters():
                p.normal_(0.0, 0.02, generator=g)
            if cfg.sandwich:
                self.norm_out = nn.Parameter(torch.ones(cfg.n_embd, device=device, dtype=torch.float32))
                for blk in self.blocks:
                    for w in (blk.attn_pre, blk.attn_post, blk.mlp_pre, blk.mlp_post):
                        w.fill_(1.0)
                    blk.attn_gate.fill_((2 * cfg.n_layer) ** -0.5)
                    blk.mlp_gate.fill_((2 * cfg.n_layer) ** -0.5)
        self.arena = None

    def arena_for(self, tokens):
        """The shared vals arena, (re)allocated for `tokens` and rewound."""
        cap = int(tokens * self.cfg.ffn_hidden * self.cfg.n_layer * self.fill)
        if self.arena is None or self.arena.n != cap:
            self.arena = bs.TensorBuffer(cap, self.wte.device, self.wte.dtype).init_buffer()
        return self.arena.reset_buffer()

    def forward(self, idx, targets=None):
        B, T = idx.shape
        x = self.wte[idx] + self.wpe[:T]
        arena = self.arena_for(B * T).as_sparse_data() if self.sparse else None
        if self.cfg.sandwich:
            pres = [blk.attn_pre for blk in self.blocks] + [self.norm_out]
            x, h = residual_norm(x, pre_weight=pres[0])
            for blk, next_pre in zip(self.blocks, pres[1:]):
                x, h = blk.sandwich_forward(x, h, arena, next_pre)
        else:
            for blk in self.blocks:
                x = blk(x, arena)
            h = F.rms_norm(x, (x.shape[-1],))
        logits = h @ self.wte.T
        if targets is None:
            return logits
        return F.cross_entropy(logits.float().view(B * T, -1), targets.view(-1))

    @torch.no_grad()
    def score(self, idx, targets=None, top_k=0, temperature=1.0, ignore_index=-100):
        """token_logprobs of the model's logits for idx [B, T]: the targets' log
        probabilities [B, T], entropies and top_k alternatives (CUDA only)."""
        return token_logprobs(self(idx), targets, top_k=top_k, temperature=temperature, ignore_index=ignore_index)


class TrainStep:
    """forward, backward and one fused AdamW step on a fixed (inputs, targets) batch."""

    def __init__(self, model, idx, targets, lr=3e-4):
        self.model, self.idx, self.targets = model, idx, targets
        self.opt = torch.optim.AdamW(model.parameters(), lr=lr, betas=(0.9, 0.95), weight_decay=0.0,
                                     fused=True)

    def __call__(self):
        loss = self.model(self.idx, self.targets)
        loss.backward()
        self.opt.step()
        self.opt.zero_grad(set_to_none=True)
        return loss.detach()


class DistillStep:
    """TrainStep whose loss is the mean of distill_topk from the teacher's top_k
    alternatives at `temperature`, times its square (so that the gradient's size
    does not depend on it), plus hard_weight times the targets' cross-entropy.

    The teacher (a GPT of the same vocabulary) is run anew each step, without
    gradient; targets of -100 are left out of both parts.  With hard_weight 0
    targets may be None.  Another target outside the vocabulary makes a loss
    with a hard part NaN, adds no gradient and sets the status word, which
    check_status() after a step reports.  The two parts' gradients are rounded
    to the logits' type each, and their sum again."""

    def __init__(self, student, teacher, idx, targets=None, top_k=64, temperature=1.0, tail="bucket", hard_weight=0.0,
                 lr=3e-4):
        if hard_weight and targets is None:
            raise ValueError("hard_weight needs targets")
        self.model, self.teacher, self.idx, self.targets = student, teacher, idx, targets
        self.top_k, self.temperature, self.tail, self.hard_weight = top_k, temperature, tail, hard_weight
        self.opt = torch.optim.AdamW(student.parameters(), lr=lr, betas=(0.9, 0.95), weight_decay=0.0, fused=True)

    def loss(self):
        T = self.temperature
        listed = self.teacher.score(self.idx, self.targets, top_k=self.top_k, temperature=T)
        logits = self.model(self.idx)
        soft = distill_topk(logits, listed.top_ids, listed.top_logp, temperature=T, tail=self.tail)
        n = soft.numel() if self.targets is None else (self.targets != -100).sum().clamp_min(1)
        loss = soft.sum() * (T * T / n)
        if self.hard_weight:
            loss = loss - token_logprobs(logits, self.targets).logp.sum() * (self.hard_weight / n)
        return loss

    def __call__(self):
        loss = self.loss()
        loss.backward()
        self.opt.step()
        self.opt.zero_grad(set_to_none=True)
        return loss.detach()


def synthetic_batch(cfg: GPTConfig, batch, device, seed=0):
    """Uniform random token ids (seeded), inputs and next-token targets."""
    g = torch.Generator(device=device).manual_seed(seed)
    toks = torch.randint(0, cfg.vocab, (batch, cfg.seq_len + 1), generator=g, device=device)
    return toks[:, :-1].contiguous(), toks[:, 1:].contiguous()


def mfu(tokens_per_s, cfg, peak_tflops):
    """Model FLOPs utilisation against a peak in TFLOP/s."""
    return tokens_per_s * flops_per_token(cfg) / (peak_tflops * 1e12)
