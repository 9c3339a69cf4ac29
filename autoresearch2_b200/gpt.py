"""A GPT-style decoder whose MLPs are the sparse ReLU^2 FFN: the end-to-end
consumer of the hot path.  The reference has no GPT model; its nearest
harness is DeepFFN (old/lib_sparse/prepare.py:50-78).

    GPTConfig(n_layer=12, n_head=12, n_embd=768, ffn_hidden=3072, vocab=50304, seq_len=1024)
    GPT(cfg, sparse=True, device="cuda", dtype=torch.bfloat16)
    TrainStep(model, idx, targets, lr=3e-4)  one AdamW step per call, returns the loss tensor
    DistillStep(student, teacher, idx, targets, top_k=64)  the same on a teacher's top logits
    model.score(idx, targets, top_k=8)  TokenLogprobs: log probabilities, entropy, alternatives
    model.packed_weights()  the blocks' weights in 8 bits, for model(idx, weights=...) and score
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
one, the gates at (2 * n_layer) ** -0.5.

GPTConfig(gated="silu") (or "gelu", "relu", "relu2") makes the MLPs gated ones,
W2 (act(Wg h) * (Wu h)), by gated_ffn (sparse=False: torch).  GPTConfig(ckpt8=True)
keeps activations for the backward in 8 bits: the gated MLPs' and, by
ckpt_linear, the inputs of the attention's projections.  Without gradients the
blocks' products also run on weights in 8 bits (fp8_matmul; activations are
packed on the way).  All of these are CUDA only.  score() and DistillStep run on token_logprobs and
distill_topk: a dense GPT teaches a sparse one, or any GPT a smaller one with
the same vocabulary.
"""
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import bitsparse as bs
from .ffn import FFNSpRelu2
from .fp8 import ckpt_linear, fp8_matmul, fp8_pack
from .glu import gated_ffn
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
    gated: Optional[str] = None  # activation of gated MLPs (None: ReLU^2, two matrices)
    ckpt8: bool = False  # activations for the backward in 8 bits


def flops_per_token(cfg: GPTConfig) -> float:
    """Training FLOPs per token: 6 x the matmul parameters (embedding tied to
    the output projection counted once, positions excluded) plus the
    attention scores and values, 12 x layers x width x sequence length."""
    d, L = cfg.n_embd, cfg.n_layer
    per_layer = 4 * d * d + (3 if cfg.gated else 2) * d * cfg.ffn_hidden
    return 6 * (L * per_layer + d * cfg.vocab) + 12 * L * d * cfg.seq_len


ACTS = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu, "relu2": lambda x: F.relu(x).square()}


class Block(nn.Module):
    def __init__(self, cfg, sparse, device, dtype):
        super().__init__()
        d, h = cfg.n_embd, cfg.ffn_hidden
        self.n_head = cfg.n_head
        self.qkv = nn.Parameter(torch.empty(3 * d, d, device=device, dtype=dtype))
        self.proj = nn.Parameter(torch.empty(d, d, device=device, dtype=dtype))
        self.gated, self.ckpt8 = cfg.gated, cfg.ckpt8
        for name in ("Wg", "Wu") if cfg.gated else ("W1",):
            self.register_parameter(name, nn.Parameter(torch.empty(h, d, device=device, dtype=dtype)))
        self.W2 = nn.Parameter(torch.empty(d, h, device=device, dtype=dtype))
        self.sparse = sparse
        if cfg.sandwich:
            for name in ("attn_pre", "attn_post", "attn_gate", "mlp_pre", "mlp_post", "mlp_gate"):
                self.register_parameter(name, nn.Parameter(torch.empty(d, device=device, dtype=torch.float32)))

    def linear(self, x, name, w8=None):
        """x times a weight: as packed in w8, or the parameter."""
        if w8 is not None:
            return fp8_matmul(x, w8[name])
        W = getattr(self, name)
        return ckpt_linear(x, W) if self.ckpt8 else x @ W.T

    def attention(self, h, w8=None):
        B, T, d = h.shape
        q, k, v = self.linear(h, "qkv", w8).split(d, dim=-1)
        q, k, v = (t.view(B, T, self.n_head, d // self.n_head).transpose(1, 2) for t in (q, k, v))
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return self.linear(y.transpose(1, 2).reshape(B, T, d), "proj", w8)

    def mlp(self, h, arena, w8=None):
        B, T, d = h.shape
        h = h.view(B * T, d)
        if w8 is not None:
            g = self.linear(h, "Wg" if self.gated else "W1", w8)
            m = self.linear(ACTS[self.gated](g) * self.linear(h, "Wu", w8) if self.gated else ACTS["relu2"](g), "W2", w8)
        elif self.gated and self.sparse:
            m = gated_ffn(h, self.Wg, self.Wu, self.W2, self.gated, "fp8" if self.ckpt8 else None)
        elif self.gated:
            m = (ACTS[self.gated](h @ self.Wg.T) * (h @ self.Wu.T)) @ self.W2.T
        elif self.sparse:
            m = FFNSpRelu2.apply(h, self.W1, self.W2, arena)
        else:
            m = torch.relu(h @ self.W1.T).square() @ self.W2.T
        return m.view(B, T, d)

    def forward(self, x, arena, w8=None):
        d = x.shape[-1]
        x = x + self.attention(F.rms_norm(x, (d,)), w8)
        return x + self.mlp(F.rms_norm(x, (d,)), arena, w8)

    def sandwich_forward(self, x, h, arena, next_pre, w8=None):
        """(x, h) after the block, h the norm for what follows (weights next_pre)."""
        x, h = residual_norm(x, self.attention(h, w8), self.mlp_pre, self.attn_post, self.attn_gate, post_norm=True)
        return residual_norm(x, self.mlp(h, arena, w8), next_pre, self.mlp_post, self.mlp_gate, post_norm=True)


class GPT(nn.Module):
    def __init__(self, cfg: GPTConfig, sparse=True, device="cuda", dtype=torch.bfloat16, fill=0.6, seed=0):
        super().__init__()
        if cfg.gated is not None and cfg.gated not in ACTS:
            raise ValueError(f"gated must be one of {', '.join(ACTS)}, got {cfg.gated!r}")
        if cfg.ckpt8 and not cfg.gated:
            raise ValueError("ckpt8 goes with gated MLPs: the sparse FFN packs its activations by itself")
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

    @torch.no_grad()
    def packed_weights(self):
        """The blocks' weights in 8 bits as they are now, one dict a block, for calls
        without gradients: model(idx, weights=...), score(..., weights=...)."""
        names = ("qkv", "proj", *(("Wg", "Wu") if self.cfg.gated else ("W1",)), "W2")
        return [{name: fp8_pack(getattr(blk, name)) for name in names} for blk in self.blocks]

    def forward(self, idx, targets=None, weights=None):
        B, T = idx.shape
        packed = weights is not None
        if not packed:
            weights = [None] * len(self.blocks)
        elif torch.is_grad_enabled() or len(weights) != len(self.blocks):
            raise ValueError("packed weights are for calls without gradients, one dict a block")
        x = self.wte[idx] + self.wpe[:T]
        arena = None
        if self.sparse and not self.cfg.gated and not packed:
            arena = self.arena_for(B * T).as_sparse_data()
        if self.cfg.sandwich:
            pres = [blk.attn_pre for blk in self.blocks] + [self.norm_out]
            x, h = residual_norm(x, pre_weight=pres[0])
            for blk, next_pre, w8 in zip(self.blocks, pres[1:], weights):
                x, h = blk.sandwich_forward(x, h, arena, next_pre, w8)
        else:
            for blk, w8 in zip(self.blocks, weights):
                x = blk(x, arena, w8)
            h = F.rms_norm(x, (x.shape[-1],))
        logits = h @ self.wte.T
        if targets is None:
            return logits
        return F.cross_entropy(logits.float().view(B * T, -1), targets.view(-1))

    @torch.no_grad()
    def score(self, idx, targets=None, top_k=0, temperature=1.0, ignore_index=-100, weights=None):
        """token_logprobs of the model's logits for idx [B, T]: the targets' log
        probabilities [B, T], entropies and top_k alternatives (CUDA only); weights:
        packed_weights() to run on."""
        return token_logprobs(self(idx, weights=weights), targets, top_k=top_k, temperature=temperature, ignore_index=ignore_index)


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
