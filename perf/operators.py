"""The scoring, distillation and block-norm operators: their cases, inputs and plain forms.

Three operators (a case's "op"):

  score    sf.token_logprobs: log probabilities of given tokens, the entropy of
           each row and its top alternatives, from logits; with "train" also the
           gradient of all three with respect to the logits
  distill  sf.distill_topk: the divergence of a student's logits from a
           teacher's top log probabilities ("renorm": the listed mass scaled to
           one; "bucket": the rest of the mass is one more class); with "train"
           also its gradient
  norm     sf.residual_norm: RMS norm after a block, gate, scaled residual add and
           the RMS norm before the next block; with "train" also every gradient

With `own` false run() computes them in elementary torch operations (32 bits,
rounded once at the end); with `own` true it calls this package.
"""
import math

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
#: A listed mass this near to one leaves no rest: less is the rounding of the scores themselves.
REST_FLOOR = 2.0 ** -20
MOST_LOGITS = 400_000_000  # elements of a drawn case's logits
MOST_STREAM = 130_000_000  # elements of a drawn case's residual stream


def listed():
    def score(name, rows, vocab, dtype, top, temperature=1.0, train=False, ignored=False, masked=False):
        return {"name": name, "op": "score", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top,
                "temperature": temperature, "train": train, "ignored": ignored, "masked": masked}

    def distill(name, rows, vocab, dtype, top, tail, temperature=1.0, train=True):
        return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "tail": tail,
                "temperature": temperature, "train": train}

    def norm(name, rows, width, stream, dtype, post, gates, scale=1.0, train=True):
        return {"name": name, "op": "norm", "rows": rows, "width": width, "stream": stream, "dtype": dtype, "post": post,
                "gates": gates, "scale": scale, "train": train}

    return [
        # one decoding step of eight sequences: the chosen tokens' log probabilities and eight alternatives each
        score("score_decode_8x50304_bf16_k8", 8, 50304, "bf16", 8, 0.8),
        # a constrained decoding step over a large vocabulary in float32, most of it masked to -inf
        score("score_masked_3x200003_f32_k100", 3, 200003, "f32", 100, masked=True),
        # held-out scoring (perplexity) of 16 sequences of 1024 tokens, padding ignored
        score("score_eval_16384x50304_bf16", 16384, 50304, "bf16", 0, ignored=True),
        # a teacher's 64 alternatives for every position of eight sequences
        score("score_teacher_8192x50304_bf16_k64", 8192, 50304, "bf16", 64, 2.0),
        # a policy-gradient step: log probabilities, entropy bonus, odd vocabulary, float32 logits
        score("score_policy_2047x32003_f32", 2047, 32003, "f32", 0, train=True, ignored=True),
        # a small distillation step: few tokens, 16 alternatives, renormalised
        distill("distill_512x32003_f16_k16", 512, 32003, "f16", 16, "renorm", 2.0),
        # the distillation step of the GPT harness: 16 sequences of 1024, 64 alternatives and the rest's bucket
        distill("distill_16384x50304_bf16_k64", 16384, 50304, "bf16", 64, "bucket"),
        # the distance of a finished student on held-out tokens: forward only
        distill("distill_eval_1000x131072_f32_k128", 1000, 131072, "f32", 128, "bucket", train=False),
        # one new token for each of eight sequences
        norm("norm_decode_8x768_bf16", 8, 768, "bf16", "bf16", True, 1, train=False),
        # the GPT harness's training step: 32 sequences of 1024 tokens, learned gate
        norm("norm_train_32768x768_bf16", 32768, 768, "bf16", "bf16", True, 1, 0.7),
        # a wide stack with a float32 residual stream and one gate for each of 8 sequences
        norm("norm_train_8192x8192_f32_bf16", 8192, 8192, "f32", "bf16", True, 8),
        # an odd width and an odd number of rows, no norm after the block
        norm("norm_train_4999x1001_f32", 4999, 1001, "f32", "f32", False, 1, 0.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case: rows from one token to a large batch, vocabularies of 300 to
    262144, widths of 48 to 16384, every type, odd sizes among them."""
    op = rng.choice(("score", "distill", "norm"))
    if op == "norm":
        width = _log_int(rng, 48, 16384)
        if rng.random() < 0.6:
            width = -(-width // 64) * 64
        gates = rng.choice((0, 1, 1, _log_int(rng, 2, 32)))
        per = _log_int(rng, 1, max(1, min(65536, MOST_STREAM // width) // max(1, gates)))
        stream, dtype = rng.choice((("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f32", "f16")))
        return {"op": op, "rows": per * max(1, gates), "width": width, "stream": stream, "dtype": dtype,
                "post": rng.random() < 0.6, "gates": gates, "scale": rng.choice((1.0, 0.5, 0.9)),
                "train": rng.random() < 0.7}
    vocab = _log_int(rng, 300, 262144)
    if rng.random() < 0.5:
        vocab = -(-vocab // 64) * 64
    rows = _log_int(rng, 1, min(16384, MOST_LOGITS // vocab))
    c = {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(("bf16", "f16", "f32")),
         "temperature": rng.choice((1.0, 0.7, 2.0))}
    if op == "score":
        c["top"] = rng.choice((0, 1, _log_int(rng, 2, 128)))
        return {**c, "train": rng.random() < 0.4, "ignored": rng.random() < 0.3, "masked": rng.random() < 0.2}
    return {**c, "top": _log_int(rng, 1, 128), "tail": rng.choice(("renorm", "bucket")), "train": rng.random() < 0.7}


class _State:
    pass


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = _State()
    s.case = case
    dtype = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0, base=0.0, dtype=torch.float32):
        return torch.randn(*shape, device=dev, generator=g).mul_(scale).add_(base).to(dtype)

    if case["op"] == "norm":
        R, D, G = case["rows"], case["width"], case["gates"]
        sdt = DTYPES[case["stream"]]
        s.x = rand(R, D, scale=2.0, dtype=sdt)
        s.y = rand(R, D, scale=0.8, dtype=dtype)
        s.pre = rand(D, scale=0.1, base=1.0)
        s.post = rand(D, scale=0.1, base=1.0) if case["post"] else None
        s.gate = rand(G, D, scale=0.2, base=0.5, dtype=dtype) if G > 1 else rand(D, scale=0.2, base=0.5) if G else None
        if case["train"]:
            s.dx_new = rand(R, D, dtype=sdt)
            s.dh = rand(R, D, dtype=dtype)
            s.leaves = [t.requires_grad_() for t in (s.x, s.y, s.pre, s.post, s.gate) if t is not None]
        return s

    R, V = case["rows"], case["vocab"]
    s.logits = torch.empty(R, V, device=dev, dtype=dtype)
    if case["op"] == "score":
        for a in range(0, R, 2048):
            s.logits[a:a + 2048] = rand(min(2048, R - a), V, scale=2.5)
        s.targets = torch.randint(0, V, (R,), device=dev, generator=g)
        if case["masked"]:  # each row keeps its own share of the vocabulary, the first one nothing
            keep = torch.rand(R, 1, device=dev, generator=g) * 0.1
            keep[0] = 0.0
            s.logits[torch.rand(R, V, device=dev, generator=g) >= keep] = -math.inf
        if case["ignored"]:
            s.targets[torch.rand(R, device=dev, generator=g) < 0.1] = IGNORE
        if case["train"]:
            s.g_logp, s.g_entropy = rand(R), rand(R, scale=0.1)
            s.g_top = rand(R, case["top"], scale=0.1)
    else:  # the teacher's list: its alternatives and their log probabilities, from logits near the student's
        K, T = min(case["top"], V), case["temperature"]
        s.ids = torch.empty(R, K, device=dev, dtype=torch.int64)
        s.scores = torch.empty(R, K, device=dev)
        for a in range(0, R, 2048):
            n = min(2048, R - a)
            x = rand(n, V, scale=2.5)
            s.logits[a:a + n] = x
            x.add_(rand(n, V, scale=0.5)).mul_(1.0 / T)
            top, s.ids[a:a + n] = torch.topk(x, K, dim=-1)
            s.scores[a:a + n] = top - torch.logsumexp(x, dim=-1, keepdim=True)
        if case["train"]:
            s.g_loss = rand(R, scale=0.1, base=1.0)
    if case["train"]:
        s.logits.requires_grad_()
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _softmax_parts(logits, inv_t):
    """(d, s): d = (x - max x) / T (all zero in a row of -inf), s = sum exp(d) (zero there)."""
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    d = (x - torch.where(m == -math.inf, torch.zeros_like(m), m)) * inv_t
    return d, d.exp().sum(-1, keepdim=True)


def _plain_score(st):
    c = st.case
    R, V = st.logits.shape
    k, inv_t = min(c["top"], V), 1.0 / c["temperature"]
    logits = st.logits.detach()
    d, s = _softmax_parts(logits, inv_t)
    ln_s = s.log()
    empty, skip = s == 0, (st.targets == IGNORE)[:, None]
    t = st.targets.clamp_min(0)[:, None]
    inf = torch.full_like(ln_s, -math.inf)
    zero = torch.zeros_like(ln_s)
    lp = torch.where(empty, inf, d - ln_s)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1, keepdim=True)
    logp = torch.where(skip, zero, lp.gather(1, t))
    entropy = torch.where(skip, zero, entropy)
    out = {"logp": logp[:, 0], "entropy": entropy[:, 0]}
    ids = None
    if k:
        ids = torch.sort(logits.float(), dim=-1, descending=True, stable=True)[1][:, :k]
        out["top_logp"] = torch.where(skip, inf, lp.gather(1, ids))
        out["top_ids"] = torch.where(skip, torch.full_like(ids, -1), ids)
    if c["train"]:
        g, gh = st.g_logp[:, None], st.g_entropy[:, None]
        total = g + (st.g_top.sum(-1, keepdim=True) if k else 0.0)
        grad = -p * total - gh * torch.where(p > 0, p * (lp + entropy), torch.zeros_like(p))
        grad.scatter_add_(1, t, g)
        if k:
            grad.scatter_add_(1, ids, st.g_top[:, :k])
        grad = torch.where(skip | empty, torch.zeros_like(grad), grad * inv_t)
        out["grad"] = grad.to(logits.dtype)
    return out


def _plain_distill(st):
    c = st.case
    inv_t, bucket = 1.0 / c["temperature"], c["tail"] == "bucket"
    logits = st.logits.detach()
    d, s = _softmax_parts(logits, inv_t)
    ln_s = s.log()
    if bucket:
        q = st.scores.exp()
        rest = (1.0 - st.scores.double().exp().sum(-1, keepdim=True)).float()
        rest = torch.where(rest < REST_FLOOR, torch.zeros_like(rest), rest)
        off = d.exp().scatter(1, st.ids, 0.0).sum(-1, keepdim=True)  # the student's mass off the list, times s
        if st.ids.shape[1] == logits.shape[1]:  # the list names every class: no rest
            rest = torch.zeros_like(rest)
    else:
        q = torch.softmax(st.scores, dim=-1)
    ln_q = q.log()
    ln_p = d.gather(1, st.ids) - ln_s
    loss = torch.where(q > 0, q * (ln_q - ln_p), torch.zeros_like(q)).sum(-1, keepdim=True)
    if bucket:
        loss = loss + torch.where(rest > 0, rest * (rest.log() - (off.log() - ln_s)), torch.zeros_like(rest))
    out = {"loss": loss[:, 0]}
    if c["train"]:
        p = (d - ln_s).exp()
        mass = q.sum(-1, keepdim=True)
        if bucket:
            on_list = p.gather(1, st.ids) * (mass + rest) - q
            grad = (p * (mass + rest - torch.where(rest > 0, rest * s / off, torch.zeros_like(rest)))).scatter(1, st.ids, on_list)
        else:
            grad = (p * mass).scatter_add(1, st.ids, -q)
        out["grad"] = (grad * (st.g_loss[:, None] * inv_t)).to(logits.dtype)
    return out


def _plain_norm(st, eps=1e-6):
    c = st.case
    R, D = st.x.shape
    x, y, pre = st.x.detach().float(), st.y.detach().float(), st.pre.detach().float()
    G = max(1, c["gates"])
    gate = st.gate.detach().float().view(G, 1, D).expand(G, R // G, D).reshape(R, D) if c["gates"] else 1.0
    post = st.post.detach().float() if c["post"] else 1.0
    r1 = torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) if c["post"] else 1.0
    u = y * r1 * post
    xn = x * c["scale"] + gate * u
    r2 = torch.rsqrt(xn.square().mean(-1, keepdim=True) + eps)
    xh = xn * r2
    out = {"x": xn.to(st.x.dtype), "h": (xh * pre).to(st.y.dtype)}
    if c["train"]:
        dh = st.dh.float()
        t = dh * pre
        e = st.dx_new.float() + r2 * (t - xh * (t * xh).mean(-1, keepdim=True))
        out["dx"] = (e * c["scale"]).to(st.x.dtype)
        out["dpre"] = (dh * xh).sum(0, dtype=torch.float64).to(st.pre.dtype)
        if c["gates"]:
            out["dgate"] = (e * u).view(G, R // G, D).sum(1, dtype=torch.float64).view(st.gate.shape).to(st.gate.dtype)
        du = e * gate
        if c["post"]:
            yh = y * r1
            out["dpost"] = (du * yh).sum(0, dtype=torch.float64).to(st.post.dtype)
            v = du * post
            du = r1 * (v - yh * (v * yh).mean(-1, keepdim=True))
        out["dy"] = du.to(st.y.dtype)
    return out


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------
def _own_score(st):
    import autoresearch2_b200 as sf
    c = st.case
    k = min(c["top"], c["vocab"])
    r = sf.token_logprobs(st.logits, st.targets, top_k=k, temperature=c["temperature"])
    out = {"logp": r.logp.detach(), "entropy": r.entropy.detach()}
    if k:
        out["top_ids"], out["top_logp"] = r.top_ids, r.top_logp.detach()
    if c["train"]:
        outs, gs = [r.logp, r.entropy], [st.g_logp, st.g_entropy]
        if k:
            outs, gs = outs + [r.top_logp], gs + [st.g_top[:, :k]]
        out["grad"] = torch.autograd.grad(outs, st.logits, gs)[0]
    return out


def _own_distill(st):
    import autoresearch2_b200 as sf
    c = st.case
    loss = sf.distill_topk(st.logits, st.ids, st.scores, temperature=c["temperature"], tail=c["tail"])
    out = {"loss": loss.detach()}
    if c["train"]:
        out["grad"] = torch.autograd.grad(loss, st.logits, st.g_loss)[0]
    return out


def _own_norm(st):
    import autoresearch2_b200 as sf
    c = st.case
    x, y, gate = st.x, st.y, st.gate
    xn, h = sf.residual_norm(x, y, pre_weight=st.pre, post_weight=st.post, gate=gate, post_norm=c["post"],
                             residual_scale=c["scale"], eps=1e-6)
    out = {"x": xn.detach(), "h": h.detach()}
    if c["train"]:
        grads = iter(torch.autograd.grad([xn, h], st.leaves, [st.dx_new, st.dh]))
        out["dx"], out["dy"], out["dpre"] = next(grads), next(grads), next(grads)
        if c["post"]:
            out["dpost"] = next(grads)
        if c["gates"]:
            out["dgate"] = next(grads)
    return out


def run(state):
    op = state.case["op"]
    if op == "score":
        return _own_score(state) if own else _plain_score(state)
    if op == "distill":
        return _own_distill(state) if own else _plain_distill(state)
    return _own_norm(state) if own else _plain_norm(state)


def work(case):
    """Each input read once, each output written once (a gradient among them)."""
    es = BYTES[case["dtype"]]
    if case["op"] == "norm":
        R, D, ss = case["rows"], case["width"], BYTES[case["stream"]]
        n = R * D
        gate = max(case["gates"], 0) * D * (4 if case["gates"] == 1 else es)
        params = D * 4 * (2 if case["post"] else 1) + gate
        return {"bytes": n * (ss + es) * (4 if case["train"] else 2) + params * (2 if case["train"] else 1),
                "flops": n * (40 if case["train"] else 12)}
    R, V = case["rows"], case["vocab"]
    k = min(case["top"], V)
    n = R * V
    if case["op"] == "score":
        small = R * 16 + R * k * 12 + (R * (8 + 4 * k) if case["train"] else 0)
    else:
        small = R * 4 + R * k * 12 + (R * 4 if case["train"] else 0)
    return {"bytes": n * es * (2 if case["train"] else 1) + small, "flops": n * (14 if case["train"] else 6)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    """What run() returns for these inputs, from the definitions in float64: softmax
    by torch's own float64 log-sum-exp, gradients of each row from the row's
    distribution, block by block of rows."""
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "norm":
        R, D, G = case["rows"], case["width"], max(1, case["gates"])
        per = R // G
        one = torch.ones(D, device=s.x.device, dtype=f8)
        pre = s.pre.detach().to(f8)
        post = s.post.detach().to(f8) if case["post"] else one
        gates = s.gate.detach().to(f8).view(G, D) if case["gates"] else one[None]
        sums = {"dpre": torch.zeros_like(one), "dpost": torch.zeros_like(one), "dgate": torch.zeros(G, D, device=one.device, dtype=f8)}
        parts = {"x": [], "h": [], "dx": [], "dy": []}
        step = max(1, (1 << 26) // D)
        for gi in range(G):
            for a in range(gi * per, (gi + 1) * per, step):
                b = min(a + step, (gi + 1) * per)
                x, y = s.x.detach()[a:b].to(f8), s.y.detach()[a:b].to(f8)
                n1 = (y.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() if case["post"] else torch.ones(b - a, 1, device=x.device, dtype=f8)
                u = y / n1 * post
                z = case["scale"] * x + gates[gi] * u
                n2 = (z.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt()
                parts["x"].append(z)
                parts["h"].append(z / n2 * pre)
                if case["train"]:
                    dh, dz = s.dh[a:b].to(f8), s.dx_new[a:b].to(f8)
                    w = dh * pre
                    dz = dz + w / n2 - z * (w * z).sum(-1, keepdim=True) / (D * n2.pow(3))
                    sums["dpre"] += (dh * z / n2).sum(0)
                    sums["dgate"][gi] += (dz * u).sum(0)
                    parts["dx"].append(dz * case["scale"])
                    du = dz * gates[gi]
                    if case["post"]:
                        sums["dpost"] += (du * y / n1).sum(0)
                        v = du * post
                        du = v / n1 - y * (v * y).sum(-1, keepdim=True) / (D * n1.pow(3))
                    parts["dy"].append(du)
        out = {k: torch.cat(v) for k, v in parts.items() if v}
        if case["train"]:
            out["dpre"] = sums["dpre"]
            if case["post"]:
                out["dpost"] = sums["dpost"]
            if case["gates"]:
                out["dgate"] = sums["dgate"].view(s.gate.shape)
        return out

    R, V = case["rows"], case["vocab"]
    k, T = min(case["top"], V), case["temperature"]
    logits = s.logits.detach()
    step = max(1, (1 << 26) // V)
    parts = {}

    def put(**kw):
        for name, v in kw.items():
            parts.setdefault(name, []).append(v)

    for a in range(0, R, step):
        z = logits[a:a + step].to(f8) / T
        lz = torch.logsumexp(z, dim=-1, keepdim=True)
        lp = torch.where(lz == -math.inf, torch.full_like(z, -math.inf), z - lz)
        p = torch.exp(lp)
        rows = torch.arange(z.shape[0], device=z.device)
        if case["op"] == "score":
            t = s.targets[a:a + step]
            live = (t != IGNORE)
            tt = torch.where(live, t, torch.zeros_like(t))
            plnp = torch.special.xlogy(p, p)
            h = torch.where(live, -plnp.sum(-1), 0.0)
            put(logp=torch.where(live, lp[rows, tt], 0.0), entropy=h)
            if k:
                top, _ = torch.topk(z, k, dim=-1)
                put(top_logp=torch.where(live[:, None] & (lz > -math.inf), top - lz, -math.inf))
            if case["train"]:
                g, gh = s.g_logp[a:a + step].to(f8), s.g_entropy[a:a + step].to(f8)
                gt = s.g_top[a:a + step, :k].to(f8)
                grad = -p * (g + gt.sum(-1))[:, None] - gh[:, None] * (plnp + p * h[:, None])
                grad[rows, tt] += g
                if k:
                    at = torch.sort(logits[a:a + step], dim=-1, descending=True, stable=True)[1][:, :k]
                    grad[rows[:, None], at] += gt
                grad = grad / T
                grad[~live | (lz[:, 0] == -math.inf)] = 0.0
                put(grad=grad.to(torch.float32) if R * V > 1 << 28 else grad)
        else:
            ids, c = s.ids[a:a + step], s.scores[a:a + step].to(f8)
            on = torch.zeros_like(z)
            if case["tail"] == "renorm":
                q = torch.exp(c - torch.logsumexp(c, dim=-1, keepdim=True))
                on[rows[:, None], ids] = q
                loss = (torch.special.xlogy(q, q) - q * lp[rows[:, None], ids]).sum(-1)
                grad = p - on
            else:
                q = torch.exp(c)
                r = 1.0 - q.sum(-1)
                r = torch.where((r < REST_FLOOR) | (k == V), torch.zeros_like(r), r)
                pr = p.clone()
                pr[rows[:, None], ids] = 0.0
                pr = pr.sum(-1)
                on[rows[:, None], ids] = q
                loss = (torch.special.xlogy(q, q) - q * lp[rows[:, None], ids]).sum(-1)
                loss = loss + torch.where(r > 0, r * (torch.log(r) - torch.log(pr)), torch.zeros_like(r))
                listed_ = torch.zeros_like(z, dtype=torch.bool)
                listed_[rows[:, None], ids] = True
                share = torch.where(r > 0, r / pr, torch.zeros_like(r))[:, None]
                grad = p * (q.sum(-1) + r)[:, None] - torch.where(listed_, on, p * share)
            put(loss=loss)
            if case["train"]:
                grad = grad * (s.g_loss[a:a + step].to(f8) / T)[:, None]
                put(grad=grad.to(torch.float32) if R * V > 1 << 28 else grad)
    out = {name: torch.cat(v) for name, v in parts.items()}
    if case["op"] == "score" and k:
        out["top_ids"] = None
    return out
