"""The 8-bit block format, its products and the gated feed-forward block: cases, inputs and plain forms.

Four operators (a case's "op"):

  pack    sf.fp8_pack and sf.fp8_unpack: an activation kept in 8 bits (e4m3, one
          power-of-two scale for each 128 elements of a row) and read back
  linear  sf.ckpt_linear: y = x W^T that keeps x in 8 bits for its backward
  gated   sf.gated_ffn: y = (act(x Wg^T) * (x Wu^T)) W2^T; with "train" also every
          gradient, from x, x Wg^T and x Wu^T as the forward kept them: in the
          inputs' type, or ("fp8") in 8 bits
  fp8mm   sf.fp8_matmul: a b^T of two matrices in the 8-bit format (with "plain_a"
          the first one is packed within the call)

The format: values [rows, width] in float8_e4m3fn, rows 16 bytes aligned; scales one
exponent byte a block (2^(byte - 127)), stored as tiles of 128 rows x 4 blocks,
[rows / 128][blocks / 4][row % 32][row % 128 / 32][block % 4].  With amax the
largest finite magnitude of a block, the scale is the smallest 2^e with
amax <= 448 * 2^e and e >= -118 (1 for a block of zeros).

With `own` false run() computes them in elementary torch operations (32 bits,
rounded once at the end); with `own` true it calls this package.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
BLOCK = 128
LOWEST = -118  # smallest exponent of a scale
MOST_PACK = 1 << 28         # elements of a drawn activation
MOST_LINEAR = 1 << 38       # rows x in x out of a drawn linear layer
MOST_GATED = 1 << 38        # tokens x width x hidden of a drawn feed-forward block
MOST_PRODUCT = 1 << 39      # rows x out x in of a drawn 8-bit product


def listed():
    def pack(name, rows, width, dtype):
        return {"name": name, "op": "pack", "rows": rows, "width": width, "dtype": dtype}

    def linear(name, rows, width, out, dtype):
        return {"name": name, "op": "linear", "rows": rows, "width": width, "out": out, "dtype": dtype}

    def gated(name, rows, width, hidden, dtype, act, train=False, fp8=False):
        return {"name": name, "op": "gated", "rows": rows, "width": width, "hidden": hidden, "dtype": dtype, "act": act,
                "train": train, "fp8": fp8}

    def fp8mm(name, rows, out, width, dtype, plain_a=False):
        return {"name": name, "op": "fp8mm", "rows": rows, "out": out, "width": width, "dtype": dtype, "plain_a": plain_a}

    return [
        # one layer's input of a small batch, odd sizes, float16
        pack("pack_333x1001_f16", 333, 1001, "f16"),
        # the activation of a wide layer: 65536 tokens
        pack("pack_65536x4096_bf16", 65536, 4096, "bf16"),
        # the GPT harness's qkv projection in training: 32 sequences of 1024 tokens
        linear("linear_train_32768x768x2304_bf16", 32768, 768, 2304, "bf16"),
        # an odd layer of a small model in float16
        linear("linear_train_1499x1001x515_f16", 1499, 1001, 515, "f16"),
        # one new token through the GPT harness's width
        gated("gated_decode_1x768x2048_bf16", 1, 768, 2048, "bf16", "silu"),
        # one step of 16 sequences through a wide layer
        gated("gated_decode_16x4096x14336_f16", 16, 4096, 14336, "f16", "gelu"),
        # the GPT harness's training step, activations kept in 8 bits
        gated("gated_train_32768x768x2048_bf16_fp8", 32768, 768, 2048, "bf16", "silu", train=True, fp8=True),
        # a wide layer's training step, activations kept in 16 bits
        gated("gated_train_8192x4096x14336_bf16", 8192, 4096, 14336, "bf16", "silu", train=True),
        # odd sizes, few tokens, squared ReLU
        gated("gated_train_777x1001x1357_f16_fp8", 777, 1001, 1357, "f16", "relu2", train=True, fp8=True),
        # one new token against weights kept in 8 bits
        fp8mm("fp8mm_decode_1x14336x4096_bf16", 1, 14336, 4096, "bf16"),
        # a prompt batch against weights kept in 8 bits
        fp8mm("fp8mm_16384x8192x4096_bf16", 16384, 8192, 4096, "bf16"),
        # odd sizes, the activations packed within the call
        fp8mm("fp8mm_1023x1777x1333_f16_plain", 1023, 1777, 1333, "f16", plain_a=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _width(rng, lo, hi):
    n = _log_int(rng, lo, hi)
    return min(hi, -(-n // 64) * 64) if rng.random() < 0.6 else n


def draw(rng):
    """One more case: from one token to a large batch, widths of 64 to 16384, odd
    sizes among them, every type and activation."""
    op = rng.choice(("pack", "linear", "gated", "gated", "fp8mm", "fp8mm"))
    c = {"op": op, "dtype": rng.choice(("bf16", "f16"))}
    if op == "pack":
        width = _width(rng, 1, 16384)
        return {**c, "dtype": rng.choice(("bf16", "f16", "f32")), "rows": _log_int(rng, 1, min(65536, MOST_PACK // width)),
                "width": width}
    if op == "linear":
        width, out = _width(rng, 64, 8192), _width(rng, 64, 8192)
        return {**c, "rows": _log_int(rng, 1, min(32768, MOST_LINEAR // (width * out))), "width": width, "out": out}
    if op == "gated":
        width, hidden = _width(rng, 64, 8192), _width(rng, 64, 16384)
        train = rng.random() < 0.6
        return {**c, "rows": _log_int(rng, 1, min(32768, MOST_GATED // (width * hidden))), "width": width, "hidden": hidden,
                "act": rng.choice(("silu", "gelu", "relu", "relu2")), "train": train, "fp8": train and rng.random() < 0.5}
    width, out = _width(rng, 64, 16384), _width(rng, 64, 16384)
    return {**c, "rows": _log_int(rng, 1, min(16384, MOST_PRODUCT // (width * out))), "out": out, "width": width,
            "plain_a": rng.random() < 0.4}


class _State:
    pass


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = _State()
    s.case = case
    dtype = DTYPES[case["dtype"]]
    R, D = case["rows"], case["width"]

    def rand(rows, cols, scale=1.0):
        out = torch.empty(rows, cols, device=dev, dtype=dtype)
        for a in range(0, rows, 8192):
            n = min(8192, rows - a)
            out[a:a + n] = torch.randn(n, cols, device=dev, generator=g).mul_(scale)
        return out

    # normed activations: rows of somewhat unlike size, a few channels much larger than the rest
    s.x = rand(R, D)
    s.x *= torch.exp(torch.randn(R, 1, device=dev, generator=g) * 0.25).to(dtype)
    s.x[:, torch.randint(0, D, (max(1, D // 256),), device=dev, generator=g)] *= 8
    if case["op"] == "linear":
        s.W = rand(case["out"], D, D ** -0.5).requires_grad_()
        s.dy = rand(R, case["out"])
        s.x.requires_grad_()
    elif case["op"] == "gated":
        F = case["hidden"]
        s.Wg, s.Wu, s.W2 = rand(F, D, D ** -0.5), rand(F, D, D ** -0.5), rand(D, F, F ** -0.5)
        if case["train"]:
            s.dy = rand(R, D)
            s.leaves = [t.requires_grad_() for t in (s.x, s.Wg, s.Wu, s.W2)]
    elif case["op"] == "fp8mm":
        s.w = _blocks(rand(case["out"], D, D ** -0.5))
        if not case["plain_a"]:
            s.a = _blocks(s.x)
            s.x = None
    return s


# ---------------------------------------------------------------------------
# The format in torch operations
# ---------------------------------------------------------------------------
def _quantise(x):
    """(values as float32 before their scale, exponents [rows, blocks]) of x [rows, width]."""
    rows, width = x.shape
    nb = -(-width // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - width)).view(rows, nb, BLOCK)
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp_min(LOWEST)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    v = (x * _two_to(-e)[..., None]).to(torch.float8_e4m3fn).float()
    return v.view(rows, nb * BLOCK)[:, :width], e


def _two_to(e):
    """2^e in float32, by its bits."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _scaled(v, e):
    """Values times their block's 2^e."""
    rows, width = v.shape
    scale = _two_to(e).repeat_interleave(BLOCK, dim=1)[:, :width]
    return v * scale


def _blocks(x):
    """(values, scale tiles, shape) of x [rows, width], in the stored format."""
    rows, width = x.shape
    v, e = _quantise(x)
    ld = -(-width // 16) * 16
    values = torch.zeros(rows, ld, device=x.device, dtype=torch.float8_e4m3fn)
    values.view(torch.uint8)[:, :width] = v.to(torch.float8_e4m3fn).view(torch.uint8)
    nb = e.shape[1]
    rt, bt = -(-rows // 128), -(-nb // 4)
    s = torch.zeros(rt * 128, bt * 4, device=x.device, dtype=torch.uint8)
    s[:rows, :nb] = (e + 127).to(torch.uint8)
    tiles = s.view(rt, 4, 32, bt, 4).permute(0, 3, 2, 1, 4).contiguous()
    return values[:, :width], tiles, (rows, width)


def _unblock(q):
    """The matrix that (values, scale tiles, shape) stands for, in float32."""
    values, tiles, (rows, width) = q
    e = tiles.permute(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, -1)[:rows, :-(-width // BLOCK)].int() - 127
    return _scaled(values.float(), e)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _act(g, name):
    """(act(g), act'(g))."""
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if name == "gelu":
        c = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
        return g * c, c + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5
    r = torch.where(g > 0, g, torch.zeros_like(g))
    if name == "relu":
        return r, (g > 0).to(g.dtype)
    return r * r, 2.0 * r


def _plain_pack(st):
    return {"x": _scaled(*_quantise(st.x)).to(st.x.dtype)}


def _plain_linear(st):
    dt = st.x.dtype
    x, W, dy = st.x.detach().float(), st.W.detach().float(), st.dy.float()
    kept = _scaled(*_quantise(x))
    return {"y": (x @ W.T).to(dt), "dx": (dy @ W).to(dt), "dW": (dy.T @ kept).to(dt)}


def _plain_gated(st):
    c = st.case
    dt = st.x.dtype
    x, Wg, Wu, W2 = (t.detach().float() for t in (st.x, st.Wg, st.Wu, st.W2))
    g, u = x @ Wg.T, x @ Wu.T
    h = _act(g, c["act"])[0] * u
    out = {"y": (h @ W2.T).to(dt)}
    if c["train"]:
        if c["fp8"]:
            x, g, u = (_scaled(*_quantise(t)) for t in (x, g, u))
        else:  # kept in the inputs' type
            g, u = g.to(dt).float(), u.to(dt).float()
        a, da = _act(g, c["act"])
        dy = st.dy.float()
        dh = dy @ W2
        out["dW2"] = (dy.T @ (a * u)).to(dt)
        dg, du = dh * u * da, dh * a
        out["dx"] = (dg @ Wg + du @ Wu).to(dt)
        out["dWg"], out["dWu"] = (dg.T @ x).to(dt), (du.T @ x).to(dt)
    return out


def _plain_fp8mm(st):
    a = _scaled(*_quantise(st.x)) if st.case["plain_a"] else _unblock(st.a)
    return {"y": (a @ _unblock(st.w).T).to(DTYPES[st.case["dtype"]])}


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------
def _own_pack(st):
    import autoresearch2_b200 as sf
    return {"x": sf.fp8_unpack(sf.fp8_pack(st.x), st.x.dtype)}


def _own_linear(st):
    import autoresearch2_b200 as sf
    y = sf.ckpt_linear(st.x, st.W)
    dx, dW = torch.autograd.grad(y, [st.x, st.W], st.dy)
    return {"y": y.detach(), "dx": dx, "dW": dW}


def _own_gated(st):
    import autoresearch2_b200 as sf
    c = st.case
    y = sf.gated_ffn(st.x, st.Wg, st.Wu, st.W2, activation=c["act"], checkpoint="fp8" if c["fp8"] else None)
    out = {"y": y.detach()}
    if c["train"]:
        out["dx"], out["dWg"], out["dWu"], out["dW2"] = torch.autograd.grad(y, st.leaves, st.dy)
    return out


def _own_fp8mm(st):
    import autoresearch2_b200 as sf
    a = st.x if st.case["plain_a"] else sf.Fp8Tensor(*st.a)
    return {"y": sf.fp8_matmul(a, sf.Fp8Tensor(*st.w), out_dtype=DTYPES[st.case["dtype"]])}


def run(state):
    op = state.case["op"]
    if op == "pack":
        return _own_pack(state) if own else _plain_pack(state)
    if op == "linear":
        return _own_linear(state) if own else _plain_linear(state)
    if op == "gated":
        return _own_gated(state) if own else _plain_gated(state)
    return _own_fp8mm(state) if own else _plain_fp8mm(state)


def work(case):
    """Each input read once, each output written once (a gradient among them), what is kept for a backward written and read once."""
    es, R, D = BYTES[case["dtype"]], case["rows"], case["width"]
    kept = 1 + 1 / BLOCK  # bytes an element in 8 bits
    if case["op"] == "pack":
        return {"bytes": R * D * (2 * es + 2 * kept), "flops": 6 * R * D}
    if case["op"] == "linear":
        N = case["out"]
        return {"bytes": es * (2 * (R * D + R * N + N * D)) + 2 * kept * R * D, "flops": 6 * R * D * N}
    if case["op"] == "gated":
        F = case["hidden"]
        if not case["train"]:
            return {"bytes": es * (2 * R * D + 3 * D * F), "flops": 6 * R * D * F}
        state = kept * (R * D + 2 * R * F) if case["fp8"] else es * 2 * R * F
        return {"bytes": es * (4 * R * D + 6 * D * F) + 2 * state, "flops": 18 * R * D * F}
    N = case["out"]
    a = R * D * (es if case["plain_a"] else kept)
    return {"bytes": a + N * D * kept + es * R * N, "flops": 2 * R * N * D}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_kept(x):
    """x [rows, width] (float64) after the 8-bit format: the nearest multiple of the
    step that e4m3 has at x's size (3 bits after the leading one, 2^-9 at least), on
    the block's scale, ties to even."""
    out = torch.empty_like(x)
    for a in range(0, x.shape[1], BLOCK):
        b = x[:, a:a + BLOCK]
        amax = b.abs().max(dim=1, keepdim=True).values
        e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, 448.0)) / 448.0)).clamp(min=LOWEST)
        # log2 may round across an integer: the definition decides
        e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)
        e = torch.where((amax <= 448.0 * torch.exp2(e - 1)) & (e > LOWEST) & (amax > 0), e - 1, e)
        y = b / torch.exp2(e)
        top = torch.frexp(y)[1] - 1
        step = torch.exp2((top.clamp(min=-6) - 3).to(torch.float64))
        out[:, a:a + BLOCK] = torch.round(y / step) * step * torch.exp2(e)
    return out


def _exact_act(g, name):
    if name == "silu":
        return g * torch.sigmoid(g), torch.sigmoid(g) + g * torch.sigmoid(g) * torch.sigmoid(-g)
    if name == "gelu":
        phi = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        return g * phi, phi + g * torch.exp(-g.square() / 2) / math.sqrt(2.0 * math.pi)
    if name == "relu":
        return g.clamp(min=0), (g > 0).to(g.dtype)
    return g.clamp(min=0).square(), 2 * g.clamp(min=0)


def exact(case, seed):
    """What run() returns for these inputs, from the definitions in float64."""
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "pack":
        if s.x.numel() > 1 << 27:  # in parts
            return {"x": torch.cat([_exact_kept(p.to(f8)).to(s.x.dtype) for p in s.x.split(8192)])}
        return {"x": _exact_kept(s.x.to(f8))}
    if case["op"] == "linear":
        x, W, dy = s.x.detach().to(f8), s.W.detach().to(f8), s.dy.to(f8)
        return {"y": x @ W.T, "dx": dy @ W, "dW": dy.T @ _exact_kept(x)}
    if case["op"] == "gated":
        x, Wg, Wu, W2 = (t.detach().to(f8) for t in (s.x, s.Wg, s.Wu, s.W2))
        g, u = x @ Wg.T, x @ Wu.T
        out = {"y": (_exact_act(g, case["act"])[0] * u) @ W2.T}
        if case["train"]:
            if case["fp8"]:
                x, g, u = _exact_kept(x), _exact_kept(g), _exact_kept(u)
            else:
                g, u = (t.to(s.x.dtype).to(f8) for t in (g, u))
            a, da = _exact_act(g, case["act"])
            dy = s.dy.to(f8)
            out["dW2"] = dy.T @ (a * u)
            dh = dy @ W2
            du, dg = dh * a, dh * u * da
            out["dx"] = torch.addmm(dg @ Wg, du, Wu)
            out["dWg"], out["dWu"] = dg.T @ x, du.T @ x
        return out

    def matrix(q):
        values, tiles, (rows, width) = q
        out = values.to(f8)
        for k in range(-(-width // BLOCK)):
            r = torch.arange(rows, device=out.device)
            byte = tiles[r // 128, k // 4, r % 32, r % 128 // 32, k % 4].to(f8)
            out[:, k * BLOCK:(k + 1) * BLOCK] *= torch.exp2(byte - 127)[:, None]
        return out

    a = _exact_kept(s.x.to(f8)) if case["plain_a"] else matrix(s.a)
    return {"y": a @ matrix(s.w).T}
