"""Performance cases of the 8-bit inference and training operators of rns8_b200.quant.

Each case names one operator and its sizes. run() computes it either in plain
torch operations in 32 bits (own = False) or through the package (own = True)
on the same inputs; exact() restates the definition in 64 bits.

Operators:
  linear    y = scaled int8 product of dynamically quantised rows of x with
            quantised weights (+ bias), optionally gated (SiLU(gate) * up)
  norm      x' = x + c * gate * N(y) and h = N(x'): the residual update after
            a block with the norm before the next one
  norm_bwd  the gradients of norm with respect to x, y, both weights and gate
  block     norm with int8 tokens out, gated product, product: the gated MLP
            of a block with the norms in front of it
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
RES_SCALE = 0.5


def listed():
    return [
        # One new token through a square projection: latency of the smallest serving call.
        dict(name="linear 1 token", op="linear", m=1, n=4096, k=4096, dtype="bf16", gated=False, bias=False),
        # A handful of concurrent requests through the gated half of an MLP.
        dict(name="linear gated 5 tokens", op="linear", m=5, n=8192, k=4096, dtype="f16", gated=True, bias=False),
        # A decode batch: the weights' bytes bound it.
        dict(name="linear 64 tokens", op="linear", m=64, n=8192, k=8192, dtype="bf16", gated=False, bias=True),
        # Odd sizes throughout, 32-bit activations: a classifier or adapter head on a ragged chunk.
        dict(name="linear odd f32", op="linear", m=333, n=1001, k=2040, dtype="f32", gated=False, bias=True),
        # A prefill chunk through the gated half of an MLP.
        dict(name="linear gated prefill", op="linear", m=4096, n=8192, k=4096, dtype="bf16", gated=True, bias=False),
        # The largest: a long prefill through a wide projection, bound by the tensor cores.
        dict(name="linear prefill", op="linear", m=8192, n=8192, k=8192, dtype="bf16", gated=False, bias=True),
        # One new token between two blocks.
        dict(name="norm 1 token", op="norm", tokens=1, dim=4096, groups=1, dtype="bf16"),
        # A chunk of odd width in 32 bits, one gate row per token.
        dict(name="norm odd f32", op="norm", tokens=777, dim=1001, groups=777, dtype="f32"),
        # A long prefill with one gate row for each of eight sequences.
        dict(name="norm prefill", op="norm", tokens=8192, dim=8192, groups=8, dtype="bf16"),
        # A small fine-tuning step with a gate for each token.
        dict(name="norm_bwd 250 tokens", op="norm_bwd", tokens=250, dim=2048, groups=250, dtype="f16"),
        # A training step's tokens with learned channel gates.
        dict(name="norm_bwd training", op="norm_bwd", tokens=16384, dim=4096, groups=1, dtype="bf16"),
        # The gated MLP of a block on a decode batch, int8 tokens straight from the norm.
        dict(name="block 48 tokens", op="block", tokens=48, dim=4096, hidden=8192, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width: mostly multiples of 64, sometimes of 8, sometimes any."""
    v = _log_int(rng, low, high)
    step = rng.choice([64, 64, 64, 8, 1])
    return max(low, min(high, v // step * step))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "norm", "norm_bwd", "block"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "linear":
        gated = rng.random() < 0.4
        return dict(op=op, m=_log_int(rng, 1, 8192), n=_width(rng, 256, 4096 if gated else 8192),
                    k=_width(rng, 256, 8192), dtype=dtype, gated=gated, bias=rng.random() < 0.5)
    if op == "block":
        return dict(op=op, tokens=_log_int(rng, 1, 4096), dim=_width(rng, 256, 4096), hidden=_width(rng, 256, 8192),
                    dtype=rng.choice(["bf16", "f16"]))
    tokens = _log_int(rng, 1, 8192)
    divisors = [d for d in range(1, min(tokens, 16) + 1) if tokens % d == 0]
    return dict(op=op, tokens=tokens, dim=_width(rng, 256, 8192), groups=rng.choice([1, tokens, rng.choice(divisors)]),
                dtype=dtype)


def _activations(gen, rows, cols, dtype):
    """Gaussian activations with a few channels far larger than the rest, and
    an all-zero padding row at the end of larger batches."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    channel = torch.rand(cols, generator=gen, device="cuda")
    x *= torch.where(channel > 0.995, 12.0, 0.7 + 0.6 * channel)
    if rows >= 8:
        x[-1] = 0
    return x.to(dtype)


def _int8_weights(gen, n, k):
    """Quantised weights as a checkpoint holds them: int8 rows with one scale
    per output channel."""
    w = torch.empty(n, k, dtype=torch.int8, device="cuda")
    for r in range(0, n, 4096):
        rows = min(4096, n - r)
        w[r:r + rows] = (torch.randn(rows, k, generator=gen, device="cuda") * 40).round_().clamp_(-127, 127).to(torch.int8)
    s = (0.5 + torch.rand(n, generator=gen, device="cuda")) / (40 * math.sqrt(k))
    return w, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    op = case["op"]
    st = dict(op=op, dtype=dt)
    if op == "linear":
        rows = case["n"] * (2 if case["gated"] else 1)
        st["x"] = _activations(gen, case["m"], case["k"], dt)
        st["w"], st["ws"] = _int8_weights(gen, rows, case["k"])
        st["bias"] = torch.randn(rows, generator=gen, device="cuda") if case["bias"] else None
        st["gated"] = case["gated"]
        return st
    t, d = case["tokens"], case["dim"]
    g = case.get("groups", 1)
    st["y"] = _activations(gen, t, d, dt)
    st["post"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dt)
    st["pre"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dt)
    st["gate"] = (0.6 + 0.3 * torch.randn(g, d, generator=gen, device="cuda")).to(dt)
    st["x"] = _activations(gen, t, d, dt)
    if op == "norm_bwd":
        st["dx"] = torch.randn(t, d, generator=gen, device="cuda").to(dt)
        st["dh"] = torch.randn(t, d, generator=gen, device="cuda").to(dt)
        if t >= 8:  # the padding row takes no part in the loss
            st["dx"][-1] = 0
            st["dh"][-1] = 0
    if op == "block":
        st["w1"], st["s1"] = _int8_weights(gen, 2 * case["hidden"], d)
        st["w2"], st["s2"] = _int8_weights(gen, d, case["hidden"])
    return st


def run(st):
    return _run_own(st) if own else _run_plain(st)


# ---- the package's operators ---------------------------------------------------
def _run_own(st):
    from rns8_b200 import quant

    op = st["op"]
    if op == "linear":
        return quant.linear(st["x"], st["w"], st["ws"], bias=st["bias"], gated=st["gated"])
    if op == "norm":
        return quant.residual_norm(st["x"], st["y"], post_weight=st["post"], pre_weight=st["pre"], gate=st["gate"],
                                   scale=RES_SCALE, eps=EPS)
    if op == "norm_bwd":
        return quant.residual_norm_backward(st["dx"], st["dh"], st["x"], st["y"], post_weight=st["post"],
                                            pre_weight=st["pre"], gate=st["gate"], scale=RES_SCALE, eps=EPS)
    x, q, s = quant.residual_norm_quantized(st["x"], st["y"], post_weight=st["post"], pre_weight=st["pre"],
                                            gate=st["gate"], scale=RES_SCALE, eps=EPS)
    h = quant.gemm_scaled(q, s, st["w1"], st["s1"], gated=True, out_dtype=st["dtype"])
    return x, quant.linear(h, st["w2"], st["s2"])


# ---- plain forms: elementary torch operations in 32 bits -------------------------
def _plain_quantize(x):
    amax = x.abs().amax(dim=1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    q = torch.where(amax > 0, torch.round(x * (torch.full_like(amax, 127.0) / amax)), torch.zeros_like(x))
    return q, scale


def _plain_product(q, scale, w, ws, bias, gated):
    y = (q @ w.float().t()) * scale * ws
    if bias is not None:
        y = y + bias
    if gated:
        g, u = y.chunk(2, dim=1)
        y = g / (1 + torch.exp(-g)) * u
    return y


def _plain_norm(st):
    x, y = st["x"].float(), st["y"].float()
    gate = st["gate"].float().repeat_interleave(x.shape[0] // st["gate"].shape[0], dim=0)
    p = y * torch.rsqrt((y * y).mean(dim=1, keepdim=True) + EPS) * st["post"].float()
    xo = x + RES_SCALE * gate * p
    h = xo * torch.rsqrt((xo * xo).mean(dim=1, keepdim=True) + EPS) * st["pre"].float()
    return xo, h


def _plain_norm_bwd(st):
    x, y, dx, dh = st["x"].float(), st["y"].float(), st["dx"].float(), st["dh"].float()
    groups = st["gate"].shape[0]
    gate = st["gate"].float().repeat_interleave(x.shape[0] // groups, dim=0)
    post, pre = st["post"].float(), st["pre"].float()
    rho = torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS)
    n = x * rho
    t = dh * pre
    dr = dx + rho * (t - n * (t * n).mean(dim=1, keepdim=True))
    sigma = torch.rsqrt((y * y).mean(dim=1, keepdim=True) + EPS)
    u = y * sigma
    dp = RES_SCALE * gate * dr
    v = dp * post
    dy = sigma * (v - u * (v * u).mean(dim=1, keepdim=True))
    dgate = (RES_SCALE * u * post * dr).view(groups, -1, x.shape[1]).sum(dim=1)
    return dr, dy, (u * dp).sum(dim=0), (dh * n).sum(dim=0), dgate


def _run_plain(st):
    dt, op = st["dtype"], st["op"]
    if op == "linear":
        q, scale = _plain_quantize(st["x"].float())
        return _plain_product(q, scale, st["w"], st["ws"], st["bias"], st["gated"]).to(dt)
    if op == "norm":
        xo, h = _plain_norm(st)
        return xo.to(dt), h.to(dt)
    if op == "norm_bwd":
        dx, dy, dpost, dpre, dgate = _plain_norm_bwd(st)
        # Gradients that are summed over tokens stay in 32 bits; a gate of one
        # row per token has its gradient in the activations' type.
        per_token = st["gate"].shape[0] == st["x"].shape[0]
        return dx.to(dt), dy.to(dt), dpost, dpre, dgate.to(dt) if per_token else dgate
    xo, h = _plain_norm(st)
    q, scale = _plain_quantize(h)
    h = _plain_product(q, scale, st["w1"], st["s1"], None, True)
    q, scale = _plain_quantize(h)
    return xo.to(dt), _plain_product(q, scale, st["w2"], st["s2"], None, False).to(dt)


# ---- the definitions in 64 bits -------------------------------------------------
def _exact_linear(x, w, ws, bias, gated):
    top = x.abs().max(dim=1).values.clamp_min(1e-300)
    q = torch.round(x / top[:, None] * 127)
    y = torch.einsum("mk,nk->mn", q, w.double()) * torch.outer(top / 127, ws.double())
    y = y if bias is None else y + bias.double()[None, :]
    if gated:
        half = y.shape[1] // 2
        y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    return y


def _exact_rms(v):
    return v / torch.sqrt(v.square().mean(dim=1, keepdim=True) + EPS)


def exact(case, seed):
    st = prepare(case, seed)
    if st["op"] == "linear":
        return _exact_linear(st["x"].double(), st["w"], st["ws"], st["bias"], st["gated"])
    x, y, gate = st["x"].double(), st["y"].double(), st["gate"].double()
    post, pre = st["post"].double(), st["pre"].double()
    which = torch.arange(x.shape[0], device="cuda") // (x.shape[0] // gate.shape[0])
    if st["op"] == "norm_bwd":
        # x is the updated residual here; its gradient reaches the block's
        # output through x + c * gate * N(y), whose derivative autograd takes.
        x.requires_grad_(), pre.requires_grad_()
        h = _exact_rms(x) * pre
        dr, dpre = torch.autograd.grad([h, x * 1.0], [x, pre], [st["dh"].double(), st["dx"].double()])
        y.requires_grad_(), post.requires_grad_(), gate.requires_grad_()
        update = RES_SCALE * gate[which] * (_exact_rms(y) * post)
        dy, dpost, dgate = torch.autograd.grad(update, [y, post, gate], dr)
        return dr, dy, dpost, dpre, dgate
    xo = x + RES_SCALE * gate[which] * (_exact_rms(y) * post)
    h = _exact_rms(xo) * pre
    if st["op"] == "norm":
        return xo, h
    h = _exact_linear(h, st["w1"], st["s1"], None, True)
    return xo, _exact_linear(h, st["w2"], st["s2"], None, False)


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    op = case["op"]
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        rows = n * (2 if case["gated"] else 1)
        return {"bytes": m * k * size + rows * k + 4 * rows * (2 if case["bias"] else 1) + m * n * size,
                "flops": 2 * m * rows * k}
    t, d = case["tokens"], case["dim"]
    g = case.get("groups", 1)
    params = (2 + g) * d * size
    if op == "norm":
        return {"bytes": 4 * t * d * size + params, "flops": 12 * t * d}
    if op == "norm_bwd":
        grads = 8 * d + g * d * (size if g == t else 4)
        return {"bytes": 6 * t * d * size + params + grads, "flops": 30 * t * d}
    f = case["hidden"]
    return {"bytes": 4 * t * d * size + params + 3 * d * f + 4 * (2 * f + d), "flops": 6 * t * d * f}
