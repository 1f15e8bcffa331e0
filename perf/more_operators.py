"""Workloads of the 8-bit floating-point linear (a power-of-two scale for each block of 128), of the AdamW step over many
tensors at once with its moments in 32 bits or in 8, and of the gradient norm that clips it.

Each case has a plain form in elementary torch operations (32-bit arithmetic, rounded once at the end), the call that a
program makes of ``convrot_mlx_b200``, and the definition in 64 bits.  ``own`` selects between the first two.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
SPAN = 128  # values of a token, rows and columns of a weight, that share one scale
TOP = 448.0  # the largest value of an 8-bit float with 4 exponent and 3 mantissa bits
BLOCK = 256  # values of a tensor whose 8-bit moments share their scales
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.99, 1e-8, 0.01


# ---------------------------------------------------------------------------
# cases


def listed():
    return [
        # the projection of one conditioning vector: latency, the weights are all that is read
        dict(name="fp8 linear, 1 token", op="fp8", m=1, k=5120, n=5120, dtype="bf16", bias=True, train=False),
        # a prompt through a layer whose sizes are no multiple of anything
        dict(name="fp8 linear, ragged", op="fp8", m=451, k=2203, n=1301, dtype="f16", bias=True, train=False),
        # the first MLP projection of a video transformer block
        dict(name="fp8 linear, 7800 tokens", op="fp8", m=7800, k=5120, n=13824, dtype="bf16", bias=True, train=False),
        # an attention projection in fine-tuning: output and gradient of the input, the weights frozen
        dict(name="fp8 linear, training", op="fp8", m=1536, k=5120, n=5120, dtype="bf16", bias=True, train=True),
        # the norms and biases of one block: latency
        dict(name="AdamW, few vectors", op="adamw", tensors="4*64,2*768", dtype="f32", bits=32, step=100, clip=0.0),
        # the modulations of eight blocks in full precision
        dict(name="AdamW, modulations", op="adamw", tensors="8*9216x1536,8*9216", dtype="f32", bits=32, step=1000, clip=1.0),
        # low-rank adapters around every linear of forty blocks: many tensors
        dict(name="AdamW, 8-bit adapters", op="adamw", tensors="280*16x5120,240*5120x16,40*13824x16,40*16x13824,40*5120x16",
             dtype="f32", bits=8, step=20, clip=1.0),
        # a whole block trained in 16 bits
        dict(name="AdamW, 8-bit block", op="adamw", tensors="4*5120x5120,13824x5120,5120x13824", dtype="bf16", bits=8, step=300, clip=0.0),
        # sizes that are no multiple of anything, the first step
        dict(name="AdamW, 8-bit odd", op="adamw", tensors="7*1153x333,5*77,3*1,1499", dtype="bf16", bits=8, step=1, clip=0.5),
        # the gradients of the adapters
        dict(name="gradient norm, adapters", op="norm", tensors="280*16x5120,240*5120x16,40*13824x16,40*16x13824,40*5120x16", dtype="f32"),
        # the gradients of a block
        dict(name="gradient norm, block", op="norm", tensors="4*5120x5120,13824x5120,5120x13824", dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_fp8(rng):
    return dict(op="fp8", m=_log_uniform(rng, 1, 16384), k=_log_uniform(rng, 64, 15360), n=_log_uniform(rng, 32, 15360),
                dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), bias=rng.random() < 0.7, train=rng.random() < 0.4)


def _draw_tensors(rng):
    parts = []
    for _ in range(rng.choice([1, 1, 2, 3])):
        count, rows = _log_uniform(rng, 1, 200), _log_uniform(rng, 1, 16384)
        shape = str(rows) if rng.random() < 0.3 else "%dx%d" % (rows, _log_uniform(rng, 1, 4096))
        parts.append("%d*%s" % (count, shape))
    return ",".join(parts)


def _draw_adamw(rng):
    return dict(op="adamw", tensors=_draw_tensors(rng), dtype=rng.choice(["bf16", "f16", "f32", "f32"]),
                bits=rng.choice([8, 8, 32]), step=_log_uniform(rng, 1, 100000), clip=rng.choice([0.0, 0.5, 1.0]))


def _draw_norm(rng):
    return dict(op="norm", tensors=_draw_tensors(rng), dtype=rng.choice(["bf16", "f16", "f32", "f32"]))


def draw(rng):
    """A case of the listed ranges that costs no more than the largest listed one of its operator."""

    op = rng.choice(["fp8", "adamw", "norm"])
    top = [work(c) for c in listed() if c["op"] == op]
    make = {"fp8": _draw_fp8, "adamw": _draw_adamw, "norm": _draw_norm}[op]
    while True:
        case = make(rng)
        w = work(case)
        if all(0 < w[what] <= max(t[what] for t in top) for what in ("bytes", "flops")):
            return case


def _shapes(case):
    """The tensors' shapes: "3*5x7,9" are three of (5, 7) and one of (9,)."""

    shapes = []
    for part in case["tensors"].split(","):
        count, _, shape = part.rpartition("*")
        shapes += [tuple(int(s) for s in shape.split("x"))] * int(count or 1)
    return shapes


def work(case):
    """The bytes that the inputs and outputs of one pass take, each moved once, and its arithmetic operations."""

    e = SIZE[case["dtype"]]
    if case["op"] == "fp8":
        m, k, n = case["m"], case["k"], case["n"]
        ways = 2 if case["train"] else 1
        scales = -(-n // SPAN) * -(-k // SPAN)
        return {"bytes": ways * e * m * (k + n) + n * k + scales + (4 * n if case["bias"] else 0), "flops": 2 * ways * m * n * k}
    values = sum(math.prod(s) for s in _shapes(case))
    if case["op"] == "norm":
        return {"bytes": e * values, "flops": 2 * values}
    moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK  # read and written
    return {"bytes": int((3 * e + moments) * values), "flops": (18 if case["clip"] else 15) * values}


# ---------------------------------------------------------------------------
# inputs


def _activation(shape, dtype, g):
    """Normal values with one channel in a hundred twenty times larger, as the inputs of a DiT's linears."""

    x = torch.randn(shape, generator=g, device="cuda")
    wide = torch.rand(shape[-1], generator=g, device="cuda") < 0.01
    return (x * torch.where(wide, 20.0, 1.0)).to(dtype)


def _exponent(top):
    """The least e with top <= 448 * 2^e, for magnitudes ``top`` in float32; -127 for zeros."""

    fraction, exponent = torch.frexp(top)  # top = fraction * 2^exponent, fraction in [1/2, 1)
    e = exponent - 9 + (fraction > TOP / 512).to(torch.int32)
    return torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127)


def _scales(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _weight(w):
    """8-bit codes of blocks of 128 x 128, on rows of a pitch that is a multiple of 16 bytes, and the blocks' scales."""

    n, k = w.shape
    blocks = torch.nn.functional.pad(w, (0, -k % SPAN, 0, -n % SPAN)).unflatten(1, (-1, SPAN)).unflatten(0, (-1, SPAN))
    e = _exponent(blocks.abs().amax(dim=(1, 3)))
    codes = torch.ldexp(blocks, -e[:, None, :, None]).flatten(0, 1).flatten(1)[:n, :k]
    rows = torch.zeros((n, -(-k // 16) * 16), dtype=torch.float8_e4m3fn, device="cuda")
    rows[:, :k] = codes.to(torch.float8_e4m3fn)
    return rows[:, :k], _scales(e)


def _views(flat, shapes, starts):
    return [flat[at:at + math.prod(s)].view(s) for s, at in zip(shapes, starts)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "fp8":
        m, k, n = case["m"], case["k"], case["n"]
        # channels of different strength, as trained weights have
        w = torch.randn((n, k), generator=g, device="cuda") * torch.rand((n, 1), generator=g, device="cuda") * 0.04
        qweight, wscales = _weight(w)
        state.update(x=_activation((m, k), dtype, g).requires_grad_(case["train"]), qweight=qweight, wscales=wscales,
                     bias_values=torch.randn(n, generator=g, device="cuda") * 0.01 if case["bias"] else None)
        if case["train"]:
            state["dy"] = (torch.randn((m, n), generator=g, device="cuda") * 0.1).to(dtype)
        return state
    # Tensors one after another in a flat buffer, as gradients are kept for their exchange; each starts on a multiple of 256 values.
    shapes = _shapes(case)
    starts, total = [], 0
    for s in shapes:
        starts.append(total)
        total += -(-math.prod(s) // BLOCK) * BLOCK
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for s, at in zip(shapes, starts):
        inside[at:at + math.prod(s)] = True
    strength = torch.exp(torch.randn(total, generator=g, device="cuda") * 1.5 - 5.0)  # of each value's gradient
    strength.masked_fill_(~inside, 0.0)
    state["grads"] = (torch.randn(total, generator=g, device="cuda") * strength).to(dtype)
    state["grad_views"] = _views(state["grads"], shapes, starts)
    if case["op"] == "norm":
        return state
    state["params"] = torch.randn(total, generator=g, device="cuda").mul_(0.02).masked_fill_(~inside, 0.0).to(dtype)
    state["step"] = case["step"]
    first = case["step"] == 1
    exp_avg = torch.randn(total, generator=g, device="cuda") * strength * 0.3 * (not first)
    root = strength * (0.5 + torch.rand(total, generator=g, device="cuda")) * math.sqrt(1 - BETA2 ** (case["step"] - 1))
    if case["bits"] == 32:
        state.update(exp_avg=exp_avg, exp_avg_sq=root * root)
    else:
        pairs = torch.stack((exp_avg, root)).view(2, -1, BLOCK)
        scales = pairs.abs().amax(dim=-1) / TOP
        codes = torch.where(scales[..., None] > 0, pairs / scales[..., None], torch.zeros_like(pairs)).to(torch.float8_e4m3fn)
        state.update(exp_avg=codes[0].reshape(-1).clone(), exp_avg_sq=codes[1].reshape(-1).clone(), scales=scales.T.contiguous())
        state["scale_views"] = [state["scales"][at // BLOCK:at // BLOCK - (-math.prod(s) // BLOCK)] for s, at in zip(shapes, starts)]
    for name, views in (("params", "param_views"), ("exp_avg", "exp_avg_views"), ("exp_avg_sq", "exp_avg_sq_views")):
        state[views] = _views(state[name], shapes, starts)
    return state


# ---------------------------------------------------------------------------
# the plain forms, in 32 bits


def _dequantized(x):
    """x (32 bits) as 8-bit codes with one power-of-two scale for each 128 values of a row give it back."""

    k = x.shape[1]
    blocks = torch.nn.functional.pad(x, (0, -k % SPAN)).unflatten(1, (-1, SPAN))
    e = _exponent(blocks.abs().amax(dim=-1, keepdim=True))
    codes = torch.ldexp(blocks, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(codes, e).flatten(1)[:, :k]


def _plain_fp8(s):
    n, k = s["qweight"].shape
    scales = s["wscales"].float().repeat_interleave(SPAN, 0)[:n].repeat_interleave(SPAN, 1)[:, :k]
    w = s["qweight"].float() * scales
    y = _dequantized(s["x"].float()) @ w.T
    if s["bias_values"] is not None:
        y = y + s["bias_values"]
    out = {"y": y.to(s["x"].dtype)}
    if s["train"]:
        out["dx"] = (_dequantized(s["dy"].float()) @ w).to(s["x"].dtype)
    return out


def _plain_grad_norm(grads):
    return grads.double().square().sum().sqrt().float()


def _to_codes(blocks, scales):
    q = blocks / scales
    return torch.where(scales > 0, q, torch.zeros_like(q))


def _plain_adamw(s):
    g = s["grads"].float()
    out = {}
    if s["clip"]:
        out["norm"] = _plain_grad_norm(s["grads"])
        g = g * torch.clamp(s["clip"] / (out["norm"] + 1e-6), max=1.0)
    correct1, correct2 = 1 - BETA1 ** s["step"], 1 - BETA2 ** s["step"]
    s["step"] += 1
    if s["bits"] == 32:
        s["exp_avg"].mul_(BETA1).add_(g * (1 - BETA1))
        s["exp_avg_sq"].mul_(BETA2).add_(g * g * (1 - BETA2))
        m, r = s["exp_avg"], s["exp_avg_sq"].sqrt()
    else:
        m_scale, r_scale = s["scales"][:, :1], s["scales"][:, 1:]
        m = s["exp_avg"].float().view(-1, BLOCK) * m_scale * BETA1 + g.view(-1, BLOCK) * (1 - BETA1)
        r = s["exp_avg_sq"].float().view(-1, BLOCK) * r_scale
        r = (r * r * BETA2 + (g * g * (1 - BETA2)).view(-1, BLOCK)).sqrt()
        m_scale, r_scale = m.abs().amax(dim=1, keepdim=True) / TOP, r.amax(dim=1, keepdim=True) / TOP
        s["exp_avg"].copy_(_to_codes(m, m_scale).to(torch.float8_e4m3fn).view(-1))
        # a root that is not zero stays so: it divides
        code = torch.where(r > 0, _to_codes(r, r_scale).clamp(min=2.0 ** -9), r)
        s["exp_avg_sq"].copy_(code.to(torch.float8_e4m3fn).view(-1))
        s["scales"].copy_(torch.cat((m_scale, r_scale), dim=1))
        m, r = m.view(-1), r.view(-1)
        out["scales"] = s["scales"]
    p = s["params"].float() * (1 - LR * DECAY) - (LR / correct1) * m / (r / math.sqrt(correct2) + EPS)
    s["params"].copy_(p)
    return {**out, "params": s["params"], "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"]}


def _plain_norm(s):
    return {"norm": _plain_grad_norm(s["grads"])}


# ---------------------------------------------------------------------------
# the calls of a program


def _own_fp8(s):
    from convrot_mlx_b200 import fp8_linear

    y = fp8_linear(s["x"], s["qweight"], s["wscales"], s["bias_values"])
    if not s["train"]:
        return {"y": y}
    return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}


def _own_adamw(s):
    from convrot_mlx_b200 import adamw_step

    norm = adamw_step(s["param_views"], s["grad_views"], s["exp_avg_views"], s["exp_avg_sq_views"], s.get("scale_views"), s["step"],
                      lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, max_norm=s["clip"] or None)
    s["step"] += 1
    out = {name: s[name] for name in ("params", "exp_avg", "exp_avg_sq")}
    if s["bits"] == 8:
        out["scales"] = s["scales"]
    if s["clip"]:
        out["norm"] = norm
    return out


def _own_norm(s):
    from convrot_mlx_b200 import grad_norm

    return {"norm": grad_norm(s["grad_views"])}


def run(state):
    op = state["op"]
    if own:
        return {"fp8": _own_fp8, "adamw": _own_adamw, "norm": _own_norm}[op](state)
    with torch.no_grad():
        return {"fp8": _plain_fp8, "adamw": _plain_adamw, "norm": _plain_norm}[op](state)


# ---------------------------------------------------------------------------
# the definitions, in 64 bits


def _e4m3(v):
    """v (64 bits) rounded to the nearest value of an 8-bit float: 4 significant bits down to 2^-6, then steps of 2^-9."""

    quantum = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / quantum) * quantum


def _exact_blocks(x):
    """x (64 bits) through 8-bit codes and power-of-two scales for each 128 values of a row."""

    out = torch.empty_like(x)
    for at in range(0, x.shape[1], SPAN):
        part = x[:, at:at + SPAN]
        top = part.abs().max(dim=1, keepdim=True).values
        scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -110) / TOP)))
        out[:, at:at + SPAN] = _e4m3(part / scale) * scale
    return out


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        if case["op"] == "fp8":
            n, k = s["qweight"].shape
            w = s["qweight"].double()
            for i, row in enumerate(s["wscales"].float().double()):
                w[i * SPAN:(i + 1) * SPAN] *= torch.repeat_interleave(row, SPAN)[:k]
            y = torch.einsum("mk,nk->mn", _exact_blocks(s["x"].double()), w)
            y = y + s["bias_values"].double() if case["bias"] else y
            return {"y": y, "dx": torch.einsum("mn,nk->mk", _exact_blocks(s["dy"].double()), w)} if case["train"] else {"y": y}
        g = s["grads"].double()
        norm = torch.linalg.vector_norm(g)
        if case["op"] == "norm":
            return {"norm": norm}
        out = {}
        if case["clip"]:
            out["norm"] = norm
            g = g * min(1.0, case["clip"] / (norm.item() + 1e-6))
        t = case["step"]
        if case["bits"] == 32:
            m = torch.lerp(g, s["exp_avg"].double(), BETA1)
            v = torch.lerp(g ** 2, s["exp_avg_sq"].double(), BETA2)
            out.update(exp_avg=m, exp_avg_sq=v)
        else:
            old = [s[name].double().reshape(-1, BLOCK) * s["scales"].double()[:, i, None] for i, name in enumerate(("exp_avg", "exp_avg_sq"))]
            m = torch.lerp(g, old[0].reshape(-1), BETA1)
            v = torch.lerp(g ** 2, old[1].reshape(-1) ** 2, BETA2)
            codes, tops = [], []
            for x in (m, v ** 0.5):
                x = x.reshape(-1, BLOCK)
                top = torch.linalg.vector_norm(x, ord=math.inf, dim=1, keepdim=True)
                code = _e4m3((x * TOP / top).nan_to_num(0.0))
                codes.append(code.reshape(-1))
                tops.append(top[:, 0] / TOP)
            codes[1] = torch.where((v > 0) & (codes[1] == 0), 2.0 ** -9, codes[1])
            out.update(exp_avg=codes[0], exp_avg_sq=codes[1], scales=torch.stack(tops, dim=1))
        ratio = (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
        p = s["params"].double()
        out["params"] = p - LR * DECAY * p - LR * ratio
        return out
