"""Workloads of the 8-bit and training operators: the 8-bit linear, rotary positions with several axes, layer norm with
its gradients, and the GELU whose saved input is held in 8 bits.

Each case has a plain form in elementary torch operations (32-bit arithmetic, rounded once at the end), the call that a
program makes of ``convrot_mlx_b200``, and the definition in 64 bits.  ``own`` selects between the first two.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
GROUP = 128  # features that share one scale in the saved input of the GELU
GELU_C = math.sqrt(2.0 / math.pi)
GELU_A = 0.044715


# ---------------------------------------------------------------------------
# cases


def listed():
    return [
        # a modulation or adapter projection of one sample: latency, the weights are all that is read
        dict(name="int8 linear, 1 token", op="int8", m=1, k=4096, n=4096, dtype="bf16", bias=True, train=False),
        # a short prompt through a layer whose sizes are no multiple of anything
        dict(name="int8 linear, ragged", op="int8", m=333, k=1997, n=1211, dtype="f16", bias=True, train=False),
        # the first MLP projection of a DiT block over one large image
        dict(name="int8 linear, 4096 tokens", op="int8", m=4096, k=3072, n=12288, dtype="bf16", bias=True, train=False),
        # the same block's attention projection in fine-tuning: output and gradient of the input, the weights frozen
        dict(name="int8 linear, training", op="int8", m=1536, k=3072, n=3072, dtype="bf16", bias=True, train=True),
        # the text-to-image attention of the DiT at batch 8: text at the origin, image tokens on a square grid
        dict(name="rotary, image", op="rotary", batch=8, text=512, frames=1, rows=32, cols=32, at=0, heads=24, kv=24, dim=128,
             axes="16,56,56", theta=10000.0, adjacent=True, dtype="bf16", train=False),
        # one token in the middle of a picture: latency
        dict(name="rotary, 1 token", op="rotary", batch=1, text=0, frames=1, rows=1, cols=1, at=37, heads=24, kv=8,
             dim=128, axes="16,56,56", theta=10000.0, adjacent=True, dtype="bf16", train=False),
        # video in fine-tuning: odd grid, shared key heads, pairs half a head apart, the head's tail not rotated
        dict(name="rotary, video training", op="rotary", batch=1, text=77, frames=13, rows=30, cols=45, at=0, heads=20,
             kv=4, dim=128, axes="32,40,40", theta=10000.0, adjacent=False, dtype="f16", train=True),
        # the norms before a small conditioning head
        dict(name="layer norm, small", op="norm", batch=1, rows=8, features=768, dtype="bf16", form="affine", train=False),
        # the modulated norm of a DiT block in fine-tuning, one scale and shift for each sample
        dict(name="layer norm, modulated training", op="norm", batch=8, rows=1536, features=3072, dtype="bf16",
             form="modulated", train=True),
        # odd sizes in 32 bits
        dict(name="layer norm, odd training", op="norm", batch=1, rows=5003, features=1153, dtype="f32", form="affine",
             train=True),
        # the MLP of a text stream, odd width
        dict(name="gelu, odd training", op="gelu", rows=500, features=4100, dtype="f16", train=True),
        # the MLP of all tokens of a batch: the largest tensor that a block saves
        dict(name="gelu, block training", op="gelu", rows=12288, features=12288, dtype="bf16", train=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_int8(rng):
    return dict(op="int8", m=_log_uniform(rng, 1, 8192), k=_log_uniform(rng, 64, 15360), n=_log_uniform(rng, 32, 15360),
                dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), bias=rng.random() < 0.7, train=rng.random() < 0.4)


def _draw_rotary(rng):
    adjacent = rng.random() < 0.5
    dim = rng.choice([64, 96, 128, 128, 256])
    widths = [2 * max(1, dim // 12), 2 * (dim // 6), 2 * (dim // 6)]
    if rng.random() < 0.3:
        widths = widths[1:]
    kv = rng.choice([1, 2, 4, 8])
    return dict(op="rotary", batch=rng.choice([1, 1, 2, 3, 4]), text=_log_uniform(rng, 1, 513) - (rng.random() < 0.2),
                frames=rng.choice([1, 1, 5, 9, 16]), rows=_log_uniform(rng, 1, 64), cols=_log_uniform(rng, 1, 64),
                at=rng.choice([0, 0, rng.randrange(64)]), heads=kv * rng.choice([1, 2, 3, 5]), kv=kv, dim=dim, axes=",".join(str(w) for w in widths),
                theta=rng.choice([256.0, 10000.0, 10000.0]), adjacent=adjacent,
                dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), train=rng.random() < 0.5)


def _draw_norm(rng):
    return dict(op="norm", batch=rng.choice([1, 2, 3, 8]), rows=_log_uniform(rng, 1, 16384),
                features=_log_uniform(rng, 32, 16384), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                form=rng.choice(["affine", "modulated"]), train=rng.random() < 0.6)


def _draw_gelu(rng):
    return dict(op="gelu", rows=_log_uniform(rng, 1, 16384), features=_log_uniform(rng, 32, 16384),
                dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), train=True)


def draw(rng):
    """A case of the listed ranges that costs no more than the largest listed one of its operator."""

    op = rng.choice(["int8", "rotary", "norm", "gelu"])
    top = [work(c) for c in listed() if c["op"] == op]
    make = {"int8": _draw_int8, "rotary": _draw_rotary, "norm": _draw_norm, "gelu": _draw_gelu}[op]
    while True:
        case = make(rng)
        w = work(case)
        if all(0 < w[what] <= max(t[what] for t in top) for what in ("bytes", "flops")):
            return case


def _tokens(case):
    return case["text"] + case["frames"] * case["rows"] * case["cols"]


def work(case):
    """The bytes that the inputs and outputs of one pass take, each moved once, and its arithmetic operations."""

    e = SIZE[case["dtype"]]
    if case["op"] == "int8":
        m, k, n = case["m"], case["k"], case["n"]
        vectors = 4 * n * (2 if case["bias"] else 1)
        ways = 2 if case["train"] else 1
        return {"bytes": ways * e * m * (k + n) + n * k + vectors, "flops": 2 * ways * m * n * k}
    if case["op"] == "rotary":
        ways = 2 if case["train"] else 1
        tokens, axes = _tokens(case), case["axes"].count(",") + 1
        values = case["batch"] * tokens * (case["heads"] + case["kv"]) * case["dim"]
        return {"bytes": ways * 2 * e * values + 4 * tokens * axes, "flops": ways * 3 * values}
    values = case["rows"] * case["features"]
    if case["op"] == "norm":
        values *= case["batch"]
        vectors = 2 * case["features"] * (case["batch"] if case["form"] == "modulated" else 1)
        return {"bytes": e * ((4 if case["train"] else 2) * values + (2 if case["train"] else 1) * vectors),
                "flops": (22 if case["train"] else 8) * values}
    return {"bytes": 4 * e * values, "flops": 40 * values}


# ---------------------------------------------------------------------------
# inputs


def _activation(shape, dtype, g):
    """Normal values with one channel in a hundred twenty times larger, as the inputs of a DiT's linears."""

    x = torch.randn(shape, generator=g, device="cuda")
    wide = torch.rand(shape[-1], generator=g, device="cuda") < 0.01
    return (x * torch.where(wide, 20.0, 1.0)).to(dtype)


def _axis_positions(case):
    """(tokens, axes) float32: text tokens at the origin, then the grid of frames, rows and columns, each from ``at`` on."""

    count = case["axes"].count(",") + 1
    grid = torch.cartesian_prod(*(torch.arange(case[a], device="cuda") for a in ("frames", "rows", "cols")))
    grid = grid.reshape(-1, 3)[:, 3 - count:].float()
    return torch.cat((torch.zeros((case["text"], count), device="cuda"), grid + case["at"]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "int8":
        m, k, n = case["m"], case["k"], case["n"]
        w = torch.randn((n, k), generator=g, device="cuda") * 0.02
        top = w.abs().amax(dim=1, keepdim=True)
        # 8-bit weights as they are kept: rows of k codes on a pitch that is a multiple of 16 bytes
        rows = torch.zeros((n, -(-k // 16) * 16), dtype=torch.int8, device="cuda")
        rows[:, :k] = torch.round(w * 127 / top).to(torch.int8)
        state.update(x=_activation((m, k), dtype, g).requires_grad_(case["train"]), qweight=rows[:, :k],
                     wscales=(top[:, 0] / 127).contiguous(),
                     bias_values=torch.randn(n, generator=g, device="cuda") * 0.01 if case["bias"] else None)
        if case["train"]:
            state["dy"] = (torch.randn((m, n), generator=g, device="cuda") * 0.1).to(dtype)
    elif case["op"] == "rotary":
        b, t, d, heads, kv = case["batch"], _tokens(case), case["dim"], case["heads"], case["kv"]
        # the output of a fused projection: for each token all query heads, then the key and the value heads
        qkv = torch.randn((b, t, heads + 2 * kv, d), generator=g, device="cuda").to(dtype)
        state.update(q=qkv[:, :, :heads].transpose(1, 2).requires_grad_(case["train"]),
                     k=qkv[:, :, heads:heads + kv].transpose(1, 2).requires_grad_(case["train"]),
                     positions=_axis_positions(case), widths=tuple(int(w) for w in case["axes"].split(",")))
        if case["train"]:
            state["dq"] = torch.randn((b, heads, t, d), generator=g, device="cuda").to(dtype)
            state["dk"] = torch.randn((b, kv, t, d), generator=g, device="cuda").to(dtype)
    elif case["op"] == "norm":
        b, r, f = case["batch"], case["rows"], case["features"]
        x = _activation((b, r, f), torch.float32, g) * (0.5 + torch.rand((b, r, 1), generator=g, device="cuda"))
        x = (x + torch.randn((b, r, 1), generator=g, device="cuda")).to(dtype).requires_grad_(case["train"])
        shape = (b, 1, f) if case["form"] == "modulated" else (f,)
        scale = torch.randn(shape, generator=g, device="cuda") * 0.2
        state.update(x=x, scale=(scale if case["form"] == "modulated" else 1 + scale).to(dtype),
                     shift=(torch.randn(shape, generator=g, device="cuda") * 0.2).to(dtype))
        if case["train"]:
            state["scale"].requires_grad_()
            state["shift"].requires_grad_()
            state["dy"] = torch.randn((b, r, f), generator=g, device="cuda").to(dtype)
    else:
        r, f = case["rows"], case["features"]
        state.update(x=(torch.randn((r, f), generator=g, device="cuda") * 1.5).to(dtype).requires_grad_(),
                     dy=torch.randn((r, f), generator=g, device="cuda").to(dtype))
    return state


# ---------------------------------------------------------------------------
# the plain forms, in 32 bits


def _codes(x):
    """8-bit codes of the rows of x (as 32-bit values) and their scales: the largest magnitude becomes 127."""

    top = x.abs().amax(dim=-1, keepdim=True)
    codes = torch.where(top > 0, torch.round(x * 127 / top), torch.zeros_like(x))
    return codes, top / 127


def _plain_int8(s):
    codes, scales = _codes(s["x"].float())
    w = s["qweight"].float()
    y = (codes @ w.T) * scales * s["wscales"]
    if s["bias_values"] is not None:
        y = y + s["bias_values"]
    out = {"y": y.to(s["x"].dtype)}
    if s["train"]:
        codes, scales = _codes(s["dy"].float() * s["wscales"])
        out["dx"] = ((codes @ w) * scales).to(s["x"].dtype)
    return out


def _rotate(x, cos, sin, pairs, adjacent):
    """The pairs of the head dimension of x turned by the angles; what follows them is kept."""

    xf = x.float()
    turned, rest = xf[..., :2 * pairs], xf[..., 2 * pairs:]
    if adjacent:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((y, rest), dim=-1).to(x.dtype)


def _angles(s):
    parts = [s["positions"][:, a, None] * (s["theta"] ** (torch.arange(0, w, 2, device="cuda", dtype=torch.float32) * (-1.0 / w)))
             for a, w in enumerate(s["widths"])]
    return torch.cat(parts, dim=-1)


def _plain_rotary(s):
    angle = _angles(s)
    cos, sin, pairs = torch.cos(angle), torch.sin(angle), angle.shape[-1]
    out = {"q": _rotate(s["q"], cos, sin, pairs, s["adjacent"]), "k": _rotate(s["k"], cos, sin, pairs, s["adjacent"])}
    if s["train"]:
        out["dq"] = _rotate(s["dq"], cos, -sin, pairs, s["adjacent"])
        out["dk"] = _rotate(s["dk"], cos, -sin, pairs, s["adjacent"])
    return out


EPS = 1e-6


def _plain_norm(s):
    x = s["x"].float()
    centred = x - x.mean(dim=-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=-1, keepdim=True) + EPS)
    h = centred * rstd
    modulated = s["form"] == "modulated"
    w = s["scale"].float() + 1 if modulated else s["scale"].float()
    dtype = s["x"].dtype
    out = {"y": (h * w + s["shift"].float()).to(dtype)}
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(dim=-1, keepdim=True) - h * (g * h).mean(dim=-1, keepdim=True))
        over = (1,) if modulated else (0, 1)
        out["dx"] = dx.to(dtype)
        out["dscale"] = (dy * h).sum(dim=over, keepdim=modulated).to(dtype)
        out["dshift"] = dy.sum(dim=over, keepdim=modulated).to(dtype)
    return out


def _restored(x):
    """x as its 8-bit codes in groups of 128 features give it back."""

    f = x.shape[-1]
    groups = torch.nn.functional.pad(x, (0, -f % GROUP)).unflatten(-1, (-1, GROUP))
    codes, scales = _codes(groups)
    return (codes * scales).flatten(-2)[..., :f]


def _plain_gelu(s):
    x = s["x"].float()
    y = x * torch.sigmoid(2 * GELU_C * (x + GELU_A * x * x * x))
    r = _restored(x)
    gate = torch.sigmoid(2 * GELU_C * (r + GELU_A * r * r * r))
    slope = gate + r * gate * (1 - gate) * (2 * GELU_C) * (1 + 3 * GELU_A * r * r)
    return {"y": y.to(s["x"].dtype), "dx": (s["dy"].float() * slope).to(s["x"].dtype)}


# ---------------------------------------------------------------------------
# the calls of a program


def _own_int8(s):
    from convrot_mlx_b200 import int8_linear

    y = int8_linear(s["x"], s["qweight"], s["wscales"], s["bias_values"])
    if not s["train"]:
        return {"y": y}
    return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}


def _own_rotary(s):
    from convrot_mlx_b200 import axial_rotary

    q, k = axial_rotary(s["q"], s["k"], s["positions"], s["widths"], theta=s["theta"], interleaved=s["adjacent"])
    if not s["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _own_norm(s):
    from convrot_mlx_b200 import layer_norm, modulated_layer_norm

    if s["form"] == "modulated":
        y = modulated_layer_norm(s["x"], s["shift"], s["scale"], eps=EPS)
    else:
        y = layer_norm(s["x"], s["scale"], s["shift"], eps=EPS)
    if not s["train"]:
        return {"y": y}
    dx, dscale, dshift = torch.autograd.grad(y, (s["x"], s["scale"], s["shift"]), s["dy"])
    return {"y": y, "dx": dx, "dscale": dscale, "dshift": dshift}


def _own_gelu(s):
    from convrot_mlx_b200 import gelu_tanh_saved8

    y = gelu_tanh_saved8(s["x"])
    return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}


def run(state):
    op = state["op"]
    if own:
        return {"int8": _own_int8, "rotary": _own_rotary, "norm": _own_norm, "gelu": _own_gelu}[op](state)
    with torch.no_grad():
        return {"int8": _plain_int8, "rotary": _plain_rotary, "norm": _plain_norm, "gelu": _plain_gelu}[op](state)


# ---------------------------------------------------------------------------
# the definitions, in 64 bits


def _exact_codes(x):
    top = x.abs().max(dim=-1, keepdim=True).values
    steps = (127 * x / top).nan_to_num(0.0).round()
    return steps, top / 127


def _exact_turn(x, turn, adjacent):
    n = turn.shape[-1]
    x = x.double()
    head = x[..., :2 * n]
    z = torch.view_as_complex(head.reshape(*head.shape[:-1], n, 2).contiguous()) if adjacent else torch.complex(
        head[..., :n].contiguous(), head[..., n:].contiguous())
    z = z * turn
    y = torch.view_as_real(z).flatten(-2) if adjacent else torch.cat((z.real, z.imag), dim=-1)
    return torch.cat((y, x[..., 2 * n:]), dim=-1)


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        if case["op"] == "int8":
            c, a = _exact_codes(s["x"].double())
            w = s["qweight"].double()
            weight = w * s["wscales"].double()[:, None]
            y = torch.matmul(c, weight.mT) * a
            y = y + s["bias_values"].double() if case["bias"] else y
            if not case["train"]:
                return {"y": y}
            c, a = _exact_codes(s["dy"].double() * s["wscales"].double())
            return {"y": y, "dx": torch.matmul(c, w) * a}
        if case["op"] == "rotary":
            angle = torch.cat([torch.outer(s["positions"][:, a].double(),
                                           torch.exp(-math.log(case["theta"]) * torch.arange(w // 2, device="cuda").double() * 2 / w))
                               for a, w in enumerate(s["widths"])], dim=1)
            turn = torch.polar(torch.ones_like(angle), angle)
            out = {name: _exact_turn(s[name], turn, case["adjacent"]) for name in ("q", "k")}
            if case["train"]:
                out.update({name: _exact_turn(s[name], turn.conj(), case["adjacent"]) for name in ("dq", "dk")})
            return out
        if case["op"] == "norm":
            x = s["x"].double()
            var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
            sd = (var + EPS).sqrt()
            h = (x - mean) / sd
            w = s["scale"].double() + (1.0 if case["form"] == "modulated" else 0.0)
            y = torch.addcmul(s["shift"].double(), h, w)
            if not case["train"]:
                return {"y": y}
            dy = s["dy"].double()
            g = dy * w
            n = case["features"]
            dx = (n * g - g.sum(-1, keepdim=True) - h * torch.einsum("brf,brf->br", g, h)[..., None]) / (n * sd)
            if case["form"] == "modulated":
                return {"y": y, "dx": dx, "dscale": torch.einsum("brf,brf->bf", dy, h)[:, None],
                        "dshift": dy.sum(1, keepdim=True)}
            return {"y": y, "dx": dx, "dscale": torch.einsum("brf,brf->f", dy, h), "dshift": dy.sum((0, 1))}
        x = s["x"].double()
        y = 0.5 * x * (1 + torch.tanh(GELU_C * (x + GELU_A * x ** 3)))
        r = torch.empty_like(x)
        for at in range(0, case["features"], GROUP):
            c, a = _exact_codes(x[:, at:at + GROUP])
            r[:, at:at + GROUP] = c * a
        t = torch.tanh(GELU_C * (r + GELU_A * r ** 3))
        slope = 0.5 * (1 + t) + 0.5 * r * (1 - t * t) * GELU_C * (1 + 3 * GELU_A * r * r)
        return {"y": y, "dx": s["dy"].double() * slope}
