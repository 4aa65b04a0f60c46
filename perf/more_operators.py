"""The other operators of a transformer over sampled walks, as cases that can be timed.

Between the attention over a batch of walks and the loss over all vertices a block normalises its rows,
projects them, and sends them through a feed-forward part.  A case is one such operator at one size; `run`
computes it with elementary torch operations in 32 bits, or, with `own`, with the framework's kernels.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}

# ---- the cases ---------------------------------------------------------------------------------


def norm(name, rows, dim, train, dtype="bf16"):
    return {"name": name, "operator": "norm", "rows": rows, "dim": dim, "train": train, "dtype": dtype}


def linear(name, rows, dim, out, train, activation="none", bias=True, residual=False, dtype="bf16"):
    """rows vectors of `dim` places to vectors of `out`."""
    return {"name": name, "operator": "linear", "rows": rows, "dim": dim, "out": out, "train": train,
            "activation": activation, "bias": bias, "residual": residual, "dtype": dtype}


def mlp(name, rows, dim, inner, train, activation="silu", gated=True, bias=False, residual=True, dtype="bf16"):
    """rows vectors of `dim` places through `inner` hidden ones and back; gated: two projections, one of them through
    the activation, and their product."""
    return {"name": name, "operator": "mlp", "rows": rows, "dim": dim, "inner": inner, "train": train,
            "activation": activation, "gated": gated, "bias": bias, "residual": residual, "dtype": dtype}


def listed():
    return [
        # one walk in a notebook: all latency
        norm("norm_few_rows", 101, 64, train=False),
        # a norm of a training step, both directions, the sizes of a layer's dropout
        norm("norm_layer", 8192, 1024, train=True),
        # a large batch through a wide model
        norm("norm_wide", 16384, 4096, train=True),
        # rows of an odd size, in 32 bits
        norm("norm_odd", 20011, 1021, train=True, dtype="f32"),
        # the next vertex of one walk: a single row against a whole matrix
        linear("linear_one_token", 1, 1024, 4096, train=False, activation="gelu"),
        # the first matrix of a feed-forward part, with its gradients
        linear("linear_layer", 8192, 1024, 4096, train=True, activation="gelu"),
        # scoring a large batch: the projection behind the attention, added to what went into the block
        linear("linear_projection", 16384, 2048, 2048, train=False, bias=False, residual=True),
        # odd sizes, 16-bit floats
        linear("linear_odd", 1021, 520, 1000, train=True, activation="relu", residual=True, dtype="f16"),
        # a few walks that grow side by side
        mlp("mlp_few_tokens", 16, 1024, 2816, train=False),
        # the walk model's own sizes, over a batch of 1024 walks
        mlp("mlp_walk_batch", 20483, 64, 256, train=True, activation="gelu", gated=False, bias=True),
        # a gated part of a wide model, with its gradients
        mlp("mlp_wide", 8192, 2048, 5632, train=True),
        # odd sizes, 16-bit floats
        mlp("mlp_odd", 3001, 328, 1000, train=True, activation="gelu", bias=True, dtype="f16"),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "mlp"])
    train, dtype = rng.random() < 0.6, rng.choice(["bf16", "bf16", "f16"])
    activation = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    bias, residual = rng.random() < 0.5, rng.random() < 0.5
    if kind == "norm":
        dim = _between(rng, 16, 8192)
        out = norm("", _between(rng, 1, min(65536, 67000000 // dim)), dim, train, rng.choice(["bf16", "f16", "f32"]))
    elif kind == "linear":
        dim, wide = 8 * _between(rng, 4, 512), 8 * _between(rng, 4, 512)
        rows = _between(rng, 1, min(32768, 90000000000 // (dim * wide)))
        out = linear("", rows, dim, wide, train, activation, bias, residual, dtype)
    else:
        dim = 8 * _between(rng, 4, 256)
        gated = rng.random() < 0.6
        inner = 8 * _between(rng, dim // 8, dim // 2 if dim < 1024 else 704)
        rows = _between(rng, 1, min(32768, 90000000000 // (dim * inner)))
        out = mlp("", rows, dim, inner, train, activation, gated, bias, residual, dtype)
    del out["name"]
    return out


def work(case):
    size, rows, dim, train = BYTES[case["dtype"]], case["rows"], case["dim"], case["train"]
    if case["operator"] == "norm":
        move = (2 * rows * dim + 2 * dim) * size
        if train:
            move += (2 * rows * dim + 2 * dim) * size
        return {"bytes": move, "flops": rows * dim * (19 if train else 8)}
    if case["operator"] == "linear":
        wide, weights = case["out"], case["dim"] * case["out"]
        move = (rows * dim + weights + rows * wide * (1 + case["residual"]) + wide * case["bias"]) * size
        if train:
            move += (rows * wide + rows * dim + weights + wide * case["bias"]) * size
        return {"bytes": move, "flops": 2 * rows * weights * (3 if train else 1)}
    inner, wide = case["inner"], case["inner"] * (1 + case["gated"])
    weights = dim * wide + inner * dim
    parameters = weights + (wide + dim) * case["bias"]
    move = (2 * rows * dim + parameters + rows * dim * case["residual"]) * size
    if train:
        move += (2 * rows * dim + parameters) * size
    return {"bytes": move, "flops": 2 * rows * weights * (3 if train else 1)}


# ---- inputs ------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, dim = TYPES[case["dtype"]], case["rows"], case["dim"]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std + mean).to(kind)

    state = {"case": case, "x": normal(rows, dim)}
    if case["operator"] == "norm":
        # what runs along a residual stream: rows of different sizes, not centred
        size = torch.exp(torch.randn(rows, 1, device="cuda", generator=gen))
        state["x"] = (state["x"].float() * size + 0.3 * size).to(kind)
        state["weight"], state["bias"] = normal(dim, std=0.2, mean=1.0), normal(dim, std=0.1)
        wide = dim
    elif case["operator"] == "linear":
        wide = case["out"]
        state["weight"] = normal(wide, dim, std=1 / math.sqrt(dim))
        state["bias"] = normal(wide, std=0.2) if case["bias"] else None
    else:
        inner, wide = case["inner"], dim
        state["up"] = normal(inner * (1 + case["gated"]), dim, std=1 / math.sqrt(dim))
        state["down"] = normal(dim, inner, std=1 / math.sqrt(inner))
        state["up_bias"] = normal(state["up"].shape[0], std=0.2) if case["bias"] else None
        state["down_bias"] = normal(dim, std=0.2) if case["bias"] else None
    state["residual"] = normal(rows, wide) if case.get("residual") else None
    if case["train"]:
        state["dout"] = normal(rows, wide)
    return state


# ---- one pass ----------------------------------------------------------------------------------


def run(state):
    return {"norm": _run_norm, "linear": _run_linear, "mlp": _run_mlp}[state["case"]["operator"]](state)


EPS = 1e-5


def _run_norm(state):
    x, weight, bias, train = state["x"], state["weight"], state["bias"], state["case"]["train"]
    if own:
        from nextdoor_amd import ops
        out, mean, rstd = ops.layer_norm_forward(x, weight, bias, EPS)
        if not train:
            return {"out": out}
        dx, dweight, dbias = ops.layer_norm_backward(state["dout"], x, weight, mean, rstd)
        return {"out": out, "dx": dx, "dweight": dweight, "dbias": dbias}
    kind, x, weight, bias = x.dtype, x.float(), weight.float(), bias.float()
    dim = x.shape[1]
    centred = x - x.sum(1, keepdim=True) / dim
    rstd = 1 / torch.sqrt((centred * centred).sum(1, keepdim=True) / dim + EPS)
    there = centred * rstd
    out = {"out": (there * weight + bias).to(kind)}
    if train:
        dout = state["dout"].float()
        each = dout * weight
        dx = rstd * (each - each.sum(1, keepdim=True) / dim - there * ((each * there).sum(1, keepdim=True) / dim))
        out.update(dx=dx.to(kind), dweight=(dout * there).sum(0).to(kind), dbias=dout.sum(0).to(kind))
    return out


def _activate(z, name):
    """The activation of z and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).float()
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        s = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * s, s + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    inside = math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
    t = torch.tanh(inside)
    slope = math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * slope


def _run_linear(state):
    case, x, weight, bias, residual = state["case"], state["x"], state["weight"], state["bias"], state["residual"]
    if own:
        from nextdoor_amd import ops
        activation = None if case["activation"] == "none" else case["activation"]
        if not case["train"]:
            return {"out": ops.linear_forward(x, weight, bias, activation, residual)}
        out, z = ops.linear_forward(x, weight, bias, activation, residual, keep=True)
        dx, dweight, dbias = ops.linear_backward(state["dout"], x, weight, z, activation, bias is not None)
        return _named(out=out, dx=dx, dweight=dweight, dbias=dbias)
    kind, x, weight = x.dtype, x.float(), weight.float()
    z = x @ weight.T
    if bias is not None:
        z = z + bias.float()
    y, slope = _activate(z, case["activation"])
    if residual is not None:
        y = y + residual.float()
    out = {"out": y.to(kind)}
    if case["train"]:
        dz = state["dout"].float() * slope
        out.update(dx=(dz @ weight).to(kind), dweight=(dz.T @ x).to(kind))
        if bias is not None:
            out["dbias"] = dz.sum(0).to(kind)
    return out


def _named(**outputs):
    return {name: value for name, value in outputs.items() if value is not None}


def _run_mlp(state):
    case, x, up, down = state["case"], state["x"], state["up"], state["down"]
    up_bias, down_bias, residual, gated = state["up_bias"], state["down_bias"], state["residual"], case["gated"]
    if own:
        from nextdoor_amd import ops
        activation = None if case["activation"] == "none" else case["activation"]
        if not case["train"]:
            return {"out": ops.mlp_forward(x, up, down, up_bias, down_bias, activation, gated, residual)}
        out, z, h = ops.mlp_forward(x, up, down, up_bias, down_bias, activation, gated, residual, keep=True)
        dx, dup, ddown, dup_bias, ddown_bias = ops.mlp_backward(state["dout"], x, up, down, z, h, activation, gated,
                                                                up_bias is not None, down_bias is not None)
        return _named(out=out, dx=dx, dup=dup, ddown=ddown, dup_bias=dup_bias, ddown_bias=ddown_bias)
    kind, x, up, down, inner = x.dtype, x.float(), up.float(), down.float(), down.shape[1]
    z = x @ up.T
    if up_bias is not None:
        z = z + up_bias.float()
    a, slope = _activate(z[:, :inner], case["activation"])
    h = a * z[:, inner:] if gated else a
    y = h @ down.T
    if down_bias is not None:
        y = y + down_bias.float()
    if residual is not None:
        y = y + residual.float()
    out = {"out": y.to(kind)}
    if case["train"]:
        dout = state["dout"].float()
        dh = dout @ down
        dz = torch.cat([dh * z[:, inner:] * slope, dh * a], 1) if gated else dh * slope
        out.update(dx=(dz @ up).to(kind), dup=(dz.T @ x).to(kind), ddown=(dout.T @ h).to(kind))
        if up_bias is not None:
            out.update(dup_bias=dz.sum(0).to(kind), ddown_bias=dout.sum(0).to(kind))
    return out


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    """The forward pass as a formula of 64-bit tensors; the gradients are autograd's of that formula."""
    functional = torch.nn.functional
    state = prepare(case, seed)
    names = [n for n in ("x", "weight", "bias", "up", "down", "up_bias", "down_bias") if state.get(n) is not None]
    given = {n: state[n].double().requires_grad_(case["train"]) for n in names}
    act = {"none": lambda z: z, "relu": functional.relu, "silu": functional.silu, "gelu": functional.gelu,
           "gelu_tanh": lambda z: functional.gelu(z, approximate="tanh")}[case.get("activation", "none")]
    if case["operator"] == "norm":
        out = functional.layer_norm(given["x"], (case["dim"],), given["weight"], given["bias"], EPS)
    elif case["operator"] == "linear":
        out = act(functional.linear(given["x"], given["weight"], given.get("bias")))
    else:
        z = functional.linear(given["x"], given["up"], given.get("up_bias"))
        if case["gated"]:
            gate, value = z.chunk(2, 1)
            h = act(gate) * value
        else:
            h = act(z)
        out = functional.linear(h, given["down"], given.get("down_bias"))
    if state["residual"] is not None:
        out = out + state["residual"].double()
    got = {"out": out.detach()}
    if case["train"]:
        slopes = torch.autograd.grad(out, [given[n] for n in names], state["dout"].double())
        got.update({"d" + n: slope for n, slope in zip(names, slopes)})
    return got
