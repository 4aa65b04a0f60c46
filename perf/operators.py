"""The operators of a training step over sampled walks, as cases that can be timed.

Walks are the sentences of a language model whose words are the vertices.  One training step attends
over a packed batch of walks of different lengths, drops activations with the engine's own random
stream, and takes the softmax cross entropy over all vertices.  A case is one such operator at one
size; `run` computes it with elementary torch operations in 32 bits, or, with `own`, with the
framework's kernels.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}

# ---- the cases ---------------------------------------------------------------------------------


def attention(name, sequences, shortest, longest, heads, kv_heads, dim, train, dtype="bf16", tail=0, fused=False):
    """`sequences` lengths, spread between the shortest and the longest (over their logarithm), packed one after
    another; `tail` tokens after them belong to none.  fused: q, k and v are slices of one projection's output."""
    return {"name": name, "operator": "attention", "sequences": sequences, "shortest": shortest, "longest": longest,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "train": train, "dtype": dtype, "tail": tail,
            "fused": fused}


def loss(name, rows, vocabulary, dim, train, dtype="bf16"):
    return {"name": name, "operator": "loss", "rows": rows, "vocabulary": vocabulary, "dim": dim, "train": train,
            "dtype": dtype}


def dropout(name, rows, dim, p, residual, train, dtype="bf16"):
    return {"name": name, "operator": "dropout", "rows": rows, "dim": dim, "p": p, "residual": residual,
            "train": train, "dtype": dtype}


def listed():
    return [
        # scoring a few short walks in a notebook: all latency
        attention("attention_few_walks", 16, 1, 21, 4, 4, 64, train=False),
        # a training batch of walks of up to 100 steps, many of which end early
        attention("attention_walk_batch", 1024, 1, 101, 8, 8, 64, train=True),
        # training on long walks with grouped heads, packed to one row, slices of one projection, padding at the end
        attention("attention_long_walks", 5, 700, 4096, 16, 4, 128, train=True, tail=37, fused=True),
        # one long prompt through a model with few key heads
        attention("attention_prompt", 1, 16384, 16384, 16, 2, 128, train=False),
        # a head size that is no power of two, odd lengths, 16-bit floats
        attention("attention_odd_heads", 23, 3, 1999, 6, 3, 80, train=True, dtype="f16", tail=5),
        # a citation-network sized graph: 2711 vertices, a few rows, all latency
        loss("loss_small_graph", 61, 2711, 64, train=True),
        # every vertex of the benchmark's uniform-walk graph as a class, embeddings of 128
        loss("loss_57k_vertices", 8192, 56944, 128, train=True),
        # a large vocabulary and a wide model
        loss("loss_wide", 4096, 131072, 1024, train=True),
        # evaluation: no gradient, odd sizes, 16-bit floats
        loss("loss_evaluation", 1021, 100003, 520, train=False, dtype="f16"),
        # the hidden states of a few walks in 32 bits
        dropout("dropout_few_walks", 101, 64, 0.1, residual=False, train=False, dtype="f32"),
        # a residual branch of a layer, with its gradient
        dropout("dropout_layer", 8192, 1024, 0.1, residual=True, train=True),
        # the embeddings of a large batch, an odd width
        dropout("dropout_large", 65537, 1021, 0.5, residual=False, train=False),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attention", "loss", "dropout"])
    if kind == "attention":
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8]) if kv_heads <= 2 else kv_heads * rng.choice([1, 2, 4])
        heads = min(heads, 16) // kv_heads * kv_heads
        dim = 8 * rng.randint(4, 16)
        longest = _between(rng, 1, 8192)
        shortest = _between(rng, 1, longest)
        most = max(1, min(2048, 40000 // longest, 120000000 // (longest * longest)))
        out = attention("", _between(rng, 1, most), shortest, longest, heads, kv_heads, dim, rng.random() < 0.6,
                        rng.choice(["bf16", "bf16", "f16"]), rng.choice([0, 0, rng.randint(1, 99)]),
                        rng.random() < 0.5)
    elif kind == "loss":
        dim = 8 * _between(rng, 4, 128)
        rows = _between(rng, 1, 8192)
        vocabulary = _between(rng, 1000, min(500000, 550000000000 // (dim * rows), 2000000000 // rows))
        out = loss("", rows, vocabulary, dim, rng.random() < 0.6, rng.choice(["bf16", "bf16", "f16"]))
    else:
        dim = _between(rng, 16, 4096)
        rows = _between(rng, 1, 60000000 // dim)
        train = rng.random() < 0.6
        out = dropout("", rows, dim, rng.choice([0.0, 0.05, 0.1, 0.3, 0.5]), rng.random() < 0.5, train,
                      rng.choice(["bf16", "f16", "f32"]))
    del out["name"]
    return out


def lengths(case):
    """The case's sequence lengths; they belong to the case, so that its work does not depend on a seed."""
    rng = np.random.default_rng([case["sequences"], case["shortest"], case["longest"]])
    low, high = math.log(case["shortest"]), math.log(case["longest"] + 1)
    some = np.exp(rng.uniform(low, high, case["sequences"])).astype(np.int64)
    some = np.clip(some, case["shortest"], case["longest"])
    some[0] = case["longest"]
    return some


def work(case):
    size = BYTES[case["dtype"]]
    if case["operator"] == "attention":
        n = lengths(case)
        tokens = int(n.sum()) + case["tail"]
        pairs = int((n * (n + 1) // 2).sum()) * case["heads"]
        qo, kv = tokens * case["heads"] * case["dim"] * size, tokens * case["kv_heads"] * case["dim"] * size
        move = 2 * qo + 2 * kv  # q, o; k, v
        flops = 4 * case["dim"] * pairs
        if case["train"]:
            move += 2 * qo + 2 * kv  # do, dq; dk, dv
            flops += 10 * case["dim"] * pairs
        return {"bytes": move, "flops": flops}
    if case["operator"] == "loss":
        n, v, d = case["rows"], case["vocabulary"], case["dim"]
        move = (n + v) * d * size + 12 * n
        flops = 2 * n * v * d
        if case["train"]:
            move += (n + v) * d * size + 4 * n
            flops += 4 * n * v * d
        return {"bytes": move, "flops": flops}
    n = case["rows"] * case["dim"]
    passes = 2 + case["residual"] + (2 if case["train"] else 0)
    return {"bytes": passes * n * size, "flops": 2 * n * (2 if case["train"] else 1)}


# ---- inputs ------------------------------------------------------------------------------------


def prepare(case, seed):
    device = "cuda"
    kind = TYPES[case["dtype"]]
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=device, generator=gen) * std).to(kind)

    state = {"case": case}
    if case["operator"] == "attention":
        n = lengths(case)
        starts = np.concatenate([[0], np.cumsum(n)])
        tokens, heads, kv_heads, dim = int(starts[-1]) + case["tail"], case["heads"], case["kv_heads"], case["dim"]
        if case["fused"]:
            qkv = normal(tokens, heads + 2 * kv_heads, dim)
            state["q"], state["k"], state["v"] = qkv.split([heads, kv_heads, kv_heads], dim=1)
        else:
            state["q"] = normal(tokens, heads, dim)
            state["k"], state["v"] = normal(tokens, kv_heads, dim), normal(tokens, kv_heads, dim)
        if case["train"]:
            state["dout"] = normal(tokens, heads, dim)
        state["starts"] = torch.from_numpy(starts.astype(np.int32)).to(device)
        state["longest"] = int(n.max())
        if own:
            from nextdoor_amd import ops
            # one plan a batch of walks: every layer and both directions use it
            state["plan"] = ops.PackedSequences(state["starts"], tokens)
    elif case["operator"] == "loss":
        rows, vocabulary, dim = case["rows"], case["vocabulary"], case["dim"]
        state["hidden"] = normal(rows, dim)
        state["weight"] = normal(vocabulary, dim, std=2 / math.sqrt(dim))
        # a twentieth of the rows have no next vertex: their target is the engine's "no vertex", |V|
        target = torch.randint(vocabulary, (rows,), device=device, generator=gen)
        ended = torch.rand(rows, device=device, generator=gen) < 0.05
        state["target"] = torch.where(ended, torch.full_like(target, vocabulary), target).to(torch.int32)
        if case["train"]:
            # what a mean over the rows sends back, each walk with a weight of its own
            state["dloss"] = (0.5 + torch.rand(rows, device=device, generator=gen)) / rows
    else:
        rows, dim = case["rows"], case["dim"]
        state["x"] = normal(rows, dim)
        state["seed"], state["step"] = seed * 0x9E3779B97F4A7C15 % (1 << 64), seed % 1000
        if case["residual"]:
            state["residual"] = normal(rows, dim)
        if case["train"]:
            state["dout"] = normal(rows, dim)
    return state


# ---- one pass ----------------------------------------------------------------------------------


def run(state):
    return {"attention": _run_attention, "loss": _run_loss, "dropout": _run_dropout}[state["case"]["operator"]](state)


def _run_attention(state):
    train = state["case"]["train"]
    if own:
        from nextdoor_amd import ops
        out, lse = ops.packed_attention_forward(state["q"], state["k"], state["v"], state["plan"])
        if not train:
            return {"out": out}
        dq, dk, dv = ops.packed_attention_backward(state["dout"], state["q"], state["k"], state["v"], out, lse,
                                                   state["plan"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    q, k, v, starts, longest = state["q"], state["k"], state["v"], state["starts"].long(), state["longest"]
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    group, batch, kind, scale = heads // kv_heads, starts.numel() - 1, q.dtype, 1 / math.sqrt(dim)
    # the packed sequences side by side, short ones filled up: [sequence, key head, (head of the group,) place, dim]
    place = torch.arange(longest, device=q.device)
    there = place < (starts[1:] - starts[:-1])[:, None]
    token = (starts[:-1, None] + place).clamp(max=tokens - 1)
    seen = (place[:, None] >= place) & there[:, None, :]  # [sequence, query, key]

    def rows(x):  # of query heads
        x = x.float()[token].view(batch, longest, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
        return x.reshape(batch, kv_heads, group * longest, dim)

    def columns(x):
        return x.float()[token].permute(0, 2, 1, 3)

    def packed(x, of_heads):
        x = x.view(batch, of_heads, longest, dim).transpose(1, 2)
        full = torch.zeros(tokens, of_heads, dim, device=x.device)
        full[token[there]] = x[there]
        return full.to(kind)

    qs, ks, vs = rows(q), columns(k), columns(v)
    s = (qs @ ks.transpose(2, 3)).view(batch, kv_heads, group, longest, longest) * scale
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    del s
    p = p / p.sum(-1, keepdim=True)
    p = p.view(batch, kv_heads, group * longest, longest)
    out = packed(p @ vs, heads)
    if not train:
        return {"out": out}
    # a place past a sequence's end is no query: nothing comes back from it
    no_row = (~there)[:, None, None, :, None].expand(batch, kv_heads, group, longest, 1)
    dos = rows(state["dout"]).masked_fill(no_row.reshape(batch, kv_heads, group * longest, 1), 0.0)
    dv = p.transpose(2, 3) @ dos
    dp = dos @ vs.transpose(2, 3)
    ds = p * (dp - (dp * p).sum(-1, keepdim=True))
    del dp
    dq = ds @ ks * scale
    dk = ds.transpose(2, 3) @ qs * scale
    return {"out": out, "dq": packed(dq, heads), "dk": packed(dk, kv_heads), "dv": packed(dv, kv_heads)}


def _run_loss(state):
    train = state["case"]["train"]
    if own:
        from nextdoor_amd import ops
        loss_, lse = ops.vocabulary_loss_forward(state["hidden"], state["weight"], state["target"])
        if not train:
            return {"loss": loss_}
        dh, dw = ops.vocabulary_loss_backward(state["dloss"], state["hidden"], state["weight"], state["target"], lse)
        return {"loss": loss_, "dhidden": dh, "dweight": dw}
    h, w, target = state["hidden"].float(), state["weight"].float(), state["target"].long()
    known = (target >= 0) & (target < w.shape[0])
    at = torch.where(known, target, torch.zeros_like(target))[:, None]
    z = h @ w.T
    top = z.amax(1, keepdim=True)
    lse = torch.log(torch.exp(z - top).sum(1, keepdim=True)) + top
    loss_ = torch.where(known, (lse - z.gather(1, at))[:, 0], torch.zeros_like(lse[:, 0]))
    if not train:
        return {"loss": loss_}
    each = torch.where(known, state["dloss"], torch.zeros_like(state["dloss"]))[:, None]
    g = torch.exp(z - lse) * each
    del z
    g.scatter_add_(1, at, -each)
    return {"loss": loss_, "dhidden": (g @ w).to(state["hidden"].dtype), "dweight": (g.T @ h).to(state["weight"].dtype)}


def _uniforms(n, seed, step, device):
    """Draw 0 of slots 0 .. n - 1 in the engine's grouped stream: Philox4x32-10, four slots to a block."""
    low = 0xFFFFFFFF
    group = torch.arange((n + 3) // 4, device=device)
    c0, c1 = group & low, group >> 32
    c2, c3 = torch.full_like(group, step | 1 << 31), torch.zeros_like(group)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits; the shifts below drop the sign
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]
    return (words >> 8).float() * 2.0 ** -24


def _run_dropout(state):
    case = state["case"]
    x, residual, p = state["x"], state.get("residual"), case["p"]
    if own:
        from nextdoor_amd import ops
        out = {"out": ops.dropout_forward(x, p, state["seed"], state["step"], residual=residual)}
        if case["train"]:
            out["dx"] = ops.dropout_backward(state["dout"], p, state["seed"], state["step"])
        return out
    kept = (_uniforms(x.numel(), state["seed"], state["step"], x.device) >= p).view(x.shape)
    factor = torch.where(kept, 1 / (1 - p), 0.0)
    y = x.float() * factor
    if residual is not None:
        y = y + residual.float()
    out = {"out": y.to(x.dtype)}
    if case["train"]:
        out["dx"] = (state["dout"].float() * factor).to(x.dtype)
    return out


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": _exact_attention, "loss": _exact_loss, "dropout": _exact_dropout}[case["operator"]](case, state)


def _exact_attention(case, state):
    """Sequence after sequence and head after head, each row's softmax over the keys up to it."""
    if sum(int(n) ** 2 for n in lengths(case)) * case["heads"] > 6e9 or case["sequences"] * case["heads"] > 20000:
        return None
    q, k, v = (state[name].double() for name in "qkv")
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    got = {"out": out}
    if case["train"]:
        dout = state["dout"].double()
        got.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    begin = 0
    for n in lengths(case).tolist():
        at = slice(begin, begin + n)
        begin += n
        later = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        for head in range(case["heads"]):
            of = head // group
            a, b, c = q[at, head], k[at, of], v[at, of]
            logits = torch.mm(a, b.t()) / math.sqrt(case["dim"])
            logits[later] = -math.inf
            weight = torch.softmax(logits, 1)
            out[at, head] = torch.mm(weight, c)
            if case["train"]:
                d = dout[at, head]
                dweight = torch.mm(d, c.t())
                dlogits = weight * (dweight - (d * out[at, head]).sum(1)[:, None]) / math.sqrt(case["dim"])
                got["dq"][at, head] = torch.mm(dlogits, b)
                got["dk"][at, of] += torch.mm(dlogits.t(), a)
                got["dv"][at, of] += torch.mm(weight.t(), d)
    return got


def _exact_loss(case, state):
    """The classes in pieces, twice: the rows' logarithms of sums, then the gradients."""
    if case["rows"] * case["vocabulary"] * case["dim"] > 1e12:
        return None
    h, w = state["hidden"].double(), state["weight"].double()
    target, classes = state["target"].long(), case["vocabulary"]
    has = target < classes
    pieces = [(i, min(i + 8192, classes)) for i in range(0, classes, 8192)]
    parts = torch.stack([torch.logsumexp(torch.mm(h, w[i:j].t()), 1) for i, j in pieces])
    lse = torch.logsumexp(parts, 0)
    own_logit = (h * w[target.clamp(max=classes - 1)]).sum(1)
    got = {"loss": torch.where(has, lse - own_logit, torch.zeros_like(lse))}
    if case["train"]:
        each = torch.where(has, state["dloss"].double(), torch.zeros_like(lse))
        got["dhidden"], got["dweight"] = torch.zeros_like(h), torch.empty_like(w)
        for i, j in pieces:
            g = torch.exp(torch.mm(h, w[i:j].t()) - lse[:, None])
            g -= (target[:, None] == torch.arange(i, j, device=h.device)).double()
            g *= each[:, None]
            got["dhidden"] += torch.mm(g, w[i:j])
            got["dweight"][i:j] = torch.mm(g.t(), h)
    return got


def _exact_dropout(case, state):
    """Philox4x32-10 on the host, in unsigned arithmetic."""
    x = state["x"].cpu().double().numpy()
    u32 = np.uint64(0xFFFFFFFF)
    count = (x.size + 3) // 4
    ctr = [np.arange(count, dtype=np.uint64), np.zeros(count, np.uint64),
           np.full(count, state["step"] + 2 ** 31, np.uint64), np.zeros(count, np.uint64)]
    key = [state["seed"] % 2 ** 32, state["seed"] // 2 ** 32]
    for turn in range(10):
        first, second = ctr[0] * np.uint64(3528531795), ctr[2] * np.uint64(3449720151)
        ctr = [(second >> np.uint64(32)) ^ ctr[1] ^ np.uint64((key[0] + turn * 2654435769) % 2 ** 32), second & u32,
               (first >> np.uint64(32)) ^ ctr[3] ^ np.uint64((key[1] + turn * 3144134277) % 2 ** 32), first & u32]
    chance = np.stack(ctr, 1).reshape(-1)[:x.size].reshape(x.shape) // np.uint64(256)
    dropped = chance.astype(np.float64) / 2 ** 24 < np.float64(np.float32(case["p"]))
    keep = 1.0 / (1.0 - case["p"])
    y = np.where(dropped, 0.0, x * keep)
    if case["residual"]:
        y += state["residual"].cpu().double().numpy()
    got = {"out": torch.from_numpy(y)}
    if case["train"]:
        got["dx"] = torch.from_numpy(np.where(dropped, 0.0, state["dout"].cpu().double().numpy() * keep))
    return got
