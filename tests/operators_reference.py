"""The training operators from their definitions in 64 bits, and how far a kernel that rounds where ours do may be off.

Every bound is a sum of what each rounding can do at most.  With u the largest relative error of a rounding to the 16-bit
type (half the distance of neighbours: 2^-8 for bfloat16, 2^-11 for float16), weights and their gradients are rounded once
before the second product, results once at the end; what is kept in 32 bits adds SMALL of the sum of magnitudes: sums
of at most a few thousand terms in blocks (under 2^10 roundings of 2^-24 on a path), logits of at most a hundred times that.
"""
import math

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# what becomes 0: half the smallest float16; below the normal numbers of 32 bits, whose exponents bfloat16 has
LEAST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
SMALL = 2.0 ** -14


def attention(q, k, v, starts, scale, dout=None):
    """Values and bounds of out (dq, dk, dv, if dout is given), dense over all pairs of tokens; inputs on the CPU."""
    unit, least = UNIT[q.dtype], LEAST[q.dtype]
    q, k, v = q.double(), k.double(), v.double()
    tokens, heads, dim = q.shape
    group = heads // k.shape[1]
    of = torch.full((tokens,), -1)
    for i in range(len(starts) - 1):
        of[starts[i]:starts[i + 1]] = i
    at = torch.arange(tokens)
    sees = (of[:, None] == of) & (of[:, None] >= 0) & (at[:, None] >= at)
    row = sees.any(1)
    out, out_off, lse = torch.zeros_like(q), torch.zeros_like(q), torch.full((heads, tokens), -math.inf).double()
    names = ("dq", "dk", "dv")
    got = {n: torch.zeros_like(x) for n, x in zip(names, (q, k, v))}
    off = {n: torch.zeros_like(x) for n, x in zip(names, (q, k, v))}
    for h in range(heads):
        a, b, c = q[:, h], k[:, h // group], v[:, h // group]
        # what no row sees does not take part, whatever it holds
        a, b, c = (torch.where(row[:, None], x, torch.zeros_like(x)) for x in (a, b, c))
        s = torch.where(sees, a @ b.T * scale, torch.full((), -math.inf).double())
        lse[h][row] = torch.logsumexp(s[row], 1)
        p = torch.where(sees, torch.exp(s - torch.where(row, lse[h], torch.zeros(()).double())[:, None]), torch.zeros(()).double())
        out[:, h] = p @ c
        spread = p @ c.abs()
        out_off[:, h] = unit * (out[:, h].abs() + spread) + SMALL * spread + least * (1 + spread)
        if dout is None:
            continue
        d = torch.where(row[:, None], dout[:, h].double(), torch.zeros(()).double())
        dp = d @ c.T
        delta = (d * out[:, h]).sum(1)
        ds = p * (dp - delta[:, None])
        # delta comes from the rounded out
        ds_off = unit * ds.abs() + p * ((d.abs() * out_off[:, h]).sum(1) + SMALL * (d.abs() @ c.abs().T).amax(1))[:, None] + \
            least * sees.double() + SMALL * ds.abs()
        p_off = (unit + SMALL) * p + least * sees.double()
        got["dq"][:, h] = ds @ b * scale
        off["dq"][:, h] = unit * got["dq"][:, h].abs() + ds_off @ b.abs() * abs(scale) + least
        got["dk"][:, h // group] += ds.T @ a * scale
        off["dk"][:, h // group] += ds_off.T @ a.abs() * abs(scale)
        got["dv"][:, h // group] += p.T @ d
        off["dv"][:, h // group] += p_off.T @ d.abs()
    for n in ("dk", "dv"):
        off[n] += unit * got[n].abs() + least
    got.update(out=out, lse=lse)
    off.update(out=out_off, lse=SMALL * (1 + lse.abs()))
    return got, off


def vocabulary_loss(hidden, weight, target, dloss=None):
    unit, least = UNIT[hidden.dtype], LEAST[hidden.dtype]
    h, w = hidden.double(), weight.double()
    classes = w.shape[0]
    has = (target >= 0) & (target < classes)
    z = h @ w.T
    lse = torch.logsumexp(z, 1)
    at = torch.where(has, target, torch.zeros_like(target)).long()
    zero = torch.zeros(()).double()
    loss = torch.where(has, lse - z.gather(1, at[:, None])[:, 0], zero)
    # a logit: dim products summed in 32 bits
    z_off = (h.shape[1] + 8) * 2.0 ** -24 * (h.abs() @ w.abs().T).amax(1) + 2.0 ** -21 * z.abs().amax(1)
    got, off = {"loss": loss, "lse": lse}, {"lse": z_off + 2.0 ** -13, "loss": 2 * z_off + 2.0 ** -13}
    if dloss is not None:
        each = torch.where(has, dloss.double(), zero)
        p = torch.exp(z - lse[:, None])
        g = p.clone()
        g[torch.arange(len(at)), at] -= 1
        g *= each[:, None]
        most = each.abs().max() if len(each) else zero
        g_off = unit * g.abs() + (2 * z_off[:, None] + SMALL) * p * each.abs()[:, None] + SMALL * g.abs() + \
            least * 2.0 ** -15 * most * (each != 0)[:, None] + 2.0 ** -126 * each.abs()[:, None]  # (p below 2^-126 is 0)
        got["dhidden"], got["dweight"] = g @ w, g.T @ h
        off["dhidden"] = unit * got["dhidden"].abs() + g_off @ w.abs() + least
        off["dweight"] = unit * got["dweight"].abs() + g_off.T @ h.abs() + least
    return got, off


def uniforms(n, seed, step):
    """Draw 0 of slots 0 .. n - 1 in the grouped stream, from the definition of Philox4x32-10."""
    low = np.uint64(0xFFFFFFFF)
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [block & low, block >> np.uint64(32), np.full_like(block, step + (1 << 31)), np.zeros_like(block)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return (np.stack(c, 1).reshape(-1)[:n] >> np.uint64(8)).astype(np.float32) * np.float32(2.0 ** -24)


def dropout(x, p, seed, step, residual=None):
    kept = torch.from_numpy(uniforms(x.numel(), seed, step) >= np.float32(p)).view(x.shape)
    y = torch.where(kept, x.double() / (1 - p if p < 1 else 1), torch.zeros(()).double())
    spread = y.abs()
    if residual is not None:
        y, spread = y + residual.double(), spread + residual.double().abs()
    unit = UNIT[x.dtype]
    # the factor, the product and the sum in 32 bits, then the type's rounding
    return y, unit * y.abs() + 3 * 2.0 ** -24 * spread + LEAST[x.dtype] + 2.0 ** -149


def close(got, want, off):
    """Whether every value is within its bound; -inf and NaN only where they belong."""
    got, want = got.detach().cpu().double(), want.double()
    odd = ~torch.isfinite(want)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    good = torch.where(odd, same, (got - want).abs() <= off)
    if good.all():
        return True
    at = tuple(int(i) for i in (~good).nonzero()[0])
    print("%d of %d off; first at %s: %r, should be %r within %r" % (int((~good).sum()), good.numel(), at, float(got[at]),
                                                                  float(want[at]), float(off[at]) if off.shape == want.shape else off))
    return False
