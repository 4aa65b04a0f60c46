"""Layer norm, linear maps and feed-forward parts from their definitions in 64 bits, and how far a kernel that rounds where ours do
may be off.

Every bound is a sum of what each rounding can do at most.  With u the largest relative error of a rounding to the type (half the
distance of neighbours), what is kept in the type (results; z, h and the gradient of z, which a second product or the backward
pass reads) is off by u; a sum of n products in 32 bits by (n + 8) 2^-24 of the sum of their magnitudes; an activation by
2^-20 (1 + |z|) of itself - the argument of its exponential is rounded, and that of an exponential of 2 z is off by 3 |z| 2^-24 - and by
2^-21 |z|, the normal integral's polynomial being good to 2^-23.
"""
import math

import torch

from tests.operators_reference import LEAST, UNIT

MOST_SLOPE, MOST_CURVATURE = 1.13, 0.8  # of any of the activations: |a'| and |a''| are largest for gelu, 1.129 and 2 / sqrt(2 pi)


def activation(z, name):
    """(a, a') of a 64-bit tensor."""
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, torch.where(torch.isnan(z), z, 0.0)), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if name == "gelu":
        s = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * s, s + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    assert name == "gelu_tanh"
    c = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * c * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * z * z)


def _activated(z, z_off, name):
    """a(z), a'(z) and their bounds where z is off by z_off."""
    a, slope = activation(z, name)
    if name is None:
        return a, slope, z_off, torch.zeros_like(z)
    near = 2.0 ** -20 * (1 + z.abs())
    a_off = MOST_SLOPE * z_off + near * a.abs() + 2.0 ** -21 * z.abs()
    if name == "relu":
        return a, slope, z_off, (z.abs() <= z_off).double()
    return a, slope, a_off, MOST_CURVATURE * z_off + near * slope.abs() + 2.0 ** -20 * (1 + z.abs())


def _sum_off(n):
    return (n + 8) * 2.0 ** -24


def _product(a, a_off, b):
    """a b of two matrices, b exact, and its bound before it is rounded."""
    spread = a.abs() @ b.abs()
    return a @ b, a_off @ b.abs() + _sum_off(a.shape[1]) * (spread + a_off @ b.abs())


def _rounded(x, off, unit, least):
    return off + unit * (x.abs() + off) + least


def linear(x, weight, bias=None, name=None, residual=None, dout=None):
    """Values and bounds of out (dx, dweight, dbias, if dout is given); two-dimensional inputs on the CPU."""
    unit, least = UNIT[x.dtype], LEAST[x.dtype]
    x, w = x.double(), weight.double()
    none = torch.zeros((), dtype=torch.float64)
    b = none if bias is None else bias.double()
    z, z_off = _product(x, torch.zeros_like(x), w.T)
    z, z_off = z + b, z_off + 2.0 ** -24 * (z.abs() + b.abs())
    a, _, a_off, _ = _activated(z, z_off, name)
    r = none if residual is None else residual.double()
    got = {"out": a + r}
    off = {"out": _rounded(a + r, a_off + 2.0 ** -24 * (a.abs() + r.abs()), unit, least)}
    if dout is not None:
        d = dout.double()
        # slopes come from z as it was kept
        _, slope, _, slope_off = _activated(z, _rounded(z, z_off, unit, least), name)
        dz, plain_off = d * slope, d.abs() * slope_off + 2.0 ** -23 * d.abs() * slope.abs()
        dz_off = plain_off if name is None else _rounded(dz, plain_off, unit, _held(d, least))
        got["dx"], dx_off = _product(dz, dz_off, w)
        got["dweight"], dw_off = _product(dz.T, dz_off.T, x)
        got["dbias"], db_off = dz.sum(0), plain_off.sum(0) + _sum_off(len(d)) * dz.abs().sum(0)
        off.update({n: _rounded(got[n], o, unit, least) for n, o in (("dx", dx_off), ("dweight", dw_off), ("dbias", db_off))})
    return got, off


def _held(d, least):
    """What is lost of dz below the smallest number.  float16: dz is held times a power of two that takes max |dout| to 16 or more,
    and to below 256."""
    finite = d[torch.isfinite(d)]
    most = float(finite.abs().max()) if finite.numel() else 0.0
    return least * max(most / 16 if most < 16 else 1, most / 128) if least > 2.0 ** -100 else least


def mlp(x, up, down, up_bias=None, down_bias=None, name="silu", gated=True, residual=None, dout=None):
    unit, least = UNIT[x.dtype], LEAST[x.dtype]
    x, u, dn = x.double(), up.double(), down.double()
    none = torch.zeros((), dtype=torch.float64)
    b = none if up_bias is None else up_bias.double()
    z, z_off = _product(x, torch.zeros_like(x), u.T)
    z, z_off = z + b, z_off + 2.0 ** -24 * (z.abs() + b.abs())
    inner = down.shape[1]

    def hidden(z, z_off):
        g, g_off = z[:, :inner], z_off[:, :inner]
        a, slope, a_off, slope_off = _activated(g, g_off, name)
        if not gated:
            return a, a_off, a, a_off, slope, slope_off, torch.ones_like(a), torch.zeros_like(a)
        v, v_off = z[:, inner:], z_off[:, inner:]
        h_off = a_off * v.abs() + a.abs() * v_off + a_off * v_off + 2.0 ** -24 * (a * v).abs()
        return a * v, h_off, a, a_off, slope, slope_off, v, v_off

    h, h_off = hidden(z, z_off)[:2]
    h_off = _rounded(h, h_off, unit, least)
    y, y_off = _product(h, h_off, dn.T)
    for extra in (down_bias, residual):
        if extra is not None:
            y, y_off = y + extra.double(), y_off + 2.0 ** -24 * (y.abs() + extra.double().abs())
    got, off = {"out": y}, {"out": _rounded(y, y_off, unit, least)}
    if dout is not None:
        d = dout.double()
        dh, dh_off = _product(d, torch.zeros_like(d), dn)
        kept = z_off if name is None else _rounded(z, z_off, unit, least)
        if gated:
            kept = _rounded(z, z_off, 2.0 ** -15, 2.0 ** -126)
        _, _, a, a_off, slope, slope_off, v, v_off = hidden(z, kept)
        factor, factor_off = v * slope, v_off * slope.abs() + v.abs() * slope_off + v_off * slope_off
        dz, dz_off = dh * factor, dh_off * (factor.abs() + factor_off) + dh.abs() * factor_off
        if gated:
            dz = torch.cat([dz, dh * a], 1)
            dz_off = torch.cat([dz_off, dh_off * (a.abs() + a_off) + dh.abs() * a_off], 1)
        plain_off = dz_off + 2.0 ** -22 * dz.abs()
        dz_off = _rounded(dz, plain_off, unit, _held(d, least))
        got["dx"], dx_off = _product(dz, dz_off, u)
        got["dup"], du_off = _product(dz.T, dz_off.T, x)
        got["dup_bias"], db_off = dz.sum(0), plain_off.sum(0) + _sum_off(len(d)) * dz.abs().sum(0)
        dd, dd_off = _product(h.T, h_off.T, d)
        got["ddown"], dd_off = dd.T, dd_off.T
        got["ddown_bias"], de_off = d.sum(0), _sum_off(len(d)) * d.abs().sum(0)
        off.update({n: _rounded(got[n], o, unit, least)
                    for n, o in (("dx", dx_off), ("dup", du_off), ("dup_bias", db_off), ("ddown", dd_off), ("ddown_bias", de_off))})
    return got, off


def layer_norm(x, weight=None, bias=None, eps=1e-5, dout=None):
    """Sums over a row go through at most 16 places of a lane and 10 pairings of lanes: they are off by E of their magnitudes."""
    unit, least = UNIT[x.dtype], LEAST[x.dtype]
    E = 2.0 ** -24 * 32
    wide = unit if weight is None else UNIT[weight.dtype]
    x = x.double()
    w = torch.ones((), dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros((), dtype=torch.float64) if bias is None else bias.double()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    variance = (centred * centred).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(variance + eps)
    n = centred * rstd
    mean_off = E * x.abs().mean(1, keepdim=True)
    centred_off = 2.0 ** -24 * centred.abs() + mean_off
    # of the variance: its sum, twice the deviations' own errors (a common one drops out, but for its square)
    variance_off = 2 * E * variance + mean_off ** 2
    # relative to rstd; a variance that drops to or rises from 0 is between its bounds
    low = 1 / torch.sqrt((variance - variance_off).clamp(min=0) + eps)
    rstd_off = (low - rstd).abs() + 2.0 ** -22 * low
    n_off = centred_off * low + centred.abs() * rstd_off + 2.0 ** -24 * n.abs()
    got = {"out": n * w + b, "mean": mean[:, 0], "rstd": rstd[:, 0]}
    off = {"out": _rounded(n * w + b, n_off * w.abs() + 2.0 ** -23 * ((n * w).abs() + b.abs()), unit, least),
           "mean": mean_off[:, 0], "rstd": rstd_off[:, 0]}
    if dout is not None:
        d = dout.double()
        e = d * w
        along = (e * n).mean(1, keepdim=True)
        along_off = E * (e * n).abs().mean(1, keepdim=True) + (e.abs() * n_off).mean(1, keepdim=True)
        inside = e - e.mean(1, keepdim=True) - n * along
        inside_off = 2.0 ** -22 * (e.abs() + (n * along).abs()) + 2 * E * e.abs().mean(1, keepdim=True) + n_off * along.abs() + \
            (n.abs() + n_off) * along_off
        got["dx"] = rstd * inside
        off["dx"] = _rounded(got["dx"], low * inside_off + rstd_off * inside.abs(), unit, least)
        rows = _sum_off(len(x))
        got["dweight"], got["dbias"] = (d * n).sum(0), d.sum(0)
        off["dweight"] = _rounded(got["dweight"], (d.abs() * n_off).sum(0) + rows * (d.abs() * (n.abs() + n_off)).sum(0), wide, least)
        off["dbias"] = _rounded(got["dbias"], rows * d.abs().sum(0), wide, least)
    return got, off
