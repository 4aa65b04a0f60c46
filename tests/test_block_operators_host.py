"""What layer norm, linear maps and feed-forward parts refuse before a GPU is touched, and their reference's gradients."""
import pytest
import torch

from nextdoor_amd import NextDoorError, _capi, ops
from tests import block_operators_reference as ref

BASE = 1 << 40  # an address that is never dereferenced: every call is refused first


def fill(a, fields, changes):
    for name, value in {**fields, **changes}.items():
        setattr(a, name, value)
    return a


def norm_call(**changes):
    return fill(_capi.LayerNorm(), dict(rows=10, dim=64, dtype=2, weight_dtype=2, eps=1e-5, x_row=64, dout_row=64, x=BASE, weight=BASE,
                                        bias=BASE, out=BASE, mean=BASE, rstd=BASE, dout=BASE, dx=BASE, dweight=BASE, dbias=BASE, workspace=BASE,
                                        workspace_bytes=1 << 40), changes)


def linear_call(**changes):
    return fill(_capi.Linear(), dict(rows=100, dim=64, out_dim=96, dtype=2, activation=2, x_row=64, residual_row=96, dout_row=96, x=BASE,
                                     weight=BASE, bias=BASE, residual=BASE, out=BASE, z=BASE, dout=BASE, dx=BASE, dweight=BASE, dbias=BASE,
                                     workspace=BASE, workspace_bytes=1 << 40), changes)


def mlp_call(**changes):
    return fill(_capi.Mlp(), dict(rows=100, dim=64, inner=128, out_dim=64, dtype=2, activation=4, gated=1, x_row=64, residual_row=64,
                                  dout_row=64, x=BASE, up=BASE, up_bias=BASE, down=BASE, down_bias=BASE, residual=BASE, out=BASE, z=BASE, h=BASE,
                                  dout=BASE, dx=BASE, dup=BASE, dup_bias=BASE, ddown=BASE, ddown_bias=BASE, workspace=BASE,
                                  workspace_bytes=1 << 40), changes)


def refused(fn, a, match):
    assert fn(a, None) != 0, match
    why = _capi.lib().nd_last_error().decode()
    assert match in why, (match, why)


@pytest.mark.parametrize("changes,match", [
    (dict(dtype=3), "type"), (dict(dtype=2, weight_dtype=1), "weights"), (dict(rows=-1), "rows"), (dict(dim=0), "values"),
    (dict(dim=16385), "values"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(x_row=-1), "apart"), (dict(dout_row=-64), "apart"), (dict(x=None), "null"), (dict(mean=None), "null"), (dict(rstd=None), "null"),
    (dict(x=BASE + 1), "aligned"), (dict(weight=BASE + 1), "aligned")])
def test_norm_calls_are_refused(changes, match):
    lib = _capi.lib()
    for fn in (lib.nd_layer_norm_forward, lib.nd_layer_norm_backward):
        refused(fn, norm_call(**changes), match)
        refused(fn, None, "null")


def test_norm_calls_with_nothing_to_do_or_no_room():
    lib = _capi.lib()
    refused(lib.nd_layer_norm_forward, norm_call(out=None), "null")
    refused(lib.nd_layer_norm_backward, norm_call(dout=None), "null")
    for changes in (dict(workspace_bytes=16), dict(workspace=None), dict(workspace=BASE + 8)):
        refused(lib.nd_layer_norm_backward, norm_call(rows=1000, **changes), "workspace")
    refused(lib.nd_layer_norm_backward, norm_call(dx=BASE + 1), "aligned")
    assert lib.nd_layer_norm_forward(norm_call(rows=0, x=None, out=None), None) == 0
    assert lib.nd_layer_norm_backward(norm_call(dx=None, dweight=None, dbias=None), None) == 0
    assert lib.nd_layer_norm_backward(norm_call(rows=0, x=None, dout=None, dweight=None, dbias=None), None) == 0
    assert lib.nd_layer_norm_workspace(norm_call(dim=0)) == -1 and lib.nd_layer_norm_workspace(None) == -1
    room = [lib.nd_layer_norm_workspace(norm_call(rows=1000, **c)) for c in (dict(dweight=None, dbias=None), dict(dbias=None), {})]
    assert room[0] == 0 < room[1] == room[2] and lib.nd_layer_norm_workspace(norm_call()) == 0  # (one workgroup needs none)


COMMON = [(dict(dtype=0), "16-bit"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(dim=12), "multiples of 8"),
          (dict(dim=0), "multiples of 8"), (dict(out_dim=1 << 21), "multiples of 8"), (dict(out_dim=-8), "multiples of 8"),
          (dict(activation=5), "activation"), (dict(activation=-1), "activation"), (dict(x_row=-8), "apart"), (dict(x_row=68), "apart"),
          (dict(residual_row=1 << 23), "apart"), (dict(dout_row=4), "apart")]


@pytest.mark.parametrize("changes,match", COMMON)
def test_linear_calls_are_refused(changes, match):
    lib = _capi.lib()
    for fn in (lib.nd_linear_forward, lib.nd_linear_backward):
        refused(fn, linear_call(**changes), match)
        refused(fn, None, "null")
    assert lib.nd_linear_workspace(linear_call(**changes), 0) == -1 and lib.nd_linear_workspace(None, 1) == -1


def test_linear_calls_without_their_arrays_are_refused():
    lib = _capi.lib()
    for name in ("x", "weight", "out"):
        refused(lib.nd_linear_forward, linear_call(**{name: None}), "null")
    for name in ("x", "weight", "dout", "z"):
        refused(lib.nd_linear_backward, linear_call(**{name: None}), "null")
    for name in ("x", "weight", "bias", "residual", "out", "z"):
        refused(lib.nd_linear_forward, linear_call(**{name: BASE + 8}), "aligned")
    for name in ("x", "weight", "dout", "z", "dx", "dweight", "dbias"):
        refused(lib.nd_linear_backward, linear_call(**{name: BASE + 8}), "aligned")
    for changes in (dict(workspace_bytes=256), dict(workspace=None), dict(workspace=BASE + 8)):
        refused(lib.nd_linear_backward, linear_call(**changes), "workspace")
        refused(lib.nd_linear_forward, linear_call(rows=70, dim=8192, out_dim=64, x_row=8192, **changes), "workspace")
    assert lib.nd_linear_forward(linear_call(rows=0, x=None, weight=None, out=None), None) == 0
    assert lib.nd_linear_backward(linear_call(dx=None, dweight=None, dbias=None), None) == 0


@pytest.mark.parametrize("changes,match", COMMON + [(dict(inner=4), "multiples of 8"), (dict(inner=1 << 20), "inner")])
def test_mlp_calls_are_refused(changes, match):
    lib = _capi.lib()
    for fn in (lib.nd_mlp_forward, lib.nd_mlp_backward):
        refused(fn, mlp_call(**changes), match)
        refused(fn, None, "null")
    assert lib.nd_mlp_workspace(mlp_call(**changes), 0) == -1 and lib.nd_mlp_workspace(None, 1) == -1


def test_mlp_calls_without_their_arrays_are_refused():
    lib = _capi.lib()
    for name in ("x", "up", "down", "out", "h"):
        refused(lib.nd_mlp_forward, mlp_call(**{name: None}), "null")
    for name in ("x", "up", "down", "dout", "z", "h"):
        refused(lib.nd_mlp_backward, mlp_call(**{name: None}), "null")
    for name in ("x", "up", "up_bias", "down", "down_bias", "residual", "out", "z", "h"):
        refused(lib.nd_mlp_forward, mlp_call(**{name: BASE + 8}), "aligned")
    for name in ("dx", "dup", "dup_bias", "ddown", "ddown_bias"):
        refused(lib.nd_mlp_backward, mlp_call(**{name: BASE + 8}), "aligned")
    for changes in (dict(workspace_bytes=256), dict(workspace=None), dict(workspace=BASE + 8)):
        refused(lib.nd_mlp_backward, mlp_call(**changes), "workspace")
    assert lib.nd_mlp_forward(mlp_call(rows=0, x=None, up=None, down=None, out=None, h=None), None) == 0
    assert lib.nd_mlp_backward(mlp_call(dx=None, dup=None, dup_bias=None, ddown=None, ddown_bias=None), None) == 0


def test_tensors_on_the_host_are_refused():
    x, w = torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(32, 32, dtype=torch.bfloat16)
    row = torch.zeros(4)
    for call in (lambda: ops.layer_norm(x), lambda: ops.layer_norm_forward(x), lambda: ops.layer_norm_backward(x, x, None, row, row),
                 lambda: ops.linear(x, w), lambda: ops.linear_forward(x, w), lambda: ops.linear_backward(x, x, w),
                 lambda: ops.mlp(x, w, w, gated=False), lambda: ops.mlp_forward(x, w, w, gated=False),
                 lambda: ops.mlp_backward(x, x, w, w, x, x), lambda: ops.layer_norm_forward([1.0]), lambda: ops.linear_forward(x.numpy, w)):
        with pytest.raises(NextDoorError, match="GPU"):
            call()


def moved(tensors, i, direction, step):
    return [t + step * direction if j == i else t for j, t in enumerate(tensors)]


class Doubles:
    """The reference takes the types of its inputs for its bounds; here all is in 64 bits."""

    def __enter__(self):
        self.kept = ref.UNIT, ref.LEAST
        ref.UNIT, ref.LEAST = ({**d, torch.float64: 0.0} for d in self.kept)

    def __exit__(self, *_):
        ref.UNIT, ref.LEAST = self.kept


def check_gradients(fn, tensors, names, d):
    """fn's gradients against differences of its own outputs."""
    gen = torch.Generator().manual_seed(11)
    with Doubles():
        got = fn(*tensors, d)[0]
        for i, name in enumerate(names):
            direction = torch.randn(tensors[i].shape, generator=gen, dtype=torch.float64)
            value = [float((fn(*moved(tensors, i, direction, s * 1e-5), None)[0]["out"] * d).sum()) for s in (1, -1)]
            assert abs((value[0] - value[1]) / 2e-5 - float((got[name] * direction).sum())) < 1e-5, name


def random(*shapes):
    gen = torch.Generator().manual_seed(3)
    return [torch.randn(s, generator=gen, dtype=torch.float64) for s in shapes]


@pytest.mark.parametrize("name", [None, "relu", "gelu", "gelu_tanh", "silu"])
def test_reference_gradients_are_the_derivatives(name):
    x, w, b, d = random((6, 9), (7, 9), (7,), (6, 7))
    check_gradients(lambda x, w, b, d: ref.linear(x, w, b, name, None, d), (x, w, b), ("dx", "dweight", "dbias"), d)
    for gated in (True, False):
        x, up, down, a, b, d = random((6, 5), (8 * (1 + gated), 5), (4, 8), (8 * (1 + gated),), (4,), (6, 4))
        check_gradients(lambda x, up, down, a, b, d: ref.mlp(x, up, down, a, b, name, gated, None, d), (x, up, down, a, b),
                        ("dx", "dup", "ddown", "dup_bias", "ddown_bias"), d)


def test_reference_norm_gradients_are_the_derivatives():
    x, w, b, d = random((5, 12), (12,), (12,), (5, 12))
    check_gradients(lambda x, w, b, d: ref.layer_norm(x, w, b, 1e-2, d), (x, w, b), ("dx", "dweight", "dbias"), d)


def test_reference_activations_are_torchs():
    z = torch.linspace(-9, 9, 1001, dtype=torch.float64)
    f = torch.nn.functional
    for name, of in (("relu", f.relu), ("gelu", f.gelu), ("gelu_tanh", lambda z: f.gelu(z, approximate="tanh")), ("silu", f.silu)):
        assert (ref.activation(z, name)[0] - of(z)).abs().max() < 1e-14
        slope = ref.activation(z, name)[1]
        assert slope.abs().max() < ref.MOST_SLOPE
        if name != "relu":
            assert ((slope[1:] - slope[:-1]) / (z[1:] - z[:-1])).abs().max() < ref.MOST_CURVATURE
