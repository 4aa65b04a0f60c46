"""Layer norm, linear maps and feed-forward parts: what torch asks of them beside their values, without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from nextdoor_amd import _capi, ops
from tests import block_operators_reference as ref
from tests.test_block_operators_host import mlp_call, refused


@pytest.fixture
def without_kernels(monkeypatch):
    """The forward functions give something of the right shape; what is kept for a backward pass is None."""
    def norm(x, weight=None, bias=None, eps=1e-5):
        return 2 * x.detach(), None, None

    def linear(x, weight, bias=None, activation=None, residual=None, keep=False):
        out = x.detach() @ weight.detach().T
        return (out, None) if keep else out

    def mlp(x, up, down, up_bias=None, down_bias=None, activation="silu", gated=True, residual=None, keep=False):
        out = x.detach() @ down.detach().T
        return (out, None, None) if keep else out
    for name, function in (("layer_norm_forward", norm), ("linear_forward", linear), ("mlp_forward", mlp)):
        monkeypatch.setattr(ops, name, function)


CALLS = [("x", lambda x, w: ops.layer_norm(x)), ("x", lambda x, w: ops.linear(x, w)), ("weight", lambda x, w: ops.linear(x, w)),
         ("x", lambda x, w: ops.mlp(x, w, w, gated=False)), ("weight", lambda x, w: ops.mlp(x, w, w, gated=False))]


@pytest.mark.parametrize("which,call", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused_and_not_lost(without_kernels, which, call, grad):
    """no_grad switches gradients off, and not forward mode: without a tangent the result would count as constant."""
    x, w = torch.ones(4, 8), torch.ones(8, 8)
    with torch.set_grad_enabled(grad):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x if which == "x" else w, torch.ones(4 if which == "x" else 8, 8))
            with pytest.raises((NotImplementedError, RuntimeError), match="forward mode|jvp"):
                call(dual, w) if which == "x" else call(x, dual)
        of = (lambda t: call(t, w)) if which == "x" else (lambda t: call(x, t))
        at = x if which == "x" else w
        with pytest.raises(RuntimeError):
            torch.func.jvp(of, (at,), (at,))
        assert call(x, w).shape == (4, 8) and not call(x, w).requires_grad


@pytest.mark.parametrize("filled", [-1, 128, 1 << 20])
def test_more_filled_up_places_than_there_are_is_refused(filled):
    lib = _capi.lib()
    for fn in (lib.nd_mlp_forward, lib.nd_mlp_backward):
        refused(fn, mlp_call(inner_filled=filled), "filled up")
    assert lib.nd_mlp_workspace(mlp_call(inner_filled=filled), 0) == -1
    assert lib.nd_mlp_workspace(mlp_call(inner_filled=7), 1) == lib.nd_mlp_workspace(mlp_call(), 1) > 0


@pytest.mark.parametrize("dtype,unit", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_norms_notice_a_quarter_of_a_round_that_a_sum_over_rows_leaves_out(dtype, unit):
    """The bound of the GPU tests on the norm of a weight's gradient, 3 half steps, with the kernels' roundings done here."""
    rows, lost = 13553, 16
    gen = torch.Generator().manual_seed(6)
    x, d = torch.randn(rows, 40, generator=gen).to(dtype).double(), torch.randn(rows, 48, generator=gen).to(dtype).double()
    w = (torch.randn(48, 40, generator=gen) / 40 ** 0.5).to(dtype).double()
    z = x @ w.T
    want = (d * ref.activation(z, "silu")[1]).T @ x
    dz = (d * ref.activation(z.to(dtype).double(), "silu")[1]).to(dtype).double()
    off = [float(((dz[:n].T @ x[:n]).to(dtype).double() - want).norm() / want.norm()) for n in (rows, rows - lost)]
    assert off[0] < 3 * unit < off[1]
