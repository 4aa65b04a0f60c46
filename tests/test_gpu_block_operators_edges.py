"""Layer norm, linear maps and feed-forward parts on the GPU where their numbers go to the ends of the types, against their
definitions in 64 bits (block_operators_reference.py)."""
import math

import pytest
import torch

from nextdoor_amd import ops
from tests import block_operators_reference as ref
from tests.test_gpu_block_operators import BF16, F16, F32, check_all, linear_case, map_cuda, mlp_case, normal, run_linear, run_mlp, run_norm, within

pytestmark = pytest.mark.gpu

NAMES = ("dx", "dup", "ddown", "dup_bias", "ddown_bias")


# ---- float16: what the gradient of z is held times ------------------------------------------------------------


def largest_dz(case):
    """The largest finite gradient of z."""
    x, up, down, up_bias, _, name, gated, _, d = [t.double() if isinstance(t, torch.Tensor) else t for t in case]
    z = x @ up.T
    if up_bias is not None:
        z = z + up_bias
    dh = d @ down
    g = z[:, :down.shape[1]]
    a, slope = ref.activation(g, name)
    dz = torch.cat([dh * slope * z[:, down.shape[1]:], dh * a], 1) if gated else dh * slope
    return float(dz.abs().max())


def held_by(most):
    """Half the smallest number, over what dz is held times: at least 1, and so much that max |dout| is 512 or more; where the largest
    dz then is no number from 1 to 65504, so much that this is 2^14 or more."""
    def held(d, least):
        return least * max(float(d.abs().max()) / 512 if float(d.abs().max()) < 512 else 1.0, most / 2.0 ** 14)
    return held


def test_gradients_of_z_far_above_dout():
    """One row whose dz is 4096 times dout, which float16 holds, as all the gradients made of it."""
    x, up = torch.full((1, 8), 8.0).to(F16), torch.full((16, 8), 0.25).to(F16)
    down, d = torch.full((512, 8), 0.5).to(F16), torch.ones(1, 512).to(F16)
    got = run_mlp(x, up, down, None, None, "silu", True, None, d)
    # g = u = 16, logistic(16) = 1 - 1.1e-7; dh = 256, dg = du = 4096 to 2e-6, which float16 rounds to 4096
    assert got["dx"].tolist() == [[16 * 4096 * 0.25] * 8] and got["dup"].flatten().tolist() == [4096 * 8.0] * 128
    assert got["dup_bias"].tolist() == [4096.0] * 16


# Both shapes of tile that a backward pass takes two products with in one launch, and the third, that it takes alone; the first two are
# alone where ddown is not wanted.
HELD = [(5, 64, 256, 64), (300, 96, 136, 200), (2050, 64, 256, 64), (20483, 64, 256, 64), (4104, 64, 4096, 1000), (6400, 136, 448, 152),
        (8000, 64, 2048, 1000)]


@pytest.mark.parametrize("rows,dim,inner,out", HELD)
@pytest.mark.parametrize("gated,name", [(True, "silu"), (False, "gelu"), (True, None), (False, None)])
def test_rows_with_gradients_of_z_that_leave_the_range(rows, dim, inner, out, gated, name, monkeypatch):
    """A few rows of large x, with large weights: dz is thousands of times the largest dout in them, and it fits, as dx does."""
    print("held", rows, dim, inner, out, gated, name, flush=True)
    case = mlp_case(rows, dim, inner, out, F16, name, gated)
    x, d = case[0].float(), case[-1].float().clamp(-1, 1)
    large = torch.arange(rows) % (rows // 4 + 1) == 0
    x[large] *= 8 if gated else 1 / 16
    d[~large] /= 16
    # (without a gate dz is dh times a slope: that comes from larger weights alone)
    down = (case[2].float() * (2048 if not gated else 256) * (inner / out) ** 0.5).to(F16)
    case = map_cuda((x.to(F16), case[1], down, *case[3:-1], d.to(F16)))
    most = largest_dz(case)
    assert 2 ** 11 < most < 65504 and case[-1].abs().max() == 1
    monkeypatch.setattr(ref, "_held", held_by(most))
    want, off = ref.mlp(*case)
    got = run_mlp(*case)
    for n, t in got.items():
        assert within(t, want[n], off[n]), n
    x, up, down, up_bias, down_bias, _, _, r, d = case
    _, z, h = ops.mlp_forward(x, up, down, up_bias, down_bias, name, gated, r, keep=True)
    alone = dict(zip(NAMES, ops.mlp_backward(d, x, up, down, z, None, name, gated, True, False, (True, True, False))))
    for n in ("dx", "dup", "dup_bias"):
        assert within(alone[n], want[n], off[n]), ("alone", n)


@pytest.mark.parametrize("rows", [40, 700, 5000])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("big", [1.0, 3e2, 6e4])
def test_small_rows_of_a_feed_forward_part_next_to_large_ones(rows, gated, big):
    """The gradients of rows 10^8 times smaller than the largest have the errors of a rounding or two."""
    case = list(mlp_case(rows, 128, 256, 128, F16, "silu", gated, False, False))
    d = case[-1].float().clamp(-1, 1)
    d[::7] *= big
    small = torch.arange(rows) % 7 != 0
    d[small] *= 1e-3
    case[-1] = d.to(F16)
    want, got = ref.mlp(*case)[0], run_mlp(*case)
    off = (got["dx"].cpu().double() - want["dx"])[small].norm() / want["dx"][small].norm()
    # roundings of dz, of dx and of an ungated z (whose slopes change by less than it does), 2^-11 each at most; what of dz is below 2^-14
    # times the scale (1/4 or more, with dz of 1e-3) is off by 2^-23 of 2^-10
    assert off < 2.0 ** -9
    assert big > 3e2 or torch.isfinite(got["dup"]).all()


@pytest.mark.parametrize("rows", [40, 700, 5000])
@pytest.mark.parametrize("gated", [True, False])
def test_gradients_of_z_far_below_dout(rows, gated):
    """Small weights behind z: the largest dz is below 1, where one row has a large dout."""
    x, up, down, _, _, name, _, _, d = mlp_case(rows, 128, 256, 128, F16, "relu" if not gated else "silu", gated, False, False)
    down = (down.float() * 2.0 ** -16).to(F16)
    up = (up.float() * 16).to(F16)
    d = d.float().clamp(-1, 1)
    d[0] *= 1000 if gated else 20000
    case = (x, up, down, None, None, name, gated, None, d.to(F16))
    assert largest_dz(case) < 1
    want, got = ref.mlp(*case)[0], run_mlp(*case)
    for n, rest in (("dx", slice(1, None)), ("dup", slice(None))):
        off = (got[n].cpu().double() - want[n])[rest].norm() / want[n][rest].norm()
        assert off < 2.0 ** -9, n  # (as above)


@pytest.mark.parametrize("big", [1.0, 3e2, 6e4])
def test_small_rows_of_a_linear_map_next_to_large_ones(big):
    x, w, b, name, r, d = linear_case(200, 128, 256, F16, "gelu")
    d = d.float().clamp(-1, 1)
    d[::2] *= big
    d[1::2] *= 1e-3
    d = d.to(F16)
    want, got = ref.linear(x, w, b, name, r, d)[0], run_linear(x, w, b, name, r, d)
    off = (got["dx"].cpu().double() - want["dx"])[1::2].norm() / want["dx"][1::2].norm()
    assert off < 2.0 ** -9  # (roundings of dz, dx and z, as above)


@pytest.mark.parametrize("rows", [3, 300])
def test_an_infinite_dout_leaves_the_others_their_gradients(rows, monkeypatch):
    """Its row has infinities or NaN; the scale comes from the finite ones, also where they have to be scaled down."""
    case = list(mlp_case(rows, 64, 128, 64, F16, "silu", True, False, False))
    case[2] = (case[2].float() * 512).to(F16)
    want, off = None, None
    d = case[-1].float().clamp(-1, 1)
    bad = d.clone()
    bad[1, 5] = math.inf
    d[1] = 0
    case[-1] = d.to(F16)
    monkeypatch.setattr(ref, "_held", held_by(largest_dz(case)))
    want, off = ref.mlp(*case)
    case[-1] = bad.to(F16)
    got = run_mlp(*case)
    rest = [i for i in range(rows) if i != 1]
    assert not torch.isfinite(got["dx"][1]).any()
    check_all({"dx": got["dx"][rest]}, {"dx": want["dx"][rest]}, {"dx": off["dx"][rest]}, "others")


def test_a_step_that_is_held_anew_is_captured(monkeypatch):
    """Two graphs, replayed in turn over inputs of which some need another scale than their dout's and some do not."""
    case = map_cuda(mlp_case(300, 64, 256, 64, F16, "silu", True))
    x, up, down, up_bias, down_bias, name, gated, r, d = case
    down = down * 256
    inputs = [(x * a, d * b) for a, b in ((1, 1), (0.125, 2.0 ** -8), (4, 1), (1, 2.0 ** -12))]

    def step(x, d):
        out, z, h = ops.mlp_forward(x, up, down, up_bias, down_bias, name, gated, r, keep=True)
        return (out, *ops.mlp_backward(d, x, up, down, z, h, name, gated))
    eager = [step(*i) for i in inputs]
    again = [step(*i) for i in inputs]
    bits = lambda t: t.view(torch.int16)
    assert all(torch.equal(bits(s), bits(t)) for a, b in zip(eager, again) for s, t in zip(a, b))
    gx, gd = torch.empty_like(x), torch.empty_like(d)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = step(gx, gd)
        graphs.append((graph, results))
    for turn in range(8):
        gx.copy_(inputs[turn % 4][0])
        gd.copy_(inputs[turn % 4][1])
        graph, results = graphs[turn % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bits(s), bits(t)) for s, t in zip(eager[turn % 4], results)), turn
        step(*inputs[(turn + 1) % 4])


# ---- every row of a sum counts ----------------------------------------------------------------------------------
# Bounds element by element allow what all roundings could add up to, which for a gradient of weights grows with the rows, its
# values with their root: of these norms a round of 64 rows that is left out is 6 % or more.


def far(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("rows,dim,out", [(13553, 136, 544), (10768, 136, 584), (12017, 2048, 136), (5684, 136, 11280), (4104, 1000, 4096), (958, 528, 16008)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_gradients_leave_no_rows_out(rows, dim, out, dtype):
    print("norms", rows, dim, out, dtype, flush=True)
    x, w, b, name, r, d = map_cuda(linear_case(rows, dim, out, dtype, "silu"))
    want = ref.linear(x, w, b, name, r, d)[0]
    y, z = ops.linear_forward(x, w, b, name, r, keep=True)
    # roundings of z, dz and the result, of a step's half each; they are as random as the values, and add up like them
    unit = 2.0 ** -8 if dtype is BF16 else 2.0 ** -11
    for got in (ops.linear_backward(d, x, w, z, name), ops.linear_backward(d, x, w, z, name, True, (False, True))):
        for n, t in zip(("dx", "dweight", "dbias"), got):
            assert t is None or far(t, want[n]) < 3 * unit, n
    assert far(y, want["out"]) < 2 * unit


@pytest.mark.parametrize("rows,dim,inner,out", [(20483, 64, 256, 64), (6400, 136, 448, 152), (4104, 64, 4096, 1000), (4104, 1000, 4096, 64), (2581, 3480, 8, 8)])
@pytest.mark.parametrize("gated", [True, False])
def test_feed_forward_gradients_leave_no_rows_out(rows, dim, inner, out, gated):
    print("norms", rows, dim, inner, out, gated, flush=True)
    case = map_cuda(mlp_case(rows, dim, inner, out, BF16, "silu", gated, residual=False))
    want, got = ref.mlp(*case)[0], run_mlp(*case)
    for n, t in got.items():
        assert far(t, want[n]) < 3 * 2.0 ** -8, n  # (as above; of out and ddown: h and the result)


# ---- sizes that are filled up -------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,dim", [(3, 64), (100, 64), (700, 136), (70, 4096)])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_infinite_rows_of_a_part_whose_inner_size_is_filled_up(rows, dim, gated, dtype):
    """Of positive numbers all that a row with an infinity makes is infinite, and NaN nowhere: places that are filled up add 0."""
    inner, out = 13, 24
    x, d = normal(1, rows, dim).abs(), normal(2, rows, out).abs()
    up, down = normal(3, inner * (1 + gated), dim, std=dim ** -0.5).abs() + 0.01, normal(4, out, inner, std=0.25).abs() + 0.01
    x, d, up, down = (t.to(dtype) for t in (x, d, up, down))
    case = [x, up, down, None, None, "relu", gated, None, d]
    want, off = ref.mlp(*case)
    case[0] = x.clone()
    case[0][1, 5] = math.inf
    rest = [i for i in range(rows) if i != 1]
    out_ = run_mlp(*case)["out"]
    assert (out_[1] == math.inf).all()
    check_all({"out": out_[rest]}, {"out": want["out"][rest]}, {"out": off["out"][rest]}, "out")
    case[0], case[-1] = x, d.clone()
    case[-1][1, 7] = math.inf
    dx = run_mlp(*case)["dx"]
    assert (dx[1] == math.inf).all()
    check_all({"dx": dx[rest]}, {"dx": want["dx"][rest]}, {"dx": off["dx"][rest]}, "dx")


# ---- rows of layer norm -----------------------------------------------------------------------------------------


def test_the_mean_of_a_row_whose_sum_loses_a_half_step_at_every_addition():
    """1 and, for every addition on its way, what one alone leaves no trace of: 15 places of a lane, 6 pairings of a wave's
    lanes, and the other 15 waves.  A row of 16384 numbers: lanes have runs of four, 4096 places apart."""
    x = torch.zeros(1, 16384)
    x[0, [4096 * turn + i for turn in range(4) for i in range(4)]] = 2.0 ** -24
    x[0, [4 * lane for lane in (1, 2, 4, 8, 16, 32)]] = 2.0 ** -24
    x[0, [4 * 64 * wave for wave in range(1, 16)]] = 2.0 ** -24
    x[0, 0] = 1
    want, off = ref.layer_norm(x)
    mean = ops.layer_norm_forward(x.cuda())[1]
    check_all({"mean": mean}, want, off, "mean")
    # the waves' sums are added four at a time, those in pairs: 15 + 6 + 2 + 3 half steps at most
    assert abs(float(mean) * 16384 - float(x.double().sum())) <= 26 * 2.0 ** -24


@pytest.mark.parametrize("rows,dim", [(1, 64), (100, 64), (768, 64), (769, 64), (48, 1024), (49, 1024), (6, 8192), (5000, 4096), (40007, 24), (3001, 1000)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_gradient_of_rows_alone_is_that_of_all_three_together(rows, dim, dtype):
    x, w, d = normal(1, rows, dim, dtype=dtype).cuda(), normal(2, dim, dtype=dtype).cuda(), normal(3, rows, dim, dtype=dtype).cuda()
    _, mean, rstd = ops.layer_norm_forward(x, w)
    alone = ops.layer_norm_backward(d, x, w, mean, rstd, (True, False, False))[0]
    assert torch.equal(alone, ops.layer_norm_backward(d, x, w, mean, rstd)[0])


# ---- autograd and the model ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("gated", [True, False])
def test_nothing_of_the_inner_size_is_kept_for_what_dout_alone_gives(rows, gated):
    x, up, down, up_bias, down_bias, name, _, r, d = map_cuda(mlp_case(rows, 64, 128, 64, BF16, "silu", gated))
    for wanted in ((down_bias,), (r,), (down_bias, r)):
        for t in (down_bias, r):
            t.grad = None
            t.requires_grad_(any(t is w for w in wanted))
        y = ops.mlp(x, up, down, up_bias, down_bias, name, gated, r)
        assert all(t is None or t.shape != (rows, 128) and t.dtype is BF16 for t in y.grad_fn.saved_tensors)
        y.backward(d)
        for t, right in ((down_bias, d.double().sum(0)), (r, d.double())):
            assert (t.grad is not None) == any(t is w for w in wanted)
            if t.grad is not None:
                assert ((t.grad.double() - right).abs() <= 2.0 ** -8 * right.abs() + (rows + 8) * 2.0 ** -24 * d.double().abs().sum(0)).all()
        down_bias.requires_grad_(False)
        r.requires_grad_(False)


def test_z_and_h_are_asked_for_where_a_gradient_reads_them():
    x, up, down, _, _, name, _, _, d = map_cuda(mlp_case(70, 64, 128, 64))
    _, z, h = ops.mlp_forward(x, up, down, keep=True)
    every = ops.mlp_backward(d, x, up, down, z, h)
    assert torch.equal(ops.mlp_backward(d, x, up, down, None, h, "silu", True, False, True, (False, False, True))[2], every[2])
    got = ops.mlp_backward(d, x, up, down, z, None, "silu", True, True, False, (True, True, False))
    assert all(torch.equal(got[i], every[i]) for i in (0, 1, 3))
    assert torch.equal(ops.mlp_backward(d, x, up, down, None, None, "silu", True, False, True, (False, False, False))[4], every[4])
    for a, b, up_bias, needs, which in ((None, h, False, (True, False, False), "z"), (None, h, False, (False, True, False), "z"),
                                        (None, h, True, (False, False, False), "z"), (z, None, False, (False, False, True), "h"),
                                        (z[1:], h, False, (False, False, False), "z"), (z, h[1:], False, (False, False, False), "h")):
        with pytest.raises(ops.NextDoorError, match="%s is not what" % which):
            ops.mlp_backward(d, x, up, down, a, b, "silu", True, up_bias, True, needs)


def test_every_step_of_the_gated_walk_model_has_the_gradients_of_a_model_that_never_ran():
    """Nothing of the steps before is left in what a step computes; the first step's gradients are tested against the definitions."""
    import copy
    import numpy as np
    from nextdoor_amd import walk_model
    torch.manual_seed(3)
    n = 211
    rng = np.random.default_rng(4)
    model = walk_model.WalkModel(n, width=64, heads=2, kv_heads=1, layers=2, dropout=0.1, gated=True).to("cuda", BF16)
    optimizer = torch.optim.SGD(model.parameters(), lr=0.05)
    for turn in range(4):
        samples = rng.integers(0, n, (40 + 30 * turn, 25)).astype(np.int32)
        for walk in samples[::3]:
            walk[rng.integers(0, 25):] = n
        tokens, targets, starts = walk_model.pack_walks(rng.integers(0, n, len(samples)), samples, n)
        batch = walk_model.batch_of(tokens, targets, starts)
        fresh = walk_model.WalkModel(n, width=64, heads=2, kv_heads=1, layers=2, dropout=0.1, gated=True).to("cuda", BF16)
        fresh.load_state_dict(copy.deepcopy(model.state_dict()))
        losses = []
        for m in (fresh, model):
            m.zero_grad()
            each = m(*batch[:3], batch[3], 17 + turn)
            each.mean().backward()
            losses.append(each.detach())
        assert torch.equal(*losses)
        for (name, a), b in zip(model.named_parameters(), fresh.parameters()):
            assert a.grad.abs().max() > 0, name
            if name.startswith("blocks") or name.startswith("norm"):
                assert torch.equal(a.grad, b.grad), (turn, name)
            else:  # (torch adds up the embeddings' gradients, in an order that it does not promise)
                assert far(a.grad, b.grad) < 2.0 ** -8, (turn, name)
        optimizer.step()


@pytest.mark.parametrize("rows,dim", [(3, 64), (50, 64), (100, 64), (70, 4096), (2500, 520)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_slopes_of_positive_numbers_that_16_bits_do_not_hold(rows, dim, dtype):
    """z of 2^-28 and -2^-28: the slopes of a relu are 1 and 0."""
    x, w = torch.zeros(rows, dim), torch.zeros(40, dim)
    x[:, 3], w[:, 3] = 2.0 ** -14, 2.0 ** -14
    x[::2] *= -1
    x, w, d = x.to(dtype).cuda(), w.to(dtype).cuda(), torch.full((rows, 40), 0.5, dtype=dtype).cuda()
    slope = (torch.arange(rows) % 2).double()
    out, z = ops.linear_forward(x, w, None, "relu", keep=True)
    dx, dw, db = ops.linear_backward(d, x, w, z, "relu")
    # 40 products 0.5 x 2^-14; 0.5 x 2^-14 of every second row; 0.5 of those: sums that 32 bits hold
    assert torch.equal(dx[:, 3].cpu().double(), 40 * 0.5 * 2.0 ** -14 * slope)
    assert dw[:, 3].tolist() == [float(torch.tensor(0.5 * 2.0 ** -14 * int(slope.sum())).to(dtype))] * 40
    assert db.tolist() == [float(torch.tensor(0.5 * int(slope.sum())).to(dtype))] * 40
    assert out.abs().max() <= 2.0 ** -28  # (float16: 0)
    out, z, h = ops.mlp_forward(x, w, torch.ones(8, 40, dtype=dtype).cuda(), activation="relu", gated=False, keep=True)
    dx = ops.mlp_backward(torch.full((rows, 8), 0.25, dtype=dtype).cuda(), x, w, torch.ones(8, 40, dtype=dtype).cuda(), z, h, "relu", False)[0]
    assert torch.equal(dx[:, 3].cpu().double(), 40 * 2 * 2.0 ** -14 * slope)
