"""Layer norm, linear maps and feed-forward parts on the GPU, against their definitions in 64 bits (block_operators_reference.py)."""
import math

import pytest
import torch

from nextdoor_amd import _capi, ops
from tests import block_operators_reference as ref
from tests.operators_reference import close

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ACTIVATIONS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def normal(seed, *shape, dtype=BF16, std=1.0, mean=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * std + mean).to(dtype)


def cuda(x):
    return None if x is None else x.cuda()


def same_bits(a, b):
    kind = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.view(kind), b.view(kind))


def check_all(got, want, off, what):
    for name in got:
        if got[name] is None:
            continue
        value, right = got[name].cpu().double(), want[name]
        if got[name].dtype is F16:
            # the largest 16-bit float is 65504, the next one would be 65536: what is 65520 or more is rounded to infinity
            beyond = torch.isinf(value) & (right.abs() + off[name] >= 65520) & (value.sign() == right.sign())
            value = torch.where(beyond, right, value)
        assert close(value, right, off[name]), (what, name)


# ---- layer norm ------------------------------------------------------------------------------------------


def run_norm(x, weight, bias, dout, eps=1e-5):
    out, mean, rstd = ops.layer_norm_forward(cuda(x), cuda(weight), cuda(bias), eps)
    dx, dweight, dbias = ops.layer_norm_backward(cuda(dout), cuda(x), cuda(weight), mean, rstd)
    torch.cuda.synchronize()
    return {"out": out, "mean": mean, "rstd": rstd, "dx": dx, "dweight": dweight, "dbias": dbias}


@pytest.mark.parametrize("dim", [1, 2, 7, 8, 64, 100, 128, 129, 512, 513, 1000, 1021, 1024, 1025, 2048, 3001, 4096, 4104, 8192, 9999, 16384])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_of_rows_of_every_size(dim, dtype):
    rows = 37 if dim < 4096 else 5
    x = (normal(1, rows, dim, dtype=F32) * torch.exp(normal(2, rows, 1, dtype=F32)) + 0.5).to(dtype)
    w, b, d = normal(3, dim, dtype=dtype, mean=1.0, std=0.3), normal(4, dim, dtype=dtype), normal(5, rows, dim, dtype=dtype)
    want, off = ref.layer_norm(x, w, b, 1e-5, d)
    check_all(run_norm(x, w, b, d), want, off, (dim, dtype))


@pytest.mark.parametrize("dim", [3, 4, 5, 9, 15, 16, 17, 63, 65, 66, 127, 130, 255, 256, 257, 264, 1023, 2047, 2049, 4095, 8191, 8193, 16381])
@pytest.mark.parametrize("dtype,weights", [(BF16, BF16), (F16, F32), (F32, F32)])
def test_norm_of_rows_between_others(dim, dtype, weights):
    """Rows whose beginnings have the alignment of an element only, and NaN on both sides of them."""
    rows = 70 if dim < 2049 else 5
    def between(t, step):
        room = torch.full((*t.shape[:-1], dim + step), math.nan, dtype=t.dtype)
        room[..., 1:dim + 1] = t
        return room.cuda()[..., 1:dim + 1]
    x, d = normal(1, rows, dim, dtype=dtype, mean=0.5), normal(2, rows, dim, dtype=dtype)
    w, b = normal(3, dim, dtype=weights, mean=1.0, std=0.3), normal(4, dim, dtype=weights)
    want, off = ref.layer_norm(x, w, b, 1e-5, d)
    gx, gd, gw, gb = between(x, 3), between(d, 2), between(w, 2), between(b, 2)
    out, mean, rstd = ops.layer_norm_forward(gx, gw, gb, 1e-5)
    got = ops.layer_norm_backward(gd, gx, gw, mean, rstd)
    torch.cuda.synchronize()
    check_all(dict(zip(("out", "dx", "dweight", "dbias"), (out, *got))), want, off, (dim, dtype))


@pytest.mark.parametrize("rows,dim", [(0, 64), (1, 64), (1, 1024), (2049, 64), (40007, 24), (9001, 96), (3001, 1000), (1501, 1032)])
def test_norm_of_any_number_of_rows(rows, dim):
    x, w, b, d = normal(1, rows, dim), normal(2, dim), normal(3, dim), normal(4, rows, dim)
    want, off = ref.layer_norm(x, w, b, 1e-5, d)
    check_all(run_norm(x, w, b, d), want, off, (rows, dim))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("which", ["neither", "weight", "bias", "32 bits"])
def test_norm_with_other_weights(dtype, which):
    x, d = normal(1, 65, 200, dtype=dtype), normal(2, 65, 200, dtype=dtype)
    kind = F32 if which == "32 bits" else dtype
    w = None if which in ("neither", "bias") else normal(3, 200, dtype=kind)
    b = None if which in ("neither", "weight") else normal(4, 200, dtype=kind)
    want, off = ref.layer_norm(x, w, b, 1e-3, d)
    got = run_norm(x, w, b, d, 1e-3)
    assert got["dweight"].dtype is got["dbias"].dtype is (dtype if w is None else kind)
    check_all(got, want, off, which)


def test_norm_reads_slices_and_copies_other_orders():
    whole = normal(1, 50, 300)
    w, b = normal(2, 100), normal(3, 100)
    d = normal(4, 50, 100)
    for cut in (slice(0, 100), slice(104, 204), slice(33, 133)):
        x = whole[:, cut]
        want, off = ref.layer_norm(x, w, b, 1e-5, d)
        gpu = whole.cuda()[:, cut]
        assert ops._rows_in_place(gpu, 100, 1)[0] is gpu
        out, mean, rstd = ops.layer_norm_forward(gpu, w.cuda(), b.cuda())
        dx, dw, db = ops.layer_norm_backward(d.cuda(), gpu, w.cuda(), mean, rstd)
        check_all({"out": out, "dx": dx, "dweight": dw, "dbias": db}, want, off, cut)
    x = normal(5, 100, 50).t()
    want, off = ref.layer_norm(x, w, b, 1e-5, d)
    check_all(run_norm(x, w, b, d), want, off, "transposed")
    one = normal(6, 1, 100)
    want, off = ref.layer_norm(one.expand(50, 100), w, b, 1e-5, d[:1].expand(50, 100))
    out, mean, rstd = ops.layer_norm_forward(one.cuda().expand(50, 100), w.cuda(), b.cuda())
    dx, dw, db = ops.layer_norm_backward(d[:1].cuda().expand(50, 100), one.cuda().expand(50, 100), w.cuda(), mean, rstd)
    check_all({"out": out, "dx": dx, "dweight": dw, "dbias": db}, want, off, "the same row")
    x = normal(7, 3, 4, 5, 64)
    out, _, _ = ops.layer_norm_forward(x.cuda())
    want, off = ref.layer_norm(x.reshape(60, 64))
    assert out.shape == x.shape and close(out.reshape(60, 64), want["out"], off["out"])


def test_norm_of_rows_that_are_constant_far_from_zero_or_not_finite():
    x = normal(1, 8, 256, dtype=F32)
    x[1] = 3.0
    x[2] = 0.0
    x[3] += 1000.0
    x[4] *= 1e-4
    x[5] *= 1e15
    w, b, d = normal(2, 256, dtype=F32), normal(3, 256, dtype=F32), normal(4, 8, 256, dtype=F32)
    want, off = ref.layer_norm(x, w, b, 1e-5, d)
    check_all(run_norm(x, w, b, d), want, off, "odd rows")
    x[6, 17] = math.inf
    x[7, 3] = math.nan
    got = run_norm(x, w, b, d)
    for name in ("out", "dx"):
        assert torch.isnan(got[name][6:]).all() and close(got[name][:6], want[name][:6], off[name][:6])


def test_norm_gradients_that_are_not_wanted_are_not_made():
    x, w, d = normal(1, 40, 64).cuda(), normal(2, 64).cuda(), normal(3, 40, 64).cuda()
    _, mean, rstd = ops.layer_norm_forward(x, w)
    all_of_them = ops.layer_norm_backward(d, x, w, mean, rstd)
    for needs in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (False, False, False)):
        got = ops.layer_norm_backward(d, x, w, mean, rstd, needs)
        for g, a, need in zip(got, all_of_them, needs):
            assert (g is None) != need and (g is None or torch.equal(g, a))


# ---- linear -----------------------------------------------------------------------------------------------


def run_linear(x, weight, bias=None, name=None, residual=None, dout=None):
    x, weight, bias, residual, dout = map(cuda, (x, weight, bias, residual, dout))
    out, z = ops.linear_forward(x, weight, bias, name, residual, keep=True)
    got = {"out": out}
    assert same_bits(out, ops.linear_forward(x, weight, bias, name, residual))
    if dout is not None:
        got["dx"], got["dweight"], got["dbias"] = ops.linear_backward(dout, x, weight, z, name)
    torch.cuda.synchronize()
    return got


def linear_case(rows, dim, out, dtype=BF16, name=None, bias=True, residual=False, std=1.0):
    return (normal(1, rows, dim, dtype=dtype, std=std), normal(2, out, dim, dtype=dtype, std=dim ** -0.5),
            normal(3, out, dtype=dtype, std=0.3) if bias else None, name, normal(4, rows, out, dtype=dtype) if residual else None,
            normal(5, rows, out, dtype=dtype))


# Few rows (one, two and four blocks of 16), each size of tile, sums in shares and whole, rounds that end inside, one round and
# less than the tiles' stages, sizes around every edge.
SIZES = [(1, 8, 8), (1, 1024, 4096), (2, 72, 40), (15, 136, 24), (16, 64, 64), (17, 200, 120), (33, 520, 264), (64, 1032, 1000), (65, 64, 64),
         (100, 8, 16), (128, 64, 128), (129, 72, 136), (63, 2048, 8), (255, 256, 256), (257, 264, 520), (1021, 520, 1000), (300, 1000, 64),
         (70, 4096, 72), (2048, 512, 2048), (2051, 136, 2056), (5000, 64, 192), (4999, 192, 64), (700, 3080, 640)]


@pytest.mark.parametrize("rows,dim,out", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_of_many_sizes(rows, dim, out, dtype):
    print("linear", rows, dim, out, dtype, flush=True)
    x, w, b, name, r, d = linear_case(rows, dim, out, dtype, "gelu", residual=True)
    want, off = ref.linear(x, w, b, name, r, d)
    check_all(run_linear(x, w, b, name, r, d), want, off, (rows, dim, out))


@pytest.mark.parametrize("rows", [0, 3, 200, 1100])
@pytest.mark.parametrize("name", ACTIVATIONS)
@pytest.mark.parametrize("bias,residual,dtype", [(True, False, BF16), (False, True, BF16), (False, False, F16), (True, True, F16)])
def test_linear_with_every_activation(rows, name, bias, residual, dtype):
    x, w, b, name, r, d = linear_case(rows, 96, 320, dtype, name, bias, residual, std=2.0)
    want, off = ref.linear(x, w, b, name, r, d)
    check_all(run_linear(x, w, b, name, r, d), want, off, (rows, name))


@pytest.mark.parametrize("rows,dim,out", [(5, 1, 1), (7, 13, 100), (90, 100, 13), (300, 77, 301)])
def test_linear_of_sizes_that_are_no_multiples_of_8(rows, dim, out):
    x, w, b, name, r, d = linear_case(rows, dim, out, BF16, "silu", residual=True)
    want, off = ref.linear(x, w, b, name, r, d)
    got = run_linear(x, w, b, name, r, d)
    assert got["dx"].shape == x.shape and got["dweight"].shape == w.shape and got["dbias"].shape == b.shape
    check_all(got, want, off, (rows, dim, out))


@pytest.mark.parametrize("rows", [20, 300])
def test_linear_reads_slices_in_place_and_nothing_around_them(rows):
    """The rest of the buffers holds NaN."""
    x, w, b, name, r, d = linear_case(rows, 72, 200, BF16, "gelu", residual=True)
    want, off = ref.linear(x, w, b, name, r, d)

    def inside(t):
        whole = torch.full((t.shape[0] + 2, t.shape[1] + 24), math.nan, dtype=t.dtype, device="cuda")
        part = whole[1:-1, 8:-16]
        part.copy_(t)
        return part
    gx, gr, gd = inside(x), inside(r), inside(d)
    assert ops._vectors_in_place(gx, 72)[0] is gx
    out, z = ops.linear_forward(gx, w.cuda(), b.cuda(), name, gr, keep=True)
    dx, dw, db = ops.linear_backward(gd, gx, w.cuda(), z, name)
    check_all({"out": out, "dx": dx, "dweight": dw, "dbias": db}, want, off, "inside")
    # other orders, odd beginnings, the same row again and again
    others = [t.cuda().t().contiguous().t() for t in (x, r, d)]
    out, z = ops.linear_forward(others[0], w.cuda().t().contiguous().t(), b.cuda(), name, others[1], keep=True)
    got = ops.linear_backward(others[2], others[0], w.cuda(), z, name)
    check_all(dict(zip(("out", "dx", "dweight", "dbias"), (out, *got))), want, off, "by columns")
    odd = torch.zeros(rows, 73, dtype=BF16, device="cuda")
    odd[:, 1:] = x.cuda()
    assert torch.equal(ops.linear_forward(odd[:, 1:], w.cuda(), b.cuda(), name, gr), out)
    one = normal(9, 1, 200)
    want, off = ref.linear(x, w, b, name, one.expand(rows, 200), one.expand(rows, 200))
    out, z = ops.linear_forward(x.cuda(), w.cuda(), b.cuda(), name, one.cuda().expand(rows, 200), keep=True)
    got = ops.linear_backward(one.cuda().expand(rows, 200), x.cuda(), w.cuda(), z, name)
    check_all(dict(zip(("out", "dx", "dweight", "dbias"), (out, *got))), want, off, "one row")


@pytest.mark.parametrize("rows,dim,out", [(9, 64, 48), (150, 200, 136), (1100, 520, 1000)])
def test_linear_keeps_infinities_and_nan_to_the_rows_that_hold_them(rows, dim, out):
    x, w, b, name, r, d = linear_case(rows, dim, out, BF16, None)
    x[3, 5], x[rows - 1, dim - 1], x[7, 0] = math.nan, math.inf, -math.inf
    got = run_linear(x, w, b, name, r, d)["out"].cpu()
    kept = torch.ones(rows, dtype=torch.bool)
    kept[[3, 7, rows - 1]] = False
    assert not torch.isfinite(got[~kept]).any()
    x[~kept] = 0
    want, off = ref.linear(x, w, b, name, r)
    assert close(got[kept], want["out"][kept], off["out"][kept])
    # of the gradients: a row of dout sends it to its row of dx, a column to its row of dweight
    d[3, 5], d[rows - 1, out - 1] = math.nan, math.inf
    dx, dw, db = ops.linear_backward(d.cuda(), x.cuda(), w.cuda())
    assert not torch.isfinite(dx[[3, rows - 1]]).any() and torch.isfinite(dx).sum() == (rows - 2) * dim
    odd = torch.isfinite(db).logical_not().nonzero().flatten().tolist()
    assert odd == [5, out - 1] and torch.isfinite(dw[[i for i in range(out) if i not in odd]]).all()


@pytest.mark.parametrize("rows,name", [(30, "gelu"), (400, "gelu"), (400, "relu"), (400, "silu")])
@pytest.mark.parametrize("factor", [2.0 ** -18, 2.0 ** -10, 2.0 ** 10])
def test_linear_gradients_of_small_and_large_16_bit_floats(rows, name, factor):
    """What comes back for a mean over many rows: sums of it are in range where each part is not."""
    x, w, b, name, r, d = linear_case(rows, 128, 256, F16, name)
    d = (d.float() * factor).to(F16)
    want, off = ref.linear(x, w, b, name, r, d)
    check_all(run_linear(x, w, b, name, r, d), want, off, factor)


def test_an_infinite_gradient_does_not_take_the_others_their_scale():
    x, w, b, name, r, d = linear_case(300, 128, 256, F16, "gelu")
    d = (d.float() * 2.0 ** -18).to(F16)
    d[5, 7] = math.inf
    out, z = ops.linear_forward(x.cuda(), w.cuda(), b.cuda(), name, keep=True)
    dx, dw, db = ops.linear_backward(d.cuda(), x.cuda(), w.cuda(), z, name)
    d[5] = 0
    want, off = ref.linear(x, w, b, name, r, d)
    rows = [i for i in range(300) if i != 5]
    assert not torch.isfinite(dx[5]).any() and close(dx[rows], want["dx"][rows], off["dx"][rows])
    assert not torch.isfinite(dw[7]).any() and not torch.isfinite(db[7])


def test_linear_gradients_that_are_not_wanted_are_not_made():
    for name in (None, "gelu"):
        x, w, b, _, r, d = map(cuda, (*linear_case(200, 64, 96, BF16, None)[:3], None, None, linear_case(200, 64, 96)[5]))
        _, z = ops.linear_forward(x, w, b, name, keep=True)
        everything = ops.linear_backward(d, x, w, z, name)
        for with_bias, needs in ((False, (True, True)), (True, (False, True)), (True, (True, False)), (True, (False, False)),
                                 (False, (False, False))):
            got = ops.linear_backward(d, x, w, z, name, with_bias, needs)
            for g, a, need in zip(got, everything, (*needs, with_bias)):
                assert (g is None) != need and (g is None or torch.equal(g, a))


def test_linear_of_more_dimensions():
    x, w, r = normal(1, 3, 5, 7, 64), normal(2, 40, 64, std=0.1), normal(3, 3, 5, 7, 40)
    got = ops.linear(x.cuda(), w.cuda(), None, "silu", r.cuda())
    want, off = ref.linear(x.reshape(105, 64), w, None, "silu", r.reshape(105, 40))
    assert got.shape == (3, 5, 7, 40) and close(got.reshape(105, 40), want["out"], off["out"])
    assert ops.linear(x.cuda()[0, 0, 0], w.cuda()).shape == (40,)
    assert ops.linear(x.cuda()[:0], w.cuda()).shape == (0, 5, 7, 40)


# ---- mlp ----------------------------------------------------------------------------------------------------


def run_mlp(x, up, down, up_bias=None, down_bias=None, name="silu", gated=True, residual=None, dout=None):
    x, up, down, up_bias, down_bias, residual, dout = map(cuda, (x, up, down, up_bias, down_bias, residual, dout))
    out, z, h = ops.mlp_forward(x, up, down, up_bias, down_bias, name, gated, residual, keep=True)
    got = {"out": out}
    assert same_bits(out, ops.mlp_forward(x, up, down, up_bias, down_bias, name, gated, residual))
    if dout is not None:
        got.update(zip(("dx", "dup", "ddown", "dup_bias", "ddown_bias"), ops.mlp_backward(dout, x, up, down, z, h, name, gated)))
    torch.cuda.synchronize()
    return got


def mlp_case(rows, dim, inner, out, dtype=BF16, name="silu", gated=True, bias=True, residual=True):
    wide = inner * (1 + gated)
    return (normal(1, rows, dim, dtype=dtype), normal(2, wide, dim, dtype=dtype, std=dim ** -0.5),
            normal(3, out, inner, dtype=dtype, std=inner ** -0.5), normal(4, wide, dtype=dtype, std=0.3) if bias else None,
            normal(5, out, dtype=dtype, std=0.3) if bias else None, name, gated, normal(6, rows, out, dtype=dtype) if residual else None,
            normal(7, rows, out, dtype=dtype))


@pytest.mark.parametrize("rows,dim,inner,out", [(1, 8, 8, 8), (1, 1024, 2816, 1024), (16, 64, 256, 64), (17, 136, 104, 72), (40, 72, 200, 136),
                                                (64, 256, 688, 256), (65, 64, 256, 64), (129, 200, 520, 72), (1000, 64, 256, 64),
                                                (3001, 328, 1000, 328), (2050, 512, 1032, 520), (260, 2048, 264, 8)])
@pytest.mark.parametrize("gated,dtype", [(True, BF16), (False, BF16), (True, F16)])
def test_mlp_of_many_sizes(rows, dim, inner, out, gated, dtype):
    print("mlp", rows, dim, inner, out, gated, dtype, flush=True)
    case = mlp_case(rows, dim, inner, out, dtype, "gelu", gated)
    want, off = ref.mlp(*case)
    check_all(run_mlp(*case), want, off, (rows, dim, inner, out))


@pytest.mark.parametrize("rows", [0, 5, 333])
@pytest.mark.parametrize("name", ACTIVATIONS)
@pytest.mark.parametrize("gated,bias,residual,dtype", [(True, False, True, BF16), (False, True, False, BF16), (True, True, False, F16),
                                                       (False, False, True, F16)])
def test_mlp_with_every_activation(rows, name, gated, bias, residual, dtype):
    case = mlp_case(rows, 96, 256, 96, dtype, name, gated, bias, residual)
    want, off = ref.mlp(*case)
    check_all(run_mlp(*case), want, off, (rows, name))


@pytest.mark.parametrize("rows,dim,inner,out", [(5, 1, 1, 1), (90, 100, 13, 30), (300, 77, 301, 77)])
@pytest.mark.parametrize("gated", [True, False])
def test_mlp_of_sizes_that_are_no_multiples_of_8(rows, dim, inner, out, gated):
    case = mlp_case(rows, dim, inner, out, BF16, "silu", gated)
    want, off = ref.mlp(*case)
    got = run_mlp(*case)
    for name, like in zip(("dx", "dup", "ddown", "dup_bias", "ddown_bias"), case):
        assert got[name].shape == like.shape
    check_all(got, want, off, (rows, dim, inner, out))


@pytest.mark.parametrize("factor", [2.0 ** -18, 2.0 ** -10, 2.0 ** 8])
def test_mlp_gradients_of_small_and_large_16_bit_floats(factor):
    case = list(mlp_case(400, 128, 256, 128, F16, "silu"))
    case[-1] = (case[-1].float() * factor).to(F16)
    want, off = ref.mlp(*case)
    check_all(run_mlp(*case), want, off, factor)


def test_mlp_reads_slices_in_place_and_gives_what_is_wanted():
    case = mlp_case(150, 64, 256, 64)
    want, off = ref.mlp(*case)
    x, up, down, up_bias, down_bias, name, gated, r, d = [t.cuda() if isinstance(t, torch.Tensor) else t for t in case]
    whole = torch.full((150, 3, 88), math.nan, dtype=BF16, device="cuda")
    for i, t in enumerate((x, r, d)):
        whole[:, i, 8:72] = t
    x, r, d = whole[:, 0, 8:72], whole[:, 1, 8:72], whole[:, 2, 8:72]
    out, z, h = ops.mlp_forward(x, up, down, up_bias, down_bias, name, gated, r, keep=True)
    everything = ops.mlp_backward(d, x, up, down, z, h, name, gated)
    names = ("dx", "dup", "ddown", "dup_bias", "ddown_bias")
    check_all({"out": out, **dict(zip(names, everything))}, want, off, "slices")
    for needs in ((False, True, True), (True, False, False), (False, False, True), (False, False, False)):
        for biases in ((False, False), (True, False), (False, True)):
            got = ops.mlp_backward(d, x, up, down, z, h, name, gated, *biases, needs)
            for g, a, need in zip(got, everything, (*needs, *biases)):
                assert (g is None) != need and (g is None or torch.equal(g, a))


# ---- the ends of the ranges -----------------------------------------------------------------------------------


@pytest.mark.parametrize("big", [1.0, 3e2, 6e4])
def test_small_rows_next_to_large_ones_keep_their_gradients(big):
    """16-bit floats: what all rows of the gradient of z are held times does not lose the smaller ones."""
    x, w, b, name, r, d = linear_case(200, 128, 256, F16, "gelu")
    d = d.float().clamp(-1, 1)
    d[::2] *= big
    d[1::2] *= 1e-3
    d = d.to(F16)
    want, off = ref.linear(x, w, b, name, r, d)
    got = run_linear(x, w, b, name, r, d)
    check_all({n: got[n] for n in ("out", "dx", "dbias")}, want, off, big)
    small = (got["dx"].cpu().double() - want["dx"])[1::2].norm() / want["dx"][1::2].norm()
    # roundings of the gradient of z and of the result, 2^-11 each; z's own has a slope below 1; above 256 the last bits are cut
    assert small < (2.0 ** -9 if big <= 256 else 2.0 ** -4)


def test_slopes_of_pre_activations_of_any_size():
    """z from 1e-30 to 1e30: slopes are 0 or 1 at the ends, and never NaN."""
    sizes = torch.logspace(-30, 30, 61)
    x = torch.zeros(122, 64)
    x[:61, 0], x[61:, 0] = sizes, -sizes
    x, w = x.to(BF16), torch.zeros(16, 64)
    w[:, 0] = 1
    w = w.to(BF16)
    d = torch.ones(122, 16, dtype=BF16)
    for name in ACTIVATIONS:
        want, off = ref.linear(x, w, None, name, None, d)
        got = run_linear(x, w, None, name, None, d)
        assert torch.isfinite(got["dx"]).all()
        slope = got["dx"][:, 0].cpu().double() / 16
        exact = ref.activation(x[:, 0].double(), name)[1]
        exact = torch.where(torch.isfinite(exact), exact, torch.where(x[:, 0] > 0, 1.0, 0.0).double())
        assert (slope - exact).abs().max() < 2.0 ** -6, name
        up = torch.cat([w, w])
        out, z, h = ops.mlp_forward(x.cuda(), up.cuda(), torch.eye(16, dtype=BF16).cuda(), activation=name, keep=True)
        a, u = ref.activation(x[:, 0].double(), name)[0], x[:, 0].double()
        fits = (a * u).abs() < 1e38
        assert ((h[:, 0].cpu().double() - a * u).abs() <= 2.0 ** -7 * (a * u).abs() + 2.0 ** -20 * (u * u).abs() + 1e-37)[fits].all(), name


@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("out", [16, 13])
def test_slopes_where_16_bit_floats_do_not_hold_z(name, out):
    """z is 4 x 30000 and 4 x -30000, which float16 keeps as infinities: the slopes there are 1 and 0."""
    x, w = torch.zeros(70, 64), torch.zeros(out, 64)
    x[:35, 0], x[35:, 0], w[:, 0] = 30000, -30000, 4
    x, w, d = x.to(F16).cuda(), w.to(F16).cuda(), torch.full((70, out), 0.5, dtype=F16).cuda()
    z = ops.linear_forward(x, w, None, name, keep=True)[1]
    dx, dw, db = ops.linear_backward(d, x, w, z, name)
    # sums of `out` products 0.5 x 4 x slope, and of 35 of them; every one is a 16-bit float
    assert dx[:35, 0].tolist() == [2.0 * out] * 35 and dx[35:].abs().max() == 0 and db.tolist() == [17.5] * out
    # h = z of 0 or more than float16 holds; the second matrix is 0, so is what comes back to z
    got = ops.mlp_forward(x, w, torch.zeros(8, out, dtype=F16).cuda(), activation=name, gated=False, keep=True)[1]
    dx = ops.mlp_backward(torch.ones(70, 8, dtype=F16).cuda(), x, w, torch.zeros(8, out, dtype=F16).cuda(), got,
                          torch.zeros(70, out + -out % 8, dtype=F16).cuda(), name, False)[0]
    assert dx.abs().max() == 0


def test_rows_with_infinities_where_sizes_are_no_multiples_of_8():
    """Slopes of a relu are 0 or 1 whatever z is, so gradients of a row of x with an infinity are the formulas' and not NaN."""
    x, w = normal(1, 100, 64), normal(2, 13, 64)
    d = normal(3, 100, 13)
    x[7, 3] = math.inf
    z = ops.linear_forward(x.cuda(), w.cuda(), None, "relu", keep=True)[1]
    dx = ops.linear_backward(d.cuda(), x.cuda(), w.cuda(), z, "relu")[0].cpu()
    slope = (x.double() @ w.double().T > 0).double()
    want = (d.double() * slope) @ w.double()
    # 13 products, and the rounding of the result
    assert ((dx.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * ((d.double() * slope).abs() @ w.double().abs())).all()
    down = normal(4, 24, 13)
    e = normal(5, 100, 24)
    z, h = ops.mlp_forward(x.cuda(), w.cuda(), down.cuda(), activation="relu", gated=False, keep=True)[1:]
    dx = ops.mlp_backward(e.cuda(), x.cuda(), w.cuda(), down.cuda(), z, h, "relu", False)[0].cpu()
    dz = (e.double() @ down.double()) * slope
    want, spread = dz @ w.double(), dz.abs() @ w.double().abs()
    # dz is rounded, 2^-8 (1 + 2^-8), and is a sum of 24 products, of which slopes leave all or nothing; then as above
    off = 2.0 ** -7.9 * spread + 2.0 ** -18 * ((e.double().abs() @ down.double().abs()) * slope) @ w.double().abs()
    assert ((dx.double() - want).abs() <= 2.0 ** -8 * want.abs() + off).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradients_of_no_rows_are_0_whatever_the_workspace_held(dtype):
    none, up, down = torch.empty(0, 64, dtype=dtype).cuda(), normal(1, 512, 64, dtype=dtype).cuda(), normal(2, 64, 256, dtype=dtype).cuda()
    z, h = torch.empty(0, 3 * 512, dtype=torch.uint8).cuda(), torch.empty(0, 256, dtype=dtype).cuda()
    got = [torch.full(shape, math.nan, dtype=dtype).cuda() for shape in ((512, 64), (512,), (64, 256), (64,))]
    a = _capi.Mlp(0, 64, 256, 64, ops._DTYPES[dtype], 4, 1, 64, 0, 64, None, up.data_ptr(), None, down.data_ptr(), None, None, None, None, None, None, None,
                  *(t.data_ptr() for t in got))
    size = _capi.lib().nd_mlp_workspace(a, 1)
    workspace = torch.full((max(size, 16),), 255, dtype=torch.uint8).cuda()
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    ops._run(torch.cuda.current_device(), ops._library().nd_mlp_backward, a)
    torch.cuda.synchronize()
    assert all((t == 0).all() for t in got)
    assert all((t == 0).all() for t in ops.mlp_backward(none, none, up, down, z, h)[1:])


def test_biases_of_32_bits_without_a_weight():
    x, b, d = normal(1, 600, 96), normal(2, 96, dtype=F32), normal(3, 600, 96)
    gx, gb = x.cuda().requires_grad_(), b.cuda().requires_grad_()
    ops.layer_norm(gx, None, gb).backward(d.cuda())
    want, off = ref.layer_norm(x, None, b, 1e-5, d)
    assert gb.grad.dtype is F32 and close(gx.grad, want["dx"], off["dx"])
    assert (gb.grad.cpu().double() - d.double().sum(0)).abs().max() < 608 * 2.0 ** -24 * d.double().abs().sum(0).max()


def test_nothing_is_kept_where_no_gradient_is_asked_for():
    p = {n: t.cuda().requires_grad_() for n, t in block_parameters().items()}
    x = normal(1, 130, 64).cuda()
    with torch.no_grad():
        out = block(x, p)
    assert not out.requires_grad and same_bits(out, block(x, p).detach())


def test_matrices_of_more_than_4_gib():
    """Rows, columns and halves of matrices whose distances in bytes pass 32 bits."""
    rows, dim = 70001, 32768
    x = torch.empty(rows, dim, dtype=BF16, device="cuda").normal_()
    w, d = normal(1, 16, dim, std=dim ** -0.5).cuda(), normal(2, rows, 16).cuda()
    out = ops.linear_forward(x, w)
    dx, dw, db = ops.linear_backward(d, x, w)
    some = torch.tensor([0, 1, 65535, 65536, rows - 2, rows - 1], device="cuda")
    want, off = ref.linear(x[some].cpu(), w.cpu(), None, None, None, d[some].cpu())
    check_all({"out": out[some], "dx": dx[some]}, want, off, "rows")
    columns = slice(dim - 24, dim)
    exact = d.double().t() @ x[:, columns].double()
    spread = d.double().abs().t() @ x[:, columns].double().abs()
    assert ((dw[:, columns].double() - exact).abs() <= 2.0 ** -8 * exact.abs() + (rows + 8) * 2.0 ** -24 * spread).all()
    del dx
    x, d = x.view(2 * rows, dim // 2), torch.empty(2 * rows, dim // 2, dtype=BF16, device="cuda").normal_()
    out, mean, rstd = ops.layer_norm_forward(x)
    dx, dw, db = ops.layer_norm_backward(d, x, None, mean, rstd)
    some = torch.tensor([0, 65536, 131072, 2 * rows - 1], device="cuda")
    want, off = ref.layer_norm(x[some].cpu(), None, None, 1e-5, d[some].cpu())
    check_all({"out": out[some], "dx": dx[some]}, want, off, "norm")
    exact = d[:, -8:].double().sum(0)
    assert ((db[-8:].double() - exact).abs() <= 2.0 ** -8 * exact.abs() + (2 * rows + 8) * 2.0 ** -24 * d[:, -8:].double().abs().sum(0)).all()
    del x, d, out, dx
    # the two projections of a gated part lie more than 4 GiB apart
    inner = 65600
    up = torch.empty(2 * inner, dim, dtype=BF16, device="cuda").normal_(std=dim ** -0.5)
    down = torch.zeros(8, inner, dtype=BF16, device="cuda")
    for n in (3, 300):
        x = normal(3, n, dim).cuda()
        _, _, h = ops.mlp_forward(x, up, down, keep=True)
        some = torch.tensor([0, 31, 32, 63, 64, 40000, inner - 1], device="cuda")
        want, off = ref.mlp(x.cpu(), torch.cat([up[some], up[some + inner]]).cpu(), torch.eye(7, dtype=BF16))
        assert close(h[:, some], want["out"], off["out"])
    del up, down
    torch.cuda.empty_cache()


# ---- every kind of tile ----------------------------------------------------------------------------------------
# Sizes for which the rules take each of the four shapes of tiles, with whole sums and with shares of them, in the forward
# pass, for dx and for dweight (alone: both together go into one launch), and two shapes for the rows of one product.  References in 64 bits on the GPU.

LINEAR_TILES = [(958, 528, 16008), (135, 13032, 15600), (2581, 3480, 8), (65, 976, 8), (13553, 136, 544), (5684, 11280, 136),
                (958, 16008, 528), (5684, 136, 11280), (517, 1160, 12712), (12017, 15928, 136), (3479, 8, 2584), (129, 536, 13296),
                (10768, 136, 5808), (4104, 1000, 4096), (4104, 4096, 1000), (1000, 4096, 4104)]


@pytest.mark.parametrize("rows,dim,out", LINEAR_TILES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_with_every_shape_of_tile(rows, dim, out, dtype):
    print("tiles", rows, dim, out, dtype, flush=True)
    x, w, b, name, r, d = map_cuda(linear_case(rows, dim, out, dtype, "silu", residual=True))
    want, off = ref.linear(x, w, b, name, r, d)
    y, z = ops.linear_forward(x, w, b, name, r, keep=True)
    dx, _, _ = ops.linear_backward(d, x, w, z, name, False, (True, False))
    _, dw, db = ops.linear_backward(d, x, w, z, name, True, (False, True))
    both = ops.linear_backward(d, x, w, z, name)
    for i, got in enumerate(({"out": y, "dx": dx, "dweight": dw, "dbias": db}, dict(zip(("dx", "dweight", "dbias"), both)))):
        for n, t in got.items():
            assert within(t, want[n], off[n]), (i, n)


MLP_TILES = [(391, 848, 8400, 64), (133, 7072, 9264, 64), (7122, 9576, 72, 8), (2581, 3480, 8, 8), (65, 976, 8, 8), (655, 136, 10992, 800),
             (6400, 136, 448, 152), (20483, 64, 256, 64), (4104, 2000, 2048, 64), (4104, 1000, 4096, 64),
             (4104, 64, 4096, 1000)]


@pytest.mark.parametrize("rows,dim,inner,out", MLP_TILES)
@pytest.mark.parametrize("gated,dtype", [(True, BF16), (True, F16), (False, BF16)])
def test_mlp_with_every_shape_of_tile(rows, dim, inner, out, gated, dtype):
    print("tiles", rows, dim, inner, out, gated, dtype, flush=True)
    case = map_cuda(mlp_case(rows, dim, inner, out, dtype, "silu", gated))
    x, up, down, up_bias, down_bias, name, _, r, d = case
    want, off = ref.mlp(*case)
    y, z, h = ops.mlp_forward(x, up, down, up_bias, down_bias, name, gated, r, keep=True)
    names = ("dx", "dup", "ddown", "dup_bias", "ddown_bias")
    everything = dict(zip(names, ops.mlp_backward(d, x, up, down, z, h, name, gated)))
    alone = dict(zip(names, ops.mlp_backward(d, x, up, down, z, h, name, gated, True, False, (True, False, False))))
    for i, got in enumerate(({"out": y, **everything}, {n: alone[n] for n in ("dx", "dup_bias")})):
        for n, t in got.items():
            assert within(t, want[n], off[n]), (i, n)


def map_cuda(case):
    return [t.cuda() if isinstance(t, torch.Tensor) else t for t in case]


def within(got, right, off):
    value = got.double()
    if got.dtype is F16:
        value = torch.where(torch.isinf(value) & (right.abs() + off >= 65520) & (value.sign() == right.sign()), right, value)
    wrong = ((value - right).abs() > off) | torch.isnan(value)
    if wrong.any():
        at = tuple(int(i) for i in wrong.nonzero()[0])
        print("%d of %d off; first at %s: %r, should be %r within %r" % (int(wrong.sum()), wrong.numel(), at, float(value[at]), float(right[at]),
                                                                      float(off[at])))
    return not wrong.any()


# ---- autograd, streams, graphs ------------------------------------------------------------------------------


def block(x, p, seed=None):
    """Everything of a block but its attention."""
    n = ops.layer_norm(x, p["norm_weight"], p["norm_bias"])
    y = ops.linear(n, p["weight"], p["bias"], "gelu_tanh", x)
    n = ops.layer_norm(y, p["norm_weight"], p["norm_bias"])
    return ops.mlp(n, p["up"], p["down"], None, p["down_bias"], "silu", True, y)


def block_parameters(dim=64, inner=136, dtype=BF16):
    return {"norm_weight": normal(1, dim, dtype=dtype, mean=1.0, std=0.1), "norm_bias": normal(2, dim, dtype=dtype, std=0.1),
            "weight": normal(3, dim, dim, dtype=dtype, std=dim ** -0.5), "bias": normal(4, dim, dtype=dtype, std=0.1),
            "up": normal(5, 2 * inner, dim, dtype=dtype, std=dim ** -0.5), "down": normal(6, dim, inner, dtype=dtype, std=inner ** -0.5),
            "down_bias": normal(7, dim, dtype=dtype, std=0.1)}


def plain_block(x, p):
    f = torch.nn.functional
    n = f.layer_norm(x, x.shape[-1:], p["norm_weight"], p["norm_bias"])
    y = f.gelu(f.linear(n, p["weight"], p["bias"]), approximate="tanh") + x
    g, u = f.linear(f.layer_norm(y, x.shape[-1:], p["norm_weight"], p["norm_bias"]), p["up"]).chunk(2, -1)
    return f.linear(f.silu(g) * u, p["down"], p["down_bias"]) + y


@pytest.mark.parametrize("rows", [7, 300])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_block_has_the_gradients_of_plain_operations(rows, dtype):
    p = block_parameters(dtype=dtype)
    x, d = normal(8, rows, 64, dtype=dtype), normal(9, rows, 64, dtype=dtype)
    gpu = {n: t.cuda().requires_grad_() for n, t in p.items()}
    gx = x.cuda().requires_grad_()
    block(gx, gpu).backward(d.cuda())
    cpu = {n: t.double().requires_grad_() for n, t in p.items()}
    cx = x.double().requires_grad_()
    plain_block(cx, cpu).backward(d.double())
    # a chain of some 16 roundings to the type, none amplified by more than its weights, of norm about 1
    for name, got, want in [("x", gx.grad, cx.grad)] + [(n, gpu[n].grad, cpu[n].grad) for n in p]:
        off = float((got.cpu().double() - want).norm() / want.norm())
        assert off < 16 * (2.0 ** -8 if dtype is BF16 else 2.0 ** -11), (name, off)


def test_autograd_takes_only_what_is_asked_for():
    p = {n: t.cuda() for n, t in block_parameters().items()}
    x = normal(8, 30, 64).cuda()
    assert not block(x, p).requires_grad
    for names in (("weight",), ("up", "norm_bias"), ("down_bias",), ("bias", "down")):
        some = {n: t.clone().requires_grad_(n in names) for n, t in p.items()}
        block(x, some).sum().backward()
        every = {n: t.clone().requires_grad_() for n, t in p.items()}
        block(x, every).sum().backward()
        for n in p:
            assert (some[n].grad is None) == (n not in names)
            assert n not in names or torch.equal(some[n].grad, every[n].grad)
    r = normal(9, 30, 64).cuda().requires_grad_()
    ops.linear(x, p["weight"], residual=r).sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r))


def step(x, d, p):
    """Forward and backward calls of a step, without autograd."""
    n, mean, rstd = ops.layer_norm_forward(x, p["norm_weight"], p["norm_bias"])
    y, z = ops.linear_forward(n, p["weight"], p["bias"], "gelu", x, keep=True)
    out, zz, h = ops.mlp_forward(y, p["up"], p["down"], None, p["down_bias"], residual=y, keep=True)
    dy, dup, ddown, _, ddown_bias = ops.mlp_backward(d, y, p["up"], p["down"], zz, h, with_up_bias=False)
    dn, dweight, dbias = ops.linear_backward(dy, n, p["weight"], z, "gelu")
    return (out, dup, ddown, ddown_bias, dweight, dbias, *ops.layer_norm_backward(dn, x, p["norm_weight"], mean, rstd))


@pytest.mark.parametrize("rows,dtype", [(5, BF16), (300, BF16), (300, F16), (2500, BF16)])
def test_a_step_is_the_same_on_another_stream_and_in_graphs(rows, dtype):
    p = {n: t.cuda() for n, t in block_parameters(dtype=dtype).items()}
    inputs = [(normal(s, rows, 64, dtype=dtype).cuda(), normal(s + 50, rows, 64, dtype=dtype).cuda()) for s in range(4)]
    eager = [step(x, d, p) for x, d in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [step(x, d, p) for x, d in inputs]
    side.synchronize()
    for a, b in zip(eager, again):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    # two graphs over the same inputs, replayed in turn, with eager work between
    x, d = torch.empty_like(inputs[0][0]), torch.empty_like(inputs[0][1])
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = step(x, d, p)
        graphs.append((graph, results))
    for turn in range(6):
        x.copy_(inputs[turn % 4][0])
        d.copy_(inputs[turn % 4][1])
        graph, results = graphs[turn % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(eager[turn % 4], results)), turn
        step(*inputs[(turn + 1) % 4], p)


def test_an_autograd_step_is_captured():
    p = {n: t.cuda().requires_grad_() for n, t in block_parameters().items()}
    x = normal(8, 100, 64).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = torch.autograd.grad(block(x, p).float().square().mean(), list(p.values()))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = torch.autograd.grad(block(x, p).float().square().mean(), list(p.values()))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))


# ---- together ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("p", [0.0, 0.2])
def test_a_gated_walk_model_has_the_gradients_of_plain_operations(p, monkeypatch):
    """One step of the model in 16 bits against the same model with the definitions in 64 bits: every operator of the library."""
    import numpy as np
    from nextdoor_amd import walk_model
    from tests import operators_reference
    torch.manual_seed(1)
    n = 97
    rng = np.random.default_rng(2)
    samples = rng.integers(0, n, (20, 30)).astype(np.int32)
    for walk in samples[::2]:
        walk[rng.integers(0, 30):] = n
    tokens, targets, starts = walk_model.pack_walks(rng.integers(0, n, 20), samples, n)
    how = dict(width=64, heads=2, kv_heads=1, layers=1, dropout=p, gated=True)
    model = walk_model.WalkModel(n, **how).to("cuda", BF16)
    batch = walk_model.batch_of(tokens, targets, starts)
    each = model(*batch[:3], batch[3], 11)
    each.sum().backward()
    exact = walk_model.WalkModel(n, **how).double()
    exact.load_state_dict({k: v.double().cpu() for k, v in model.state_dict().items()})

    of = torch.from_numpy(np.repeat(np.arange(len(starts) - 1), np.diff(starts)))
    at = torch.arange(len(of))
    sees = (of[:, None] == of) & (at[:, None] >= at)
    f = torch.nn.functional

    def attention(q, k, v, sequences, scale=None):
        out = []
        for h in range(q.shape[1]):
            i = h // (q.shape[1] // k.shape[1])
            s = (q[:, h] @ k[:, i].T / math.sqrt(q.shape[2])).masked_fill(~sees, -math.inf)
            out.append(torch.softmax(s, 1) @ v[:, i])
        return torch.stack(out, 1)

    def drop(x, p, seed, step, residual=None):
        kept = torch.from_numpy(operators_reference.uniforms(x.numel(), seed, step) >= np.float32(p)).view(x.shape)
        y = x * kept / (1 - p)
        return y if residual is None else y + residual

    def loss(h, w, t):
        has = (t >= 0) & (t < n)
        z = h @ w.T
        return torch.where(has, torch.logsumexp(z, 1) - z.gather(1, torch.where(has, t, 0).long()[:, None])[:, 0], 0.0)

    def plain_mlp(x, up, down, residual=None):
        g, u = f.linear(x, up).chunk(2, -1)
        y = f.linear(f.silu(g) * u, down)
        return y if residual is None else y + residual

    plain = {"packed_attention": attention, "dropout": drop, "vocabulary_loss": loss, "mlp": plain_mlp,
             "linear": lambda x, w, residual=None: f.linear(x, w) if residual is None else f.linear(x, w) + residual,
             "layer_norm": lambda x, w, b, eps: f.layer_norm(x, x.shape[-1:], w, b, eps)}
    for name, function in plain.items():
        monkeypatch.setattr(ops, name, function)
    right = exact(*[torch.from_numpy(np.ascontiguousarray(a)) for a in
                    (tokens, np.arange(len(tokens)) - np.repeat(starts[:-1], np.diff(starts)), targets)], None, 11)
    right.sum().backward()
    # some thirty roundings of 2^-8 on the way there and back, each of what is of the size of the result
    assert float((each.detach().cpu().double() - right.detach()).norm() / right.detach().norm()) < 30 * 2.0 ** -8
    for (name, a), b in zip(model.named_parameters(), exact.parameters()):
        assert float((a.grad.cpu().double() - b.grad).norm() / b.grad.norm()) < 60 * 2.0 ** -8, name


def test_the_gated_walk_model_trains():
    from nextdoor_amd import Graph, walk_model
    graph = Graph.chung_lu(500, 6000, 2.2, seed=3)
    losses = [walk_model.train(graph, steps=3, walks=200, seed=5, log=None, gated=True)[1] for _ in range(2)]
    assert len(losses[0]) == 3 and all(math.isfinite(v) for v in losses[0]) and losses[0][0] == losses[1][0]
