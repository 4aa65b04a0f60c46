"""Training operators on the GPU where a definition leaves no room: results that are exactly 0, and gradients so small or so
large that a 16-bit operand could lose them."""
import math

import numpy as np
import pytest
import torch

from nextdoor_amd import NextDoorError, ops
from tests import operators_reference as ref
from tests.test_gpu_operators import BF16, F16, normal, run_attention, run_loss, starts_of, targets

pytestmark = pytest.mark.gpu

# whole sequences to a tile; longer ones; ones that are cut into chunks
ONE_KEY = {"ones": [1] * 70, "one": [1], "short": [1, 5, 1, 100, 1, 28, 1], "long": [129, 901, 1, 40, 1], "cut": [1, 1500, 1, 1, 700, 129, 1]}


@pytest.mark.parametrize("lengths", sorted(ONE_KEY))
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (4, 1, 128), (6, 2, 40)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("std", [1.0, 10.0])
def test_attention_rows_with_one_key_send_nothing_to_queries_and_keys(lengths, heads, kv_heads, dim, dtype, std):
    """Such a row's weight is 1 whatever its logit is: dq = 0, and dk = 0 of a sequence of one token, exactly; dv is the
    output's gradient."""
    starts = starts_of(ONE_KEY[lengths])
    t, first = int(starts[-1]), torch.from_numpy(starts[:-1].astype(np.int64))
    q, dout = normal(1, t, heads, dim, dtype=dtype, std=std), normal(2, t, heads, dim, dtype=dtype, std=std)
    k, v = normal(3, t, kv_heads, dim, dtype=dtype, std=std), normal(4, t, kv_heads, dim, dtype=dtype, std=std)
    got = {n: x.cpu() for n, x in run_attention(q.cuda(), k.cuda(), v.cuda(), starts, dout.cuda()).items()}
    assert not got["dq"][first].any()
    alone = first[torch.from_numpy(np.diff(starts) == 1)]
    assert not got["dk"][alone].any()
    # the group's heads added up in 32 bits and rounded once
    want = dout[alone].double().view(len(alone), kv_heads, -1, dim)
    off = (ref.UNIT[dtype] + heads * 2.0 ** -23) * want.abs().sum(2) if heads > kv_heads else torch.zeros(1, dtype=torch.float64)
    assert ref.close(got["dv"][alone], want.sum(2), off.expand(len(alone), kv_heads, dim))
    assert torch.equal(got["out"][alone], v[alone].repeat_interleave(heads // kv_heads, 1))


@pytest.mark.parametrize("lengths", [[40, 3, 70, 2], [100, 28], [200, 56, 130]])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 2)])
def test_attention_equal_values_send_nothing_to_queries_and_keys(lengths, dtype, heads, kv_heads):
    """Where all values of a sequence are equal, do . v is too, whatever the weights are: ds is 0 but for the roundings of
    delta = sum p dp / sum p, sums of n weights in 32 bits.  Logits in the thousands: weights that are made again from a rounded
    lse have a sum of 1 +- some 1e-4."""
    starts, dim, scale = starts_of(lengths), 64, 1.0
    t = int(starts[-1])
    q, dout = normal(1, t, heads, dim, dtype=dtype, std=10.0), normal(2, t, heads, dim, dtype=dtype)
    k, v = normal(3, t, kv_heads, dim, dtype=dtype, std=10.0), normal(4, len(lengths), kv_heads, dim, dtype=dtype)
    v = v.repeat_interleave(torch.tensor(lengths), 0)
    got = run_attention(q.cuda(), k.cuda(), v.cuda(), starts, dout.cuda(), scale)
    for head in range(heads):
        kv = head // (heads // kv_heads)
        dp = (dout[:, head].double().abs() * v[:, kv].double().abs()).sum(1)
        longest = torch.from_numpy(np.repeat(lengths, lengths)).double()
        # two sums and a quotient; and do . v of the two kernels, dim products in another order
        e = dp * (2 * (longest + 4) + 2 * (dim + 8)) * 2.0 ** -24
        for i in range(len(lengths)):
            at = slice(int(starts[i]), int(starts[i + 1]))
            most_k, most_q = k[at, kv].double().abs().amax(0), q[at, head].double().abs().amax(0)
            n = lengths[i]
            dq = got["dq"][at, head].cpu().double().abs()
            assert (dq <= scale * e[at, None] * most_k * 1.01 + ref.LEAST[dtype] * (1 + n * most_k)).all(), (head, i, "dq")
            if heads == kv_heads:
                dk = got["dk"][at, kv].cpu().double().abs()
                assert (dk <= scale * e[at].sum() * most_q * 1.01 + ref.LEAST[dtype] * (1 + n * most_q)).all(), (head, i, "dk")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2)])
def test_attention_of_one_token_in_odd_places(heads, kv_heads):
    """One token whose rows lie at odd pitches and places, which torch calls contiguous: as any other layout."""
    dim = 64
    gen = torch.Generator().manual_seed(1)

    def odd(n, seed):
        wide = torch.randn(3, n * dim + 3, generator=gen.manual_seed(seed)).to(BF16).cuda()
        return wide[:1, 3:].unflatten(1, (n, dim)), wide[:1, :n * dim].unflatten(1, (n, dim))

    for place in (0, 1):
        q, k, v, dout = (odd(n, i)[place] for i, n in enumerate((heads, kv_heads, kv_heads, heads)))
        want, off = ref.attention(q.cpu(), k.cpu(), v.cpu(), [0, 1], 1 / 8, dout.cpu())
        got = run_attention(q, k, v, [0, 1], dout)
        for name in got:
            assert ref.close(got[name], want[name], off[name]), name


def gradients(q, k, v, starts, scale, dout):
    """dq, dk, dv in 64 bits, and what the roundings of the backward pass can do to them where 16-bit floats hold 2^15 p and
    2^15 k ds, k at least 1 / (4 B) with B = dim max |dout| max |v|: half their smallest step is 2^-40 of p and 2^-38 B of
    ds, however small the gradient is."""
    unit, step = ref.UNIT[q.dtype], 2.0 ** -24 if q.dtype == F16 else 2.0 ** -126
    want, off = {n: torch.zeros_like(x).double() for n, x in zip(("dq", "dk", "dv"), (q, k, v))}, {}
    off = {n: torch.zeros_like(x) for n, x in want.items()}
    group, dim = q.shape[1] // k.shape[1], q.shape[2]
    most = dim * float(dout.abs().max()) * float(v.abs().max())
    for begin, end in zip(starts[:-1].tolist(), starts[1:].tolist()):
        at, n = slice(begin, end), end - begin
        later = torch.ones(n, n, dtype=torch.bool).triu(1)
        for h in range(q.shape[1]):
            a, b, c, d = (x[at, i].double() for x, i in ((q, h), (k, h // group), (v, h // group), (dout, h)))
            p = torch.softmax((a @ b.T * scale).masked_fill_(later, -math.inf), 1)
            dp, out = d @ c.T, p @ c
            ds = p * (dp - (d * out).sum(1)[:, None])
            spread = p @ c.abs()
            delta_off = (d.abs() * (unit * (out.abs() + spread) + ref.SMALL * spread + step * (1 + spread))).sum(1)
            delta_off += ref.SMALL * (d.abs() @ c.abs().T).amax(1)
            ds_off = unit * ds.abs() + p * delta_off[:, None] + ref.SMALL * ds.abs() + 2.0 ** -14 * step * most * (p > 0)
            p_off = (unit + ref.SMALL) * p + 2.0 ** -16 * step * (p > 0)
            kv = h // group
            for name, to, value, bound in (("dq", h, ds @ b * scale, ds_off @ b.abs() * scale), ("dk", kv, ds.T @ a * scale, ds_off.T @ a.abs() * scale),
                                           ("dv", kv, p.T @ d, p_off.T @ d.abs())):
                want[name][at, to] += value
                off[name][at, to] += bound
    for n in want:
        off[n] += unit * want[n].abs() + step / 2
    return want, off


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [([100, 1, 31, 77] * 8, 4, 2, 64), ([5000], 2, 1, 64), ([300, 900, 40], 3, 3, 128)])
def test_attention_small_gradients_of_16_bit_floats_are_not_lost(lengths, heads, kv_heads, dim, size):
    starts = starts_of(lengths)
    t = int(starts[-1])
    q, dout = normal(1, t, heads, dim, dtype=F16), normal(2, t, heads, dim, dtype=F16, std=size)
    k, v = normal(3, t, kv_heads, dim, dtype=F16), normal(4, t, kv_heads, dim, dtype=F16)
    want, off = gradients(q, k, v, starts, 1 / math.sqrt(dim), dout)
    got = run_attention(q.cuda(), k.cuda(), v.cuda(), starts, dout.cuda())
    for name in want:
        assert ref.close(got[name], want[name], off[name]), name
        # roundings of random sign: of the operand, of delta and of the result, each under 2^-11 of what it rounds; and half a step of
        # the smallest result
        error = float((got[name].cpu().double() - want[name]).norm())
        assert error <= 4 * 2.0 ** -11 * float(want[name].norm()) + 2.0 ** -25 * math.sqrt(want[name].numel()), (name, error)


@pytest.mark.parametrize("lengths,heads,kv_heads", [([100, 1, 31, 77], 4, 2), ([1500, 200], 2, 1)])
def test_attention_large_gradients_of_16_bit_floats(lengths, heads, kv_heads):
    """ds far above the largest 16-bit float, dq and dk below it (as the scale is small)."""
    starts, dim, scale = starts_of(lengths), 64, 2.0 ** -9
    t = int(starts[-1])
    q, dout = normal(1, t, heads, dim, dtype=F16), normal(2, t, heads, dim, dtype=F16, std=2000.0)
    k, v = normal(3, t, kv_heads, dim, dtype=F16), normal(4, t, kv_heads, dim, dtype=F16, std=8.0)
    want, off = gradients(q, k, v, starts, scale, dout)
    got = run_attention(q.cuda(), k.cuda(), v.cuda(), starts, dout.cuda(), scale)
    for name in ("dq", "dk"):
        assert float(want[name].abs().max()) < 65504
        assert ref.close(got[name], want[name], off[name]), name


def test_attention_rows_that_are_not_finite_do_not_decide_what_16_bit_floats_hold():
    """An infinite output gradient or value in one sequence leaves the small gradients of the others as they are."""
    heads, kv_heads, dim = 2, 1, 64
    for lengths in ([90, 60, 100, 40], [90, 600, 2000, 40]):
        starts = starts_of(lengths)
        t = int(starts[-1])
        q, dout = normal(1, t, heads, dim, dtype=F16), normal(2, t, heads, dim, dtype=F16, std=1e-4)
        k, v = normal(3, t, kv_heads, dim, dtype=F16), normal(4, t, kv_heads, dim, dtype=F16)
        want, off = gradients(q, k, v, starts, 1 / 8, dout)
        bad, others = int(starts[1]) + 30, torch.ones(t, dtype=torch.bool)
        others[starts[1]:starts[2]] = False
        for value in (math.inf, math.nan):
            for which in (0, 1):
                x, y = dout.clone(), v.clone()
                (x, y)[which][bad] = value
                got = run_attention(q.cuda(), k.cuda(), y.cuda(), starts, x.cuda())
                for name in want:
                    assert ref.close(got[name].cpu()[others], want[name][others], off[name][others]), (lengths, value, which, name)


def test_loss_of_the_most_classes():
    """The largest vocabulary that is accepted: three rows' loss, and the gradients of its first and last classes."""
    rows, classes, dim = 3, 2147483392, 8
    gen = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(rows, dim, device="cuda", generator=gen).to(BF16)
    w = torch.zeros(classes, dim, dtype=BF16, device="cuda")
    ends = torch.cat([torch.arange(500, device="cuda"), torch.arange(classes - 500, classes, device="cuda")])
    w[ends] = (torch.randn(1000, dim, device="cuda", generator=gen) * 4).to(BF16)
    t = torch.tensor([classes - 7, 3, classes], device="cuda")
    loss, lse = ops.vocabulary_loss_forward(h, w, t)
    dhidden, dweight = ops.vocabulary_loss_backward(torch.full((rows,), 1e6, device="cuda"), h, w, t, lse)
    # all other logits are 0
    z = h.double() @ w[ends].double().T
    z_off = (dim + 8) * 2.0 ** -24 * (h.double().abs() @ w[ends].double().abs().T).amax(1) + 2.0 ** -21 * z.abs().amax(1) + 2.0 ** -21 * 22
    want = torch.logsumexp(torch.cat([z, torch.full((rows, 1), math.log(classes - 1000), dtype=torch.float64, device="cuda")], 1), 1)
    assert ((lse.double() - want).abs() <= z_off + 2.0 ** -13).all()
    target = torch.tensor([[993], [3]], device="cuda")
    assert ((loss[:2].double() - (want[:2] - z[:2].gather(1, target)[:, 0])).abs() <= 2 * z_off[:2] + 2.0 ** -13).all() and loss[2] == 0
    p = torch.exp(z - want[:, None]) * 1e6
    p[2] = 0
    g = p.clone()
    g[[0, 1], target[:, 0]] -= 1e6
    g_off = (2.0 ** -8 + ref.SMALL) * g.abs() + (2 * (z_off[:, None] + 2.0 ** -13) + ref.SMALL) * p
    for got, value, off in ((dhidden, g @ w[ends].double(), g_off @ w[ends].double().abs()),
                            (dweight[ends], g.T @ h.double(), g_off.T @ h.double().abs())):
        assert ((got.double() - value).abs() <= 2.0 ** -8 * value.abs() + off).all()
    del w, dweight
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,classes,dim", [(60, 500, 64), (60, 500, 264), (300, 500, 264)])
@pytest.mark.parametrize("size", [1e-36, 1e-41])
def test_loss_gradients_far_below_16_bit_floats_are_zero(rows, classes, dim, size):
    h, w = normal(1, rows, dim, dtype=F16), normal(2, classes, dim, dtype=F16, std=2 / math.sqrt(dim))
    got = run_loss(h.cuda(), w.cuda(), targets(3, rows, classes).cuda(), torch.full((rows,), size, device="cuda"))
    assert not got["dhidden"].any() and not got["dweight"].any()


@pytest.mark.parametrize("rows,classes,dim", [(60, 500, 64), (60, 500, 264), (300, 500, 264)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_loss_one_row_that_is_not_finite_leaves_the_others_gradients(rows, classes, dim, value, dtype):
    h, w = normal(1, rows, dim, dtype=dtype), normal(2, classes, dim, dtype=dtype, std=2 / math.sqrt(dim))
    t = torch.arange(rows) % classes
    dloss = torch.full((rows,), 1e-4)
    want, off = ref.vocabulary_loss(h, w, t, dloss)
    dloss[7] = value
    got = run_loss(h.cuda(), w.cuda(), t.cuda(), dloss.cuda())
    others = torch.arange(rows) != 7
    assert ref.close(got["dhidden"].cpu()[others], want["dhidden"][others], off["dhidden"][others])
    assert not torch.isfinite(got["dhidden"][7]).any() and not torch.isfinite(got["dweight"]).all()


def test_plan_of_more_sequences_than_half_of_32_bits_count():
    """Over 2^30 sequences, all but the last ones empty: a batch is what its tokens are."""
    lengths = [3, 0, 40, 1, 0, 2]
    starts = np.zeros(2 ** 30 + 6, np.int32)
    starts[-6:] = np.cumsum(lengths)
    t = int(starts[-1])
    q, k, v = (normal(i, t, 2, 64).cuda() for i in range(3))
    got = ops.packed_attention_forward(q, k, v, ops.PackedSequences(starts))
    want = ops.packed_attention_forward(q, k, v, ops.PackedSequences(starts_of(lengths)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del starts, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("lengths", [[5, 1, 30], [70, 200, 9], [40, 1500, 3]])
@pytest.mark.parametrize("dim", [64, 40])
def test_attention_rows_of_logits_that_are_all_minus_infinity_are_not_a_number(lengths, dim):
    """exp(s - lse) is NaN there; lse is -inf, and the rows of other sequences are as ever."""
    starts, heads = starts_of(lengths), 2
    t = int(starts[-1])
    q, k, v, dout = (normal(i, t, heads, dim) for i in range(4))
    hit = torch.zeros(t, dtype=torch.bool)
    hit[starts[1]:starts[2]] = True
    want, off = ref.attention(q, k, v, starts, 1 / math.sqrt(dim), dout)
    q[hit], k[hit] = 1e25, -1e25
    got = run_attention(q.cuda(), k.cuda(), v.cuda(), starts, dout.cuda())
    assert torch.isinf(got["lse"].cpu()[:, hit]).all() and (got["lse"].cpu()[:, hit] < 0).all()
    for name in ("out", "dq", "dk", "dv"):
        assert torch.isnan(got[name].cpu()[hit]).all(), name
        assert ref.close(got[name].cpu()[~hit], want[name][~hit], off[name][~hit]), name


@pytest.mark.parametrize("rows,classes,dim,dtype", [(20000, 40001, 232, BF16), (20000, 40001, 232, F16), (20011, 30011, 520, F16), (20000, 25000, 776, BF16)])
def test_loss_of_longer_vectors_goes_through_several_pieces_of_the_vocabulary(rows, classes, dim, dtype):
    """More rows than one piece's workspace holds for all classes: every value of both gradients, in 64 bits on the GPU."""
    h, w = normal(1, rows, dim, dtype=dtype).cuda(), normal(2, classes, dim, dtype=dtype, std=2 / math.sqrt(dim)).cuda()
    t = targets(3, rows, classes).cuda()
    dloss = ((0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(4))) / rows).cuda()
    one = ops._loss_workspace(rows, classes, dim, 1) - ops._loss_workspace(rows, 256, dim, 1)
    assert one < 2 * rows * classes  # (g of all classes is not kept)
    want, off = ref.vocabulary_loss(h, w, t, dloss)
    got = run_loss(h, w, t, dloss)
    for name in want:
        assert ref.close(got[name], want[name].cpu(), off[name].cpu()), name
    del want, off
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,classes,dim", [(50, 100, 32), (300, 500, 64), (60, 500, 264), (300, 500, 264), (300, 9000, 264)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("known", [0.0, 0.7])
def test_loss_rows_without_a_target_send_nothing_to_the_classes(rows, classes, dim, dtype, known):
    """Whatever they and their dloss hold, among rows that have one."""
    h, w = normal(1, rows, dim, dtype=dtype), normal(2, classes, dim, dtype=dtype, std=2 / math.sqrt(dim))
    rng = np.random.default_rng(1)
    none = torch.from_numpy(rng.random(rows) >= known)
    t = torch.where(none, classes, torch.from_numpy(rng.integers(0, classes, rows)))
    dloss = torch.full((rows,), 1 / rows)
    want, off = ref.vocabulary_loss(h, w, t, dloss)
    at = none.nonzero()[:, 0]
    h[at[::2]], h[at[1::2]], dloss[at] = math.nan, math.inf, math.inf
    got = run_loss(h.cuda(), w.cuda(), t.cuda(), dloss.cuda())
    for name in ("loss", "dhidden", "dweight"):
        assert ref.close(got[name], want[name], off[name]), name
    assert not got["dhidden"].cpu()[none].any() and not got["loss"].cpu()[none].any()
    if known == 0.0:
        assert not got["dweight"].any()


def test_tensors_of_other_shapes_are_refused_as_the_rest_is():
    x, seq = normal(1, 10, 4, 64).cuda(), ops.PackedSequences([0, 10])
    out, lse = ops.packed_attention_forward(x, x, x, seq)
    one, none = x[0, 0, 0], x[..., :0]
    h, t = x[:, 0].contiguous(), torch.zeros(10, dtype=torch.int64, device="cuda")
    for fn, args in ((ops.packed_attention_forward, (one, one, one, seq)), (ops.packed_attention_forward, (none, none, none, seq)),
                     (ops.packed_attention_backward, (one, one, one, one, out, lse, seq)),
                     (ops.vocabulary_loss_forward, (one, one, t)), (ops.vocabulary_loss_backward, (lse[0], one, one, t, lse[0])),
                     (ops.vocabulary_loss_forward, (h[:, :0], h[:, :0], t)), (ops.vocabulary_loss_backward, (lse[0], h, h, t, one.float()))):
        with pytest.raises(NextDoorError):
            fn(*args)


@pytest.mark.parametrize("lengths", [[100, 1, 31, 77, 120] * 60, [100, 28, 5], [300, 70]])
def test_attention_heads_of_a_group_with_gradients_of_different_sizes(lengths):
    """Small, then large, then small ones again, in 16-bit floats: the sums of a key are those of all of them."""
    starts, heads, kv_heads, dim = starts_of(lengths), 8, 2, 64
    t = int(starts[-1])
    q, k, v = (normal(i, t, n, dim, dtype=F16) for i, n in enumerate((heads, kv_heads, kv_heads)))
    sizes = torch.tensor([1e-4, 1.0, 1e-5, 30.0, 30.0, 1e-5, 1.0, 0.0])
    dout = (normal(5, t, heads, dim, dtype=torch.float32) * sizes[:, None]).to(F16)
    want, off = gradients(q, k, v, starts, 1 / 8, dout)
    got = run_attention(q.cuda(), k.cuda(), v.cuda(), starts, dout.cuda())
    for name in want:
        assert ref.close(got[name], want[name], off[name]), name


@pytest.mark.parametrize("lengths", [[100, 28, 5, 77], [300, 1, 170]])
def test_attention_of_16_bit_floats_is_the_same_in_a_graph(lengths):
    """What they are held times is found anew at every replay."""
    starts = starts_of(lengths)
    q, k, v, dout = (normal(i, int(starts[-1]), 4, 64, dtype=F16).cuda() for i in range(4))
    seq = ops.PackedSequences(starts)

    def step():
        out, lse = ops.packed_attention_forward(q, k, v, seq)
        return (out, *ops.packed_attention_backward(dout, q, k, v, out, lse, seq))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        for x in got:
            x.zero_()
        dout.mul_(0.01 if i < 2 else 3000.0)
        want = [x.clone() for x in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
