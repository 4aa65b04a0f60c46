"""The training operators on the GPU, against their definitions in 64 bits (operators_reference.py)."""
import math

import numpy as np
import pytest
import torch

from nextdoor_amd import NextDoorError, ops
from tests import operators_reference as ref

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(seed, *shape, dtype=BF16, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def starts_of(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def check_all(got, want, off, what):
    for name in got:
        assert ref.close(got[name], want[name], off[name]), (what, name)


# ---- packed attention --------------------------------------------------------------------------

LENGTHS = {
    "one_token": [1],
    "two": [2],
    "ones": [1] * 70,
    "empty_between": [0, 3, 0, 0, 40, 0],
    "tile": [128],
    "tile_and_one": [129],
    "one_less": [127, 1],
    "across_tiles": [5, 120, 64, 63, 65, 1, 300, 7],
    "long": [901],
    "walks": list(np.random.default_rng(3).integers(1, 102, 40)),
}


def run_attention(q, k, v, starts, dout, scale=None, tokens=None):
    seq = ops.PackedSequences(starts, q.shape[0] if tokens is None else tokens)
    out, lse = ops.packed_attention_forward(q, k, v, seq, scale)
    dq, dk, dv = ops.packed_attention_backward(dout, q, k, v, out, lse, seq, scale)
    torch.cuda.synchronize()
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 2, 64, BF16), (3, 1, 128, F16), (2, 2, 32, BF16), (12, 2, 40, F16)])
def test_attention_over_lengths(lengths, heads, kv_heads, dim, dtype):
    starts = starts_of(LENGTHS[lengths])
    t = int(starts[-1])
    q, dout = normal(1, t, heads, dim, dtype=dtype), normal(2, t, heads, dim, dtype=dtype)
    k, v = normal(3, t, kv_heads, dim, dtype=dtype), normal(4, t, kv_heads, dim, dtype=dtype)
    print("attention", lengths, heads, kv_heads, dim, dtype, flush=True)
    want, off = ref.attention(q, k, v, starts, 1 / math.sqrt(dim), dout)
    check_all(run_attention(q.cuda(), k.cuda(), v.cuda(), starts, dout.cuda()), want, off, lengths)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 72, 80, 96, 104, 120])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("longest", [150, 77])
def test_attention_head_sizes(dim, dtype, longest):
    starts = starts_of([17, longest, 33])
    t = int(starts[-1])
    q, dout = normal(1, t, 2, dim, dtype=dtype), normal(2, t, 2, dim, dtype=dtype)
    k, v = normal(3, t, 1, dim, dtype=dtype), normal(4, t, 1, dim, dtype=dtype)
    want, off = ref.attention(q, k, v, starts, 1 / math.sqrt(dim), dout)
    check_all(run_attention(q.cuda(), k.cuda(), v.cuda(), starts, dout.cuda()), want, off, dim)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_attention_scales_and_large_logits(scale):
    starts = starts_of([90, 45])
    q, k, v, dout = (normal(i, 135, 2, 64, std=2.0) for i in range(4))
    want, off = ref.attention(q, k, v, starts, scale, dout)
    check_all(run_attention(q.cuda(), k.cuda(), v.cuda(), starts, dout.cuda(), scale), want, off, scale)


def test_attention_reads_slices_of_a_projection_in_place_and_copies_other_orders():
    starts = starts_of([70, 1, 99])
    t, heads, kv_heads, dim = 170, 4, 2, 64
    qkv = normal(5, t, heads + 2 * kv_heads, dim)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
    dout = normal(6, t, heads, dim)
    want, off = ref.attention(q, k, v, starts, 1 / 8, dout)
    a = qkv.cuda()
    split = a.split([heads, kv_heads, kv_heads], 1)
    assert ops._heads("q", split[0], t, dim)[0] is split[0]
    check_all(run_attention(*split, starts, dout.cuda()), want, off, "slices")
    # heads first; dim not side by side; rows that do not begin at multiples of 16 bytes; a broadcast gradient
    others = [x.cuda().transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    check_all(run_attention(*others, starts, dout.cuda()), want, off, "heads first")
    others = [x.cuda().transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    check_all(run_attention(*others, starts, dout.cuda()), want, off, "dim first")
    wide = torch.zeros(t, heads, dim + 3, dtype=BF16, device="cuda")
    wide[:, :, 3:] = dout.cuda()
    check_all(run_attention(*split, starts, wide[:, :, 3:]), want, off, "odd rows")
    one = normal(7, 1, 1, dim).expand(t, heads, dim)
    want, off = ref.attention(q, k, v, starts, 1 / 8, one)
    check_all(run_attention(*split, starts, one.cuda().expand(t, heads, dim)), want, off, "broadcast gradient")


@pytest.mark.parametrize("lengths,heads,kv_heads", [([100, 55], 2, 2), ([140, 15], 2, 2), ([100, 55], 8, 1), ([140, 15], 6, 2)])
def test_attention_leaves_tokens_of_no_sequence_alone(lengths, heads, kv_heads):
    """The rest of a buffer: not read (it holds NaN here), its rows of every result 0."""
    starts, t = starts_of(lengths), 155 + 210
    q, dout = normal(0, t, heads, 64), normal(3, t, heads, 64)
    k, v = normal(1, t, kv_heads, 64), normal(2, t, kv_heads, 64)
    want, off = ref.attention(q, k, v, starts, 1 / 8, dout)
    gpu = []
    for x in (q, k, v, dout):
        x = x.cuda()
        x[155:] = math.nan
        gpu.append(x)
    got = run_attention(*gpu[:3], starts, gpu[3])
    check_all(got, want, off, "rest")
    assert not got["out"][155:].any() and torch.isinf(got["lse"][:, 155:]).all()
    assert not got["dq"][155:].any() and not got["dk"][155:].any() and not got["dv"][155:].any()


@pytest.mark.parametrize("lengths,dim,kv_heads", [
    ([40, 50, 30], 64, 2), ([3, 17, 100, 8], 128, 1), ([1, 1, 5, 60], 32, 2), ([100, 28, 128], 96, 4),  # whole sequences to a tile
    ([200, 90, 300], 64, 2), ([129, 5, 140], 128, 4), ([70, 350, 9], 80, 1), ([20, 1500, 30], 128, 2)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_what_is_not_seen_does_not_matter(lengths, dim, kv_heads, dtype):
    """A NaN or infinity in one token reaches the rows whose formulas hold it and no other: not the sequences next to it
    in a tile, not the earlier rows of its own."""
    starts = starts_of(lengths)
    t, heads = int(starts[-1]), 4
    q, dout = normal(1, t, heads, dim, dtype=dtype), normal(2, t, heads, dim, dtype=dtype)
    k, v = normal(3, t, kv_heads, dim, dtype=dtype), normal(4, t, kv_heads, dim, dtype=dtype)
    want, off = ref.attention(q, k, v, starts, 1 / math.sqrt(dim), dout)
    seq = int(np.argmax(lengths))
    begin, end = int(starts[seq]), int(starts[seq + 1])
    bad = begin + (end - begin) * 2 // 3
    rows = torch.arange(t)
    for value in (math.nan, math.inf):
        # v of one token: out and dq of the rows from it on; through their delta, dk of the whole sequence; never dv
        x = v.clone()
        x[bad] = value
        got = run_attention(q.cuda(), k.cuda(), x.cuda(), starts, dout.cuda())
        hit = (rows >= bad) & (rows < end)
        whole = (rows >= begin) & (rows < end)
        for name, these in (("out", hit), ("dq", hit), ("dk", whole), ("dv", rows < 0)):
            assert not torch.isfinite(got[name].cpu()[these]).any(), (name, value)
            assert ref.close(got[name].cpu()[~these], want[name][~these], off[name][~these]), (name, value)
        assert ref.close(got["lse"], want["lse"], off["lse"])
        # the gradient of one row: its own dq, dk and dv of the keys up to it
        x = dout.clone()
        x[bad] = value
        got = run_attention(q.cuda(), k.cuda(), v.cuda(), starts, x.cuda())
        upto = (rows >= begin) & (rows <= bad)
        for name, these in (("out", rows < 0), ("dq", rows == bad), ("dk", upto), ("dv", upto)):
            finite = torch.isfinite(got[name].cpu()[these]).float().mean() if these.any() else 0
            assert finite < 0.5, (name, value, finite)  # (a weight that has become 0 in 16 bits times infinity is NaN too)
            assert ref.close(got[name].cpu()[~these], want[name][~these], off[name][~these]), (name, value)


def test_attention_of_tokens_that_lie_far_apart():
    """Strides of up to 32 MiB a token: the last ones lie 8 GB behind the first, and 128 rows of a tile span 4 GiB."""
    lengths = [200, 31, 20]
    starts, tokens = starts_of(lengths), sum(lengths)
    room = torch.empty(tokens << 24, dtype=BF16, device="cuda")
    wide = [room.as_strided((tokens, heads, 64), (1 << 24, 64, 1), at) for heads, at in ((4, 0), (2, 4096), (2, 8192), (4, 16384))]
    for i, x in enumerate(wide):
        x.copy_(normal(i, *x.shape))
    for length in (lengths, [120, 111, 20]):
        starts = starts_of(length)
        got = run_attention(*wide[:3], starts, wide[3])
        want = run_attention(*(x.contiguous() for x in wide[:3]), starts, wide[3].contiguous())
        for name in got:
            assert torch.equal(got[name], want[name]), name
    del room, wide
    torch.cuda.empty_cache()


@pytest.mark.parametrize("length", [96, 160])
def test_attention_of_more_elements_than_32_bits_count(length):
    """The last sequences of a batch of 2^32 elements and more give what they give alone."""
    heads, kv_heads, dim = 64, 2, 128
    tokens = (2 ** 32 // (heads * dim) // length + 20) * length
    starts = np.arange(0, tokens + 1, length, dtype=np.int32)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.zeros(tokens, n, dim, dtype=BF16, device="cuda") for n in (heads, kv_heads, kv_heads, heads)]
    last = slice(tokens - 10 * length, tokens)
    for t in x:
        t[last].normal_(generator=gen)
        t[:length].normal_(generator=gen)
    got = run_attention(*x[:3], starts, x[3])
    assert x[0].numel() > 2 ** 32
    for part, n in ((last, 10), (slice(0, length), 1)):
        q, k, v, dout = (t[part].contiguous().cpu() for t in x)
        want, off = ref.attention(q, k, v, starts[:n + 1], 1 / math.sqrt(dim), dout)
        for name in got:
            assert ref.close(got[name][:, part] if name == "lse" else got[name][part], want[name], off[name]), name
    del x, got
    torch.cuda.empty_cache()


def test_attention_without_any_sequence():
    for starts, t in (([0], 0), ([0], 5), ([0, 0, 0], 5)):
        x = normal(1, t, 2, 32).cuda()
        got = run_attention(x, x, x, starts, x, tokens=t)
        assert got["out"].shape == (t, 2, 32) and not got["out"].any() and not got["dk"].any()


def test_attention_gradients_against_differences():
    """Directional derivatives of a fixed combination of the outputs, from the kernel's own outputs in the steps."""
    starts, t, dim = starts_of([40, 21]), 61, 32
    q, k, v, dout = (normal(i, t, 2, dim, dtype=F16) for i in range(4))
    seq = ops.PackedSequences(starts)
    args = [x.cuda().requires_grad_() for x in (q, k, v)]
    (ops.packed_attention(*args, seq) * dout.cuda()).sum().backward()
    step = 2.0 ** -4
    for i, x in enumerate((q, k, v)):
        direction = torch.sign(normal(9 + i, *x.shape, dtype=F16))
        value = []
        for sign in (1, -1):
            moved = [y.double() for y in (q, k, v)]
            moved[i] = moved[i] + sign * step * direction.double()
            # the moved inputs are exact in float16 only by chance: the definition is moved, the kernel's slope compared
            want, _ = ref.attention(*[_Double(y) for y in moved], starts, 1 / math.sqrt(dim))
            value.append(float((want["out"] * dout.double()).sum()))
        slope = (value[0] - value[1]) / (2 * step)
        mine = float((args[i].grad.cpu().double() * direction.double()).sum())
        # the third derivative's share of a central difference, and t * 2 * dim roundings of 2^-11 of values near 1
        assert abs(mine - slope) <= 0.02 * abs(slope) + 2.0, (i, mine, slope)


class _Double:
    """A 64-bit tensor that the reference treats as float16 inputs (it only asks for a type's unit)."""

    def __init__(self, x):
        self._x, self.dtype = x, F16

    def double(self):
        return self._x


def test_attention_is_the_same_on_another_stream_and_in_a_graph():
    starts = starts_of([200, 77, 3])
    q, k, v, dout = (normal(i, 280, 4, 64).cuda() for i in range(4))
    seq = ops.PackedSequences(starts)

    def step():
        out, lse = ops.packed_attention_forward(q, k, v, seq)
        return (out, *ops.packed_attention_backward(dout, q, k, v, out, lse, seq))

    want = [x.clone() for x in step()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = step()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        for x in got:
            x.zero_()
        q.copy_(q.roll(1, 0) if i == 1 else q)
        want = [x.clone() for x in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_attention_refuses():
    x = normal(1, 10, 4, 64).cuda()
    seq = ops.PackedSequences([0, 10])
    out, lse = ops.packed_attention_forward(x, x, x, seq)

    def refused(match, fn, *args, **kw):
        with pytest.raises(NextDoorError, match=match):
            fn(*args, **kw)

    forward, backward = ops.packed_attention_forward, ops.packed_attention_backward
    refused("16-bit", forward, x.float(), x.float(), x.float(), seq)
    refused("different types", forward, x, x.half(), x, seq)
    refused("GPU only", forward, x.cpu(), x, x, seq)
    refused("10 tokens", forward, x[:9], x, x, seq)
    refused("another head size", forward, x, x[..., :32], x[..., :32], seq)
    refused("different shapes", forward, x, x[:, :2], x, seq)
    refused("evenly", forward, x, x[:, :3], x[:, :3], seq)
    refused("multiple of 8", forward, x[..., :12], x[..., :12], x[..., :12], seq)
    wide = normal(1, 10, 1, 136).cuda()
    refused("multiple of 8 up to 128", forward, wide, wide, wide, seq)
    refused("not finite", forward, x, x, x, seq, math.inf)
    refused("dout", backward, x[:, :2], x, x, x, out, lse, seq)
    refused("forward pass's", backward, x, x, x, x, out, lse[:2], seq)
    refused("not 0", ops.PackedSequences, [1, 10])
    refused("before it starts", ops.PackedSequences, [0, 5, 4, 10])
    refused("10 tokens in sequences, 9", ops.PackedSequences, [0, 10], 9)
    refused("list of integers", ops.PackedSequences, [0.0, 10.0])
    refused("integers", ops.PackedSequences, torch.tensor([0.0, 10.0]))


# ---- vocabulary loss -----------------------------------------------------------------------------


def run_loss(hidden, weight, target, dloss):
    loss, lse = ops.vocabulary_loss_forward(hidden, weight, target)
    dhidden, dweight = ops.vocabulary_loss_backward(dloss, hidden, weight, target, lse)
    torch.cuda.synchronize()
    return {"loss": loss, "lse": lse, "dhidden": dhidden, "dweight": dweight}


def targets(seed, rows, classes):
    """A fifth of them no class: -1, |V|, far out."""
    rng = np.random.default_rng(seed)
    t = rng.integers(0, classes, rows)
    none = rng.random(rows) < 0.2
    t[none] = rng.choice([-1, classes, 2 ** 31 - 1, -2 ** 31], int(none.sum()))
    return torch.from_numpy(t)


@pytest.mark.parametrize("rows,classes,dim,dtype", [
    (1, 1, 8, BF16), (1, 2711, 64, F16), (61, 2711, 64, BF16), (128, 128, 64, BF16), (129, 257, 72, F16),
    (127, 1, 16, BF16), (300, 1000, 128, BF16), (33, 5003, 200, F16), (257, 4099, 520, BF16), (1000, 31, 40, F16),
    (2, 70001, 32, BF16), (700, 3001, 256, BF16), (513, 2049, 264, F16)])
def test_loss_and_gradients(rows, classes, dim, dtype):
    print("loss", rows, classes, dim, dtype, flush=True)
    h, w = normal(1, rows, dim, dtype=dtype), normal(2, classes, dim, dtype=dtype, std=2 / math.sqrt(dim))
    t = targets(3, rows, classes)
    dloss = (0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(4))) / rows
    want, off = ref.vocabulary_loss(h, w, t, dloss)
    check_all(run_loss(h.cuda(), w.cuda(), t.cuda(), dloss.cuda()), want, off, (rows, classes, dim))
    got = run_loss(h.cuda(), w.cuda(), t.to(torch.int32).cuda(), dloss.cuda())
    check_all(got, want, off, "32-bit targets")


@pytest.mark.parametrize("dim", [96, 128, 136, 160, 168, 192, 200, 224, 232, 256, 272])
@pytest.mark.parametrize("rows,classes,dtype", [(300, 1501, BF16), (77, 4100, F16), (2100, 130, BF16)])
def test_loss_of_vectors_around_those_that_stay_in_registers(rows, classes, dtype, dim):
    h, w = normal(1, rows, dim, dtype=dtype), normal(2, classes, dim, dtype=dtype, std=2 / math.sqrt(dim))
    t = targets(3, rows, classes)
    dloss = (0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(4))) / rows
    want, off = ref.vocabulary_loss(h, w, t, dloss)
    check_all(run_loss(h.cuda(), w.cuda(), t.cuda(), dloss.cuda()), want, off, (rows, classes, dim))


@pytest.mark.parametrize("dim", [264, 392, 1000])
@pytest.mark.parametrize("rows,classes,dtype", [(129, 50, BF16), (500, 3001, F16), (1090, 6399, BF16), (1090, 6401, BF16)])
def test_loss_of_longer_vectors_in_few_and_in_many_tiles(rows, classes, dtype, dim):
    h, w = normal(1, rows, dim, dtype=dtype), normal(2, classes, dim, dtype=dtype, std=2 / math.sqrt(dim))
    t = targets(3, rows, classes)
    dloss = (0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(4))) / rows
    want, off = ref.vocabulary_loss(h, w, t, dloss)
    check_all(run_loss(h.cuda(), w.cuda(), t.cuda(), dloss.cuda()), want, off, (rows, classes, dim))


def test_loss_goes_through_several_pieces_of_the_vocabulary():
    """More rows than one piece's workspace holds for all classes; checked against products in 32 bits on the GPU, which
    agree with 64 bits to SMALL of the sums of magnitudes."""
    rows, classes, dim = 20000, 9001, 64
    h, w = normal(1, rows, dim).cuda(), normal(2, classes, dim, std=0.25).cuda()
    t = targets(3, rows, classes).cuda()
    dloss = (0.5 + torch.rand(rows, device="cuda")) / rows
    got = run_loss(h, w, t, dloss)
    z = h.double() @ w.double().T
    lse = torch.logsumexp(z, 1)
    g = torch.exp(z - lse[:, None])
    has = (t >= 0) & (t < classes)
    g[has.nonzero()[:, 0], t[has]] -= 1
    g *= torch.where(has, dloss, torch.zeros_like(dloss)).double()[:, None]
    assert torch.allclose(got["lse"].double(), lse, rtol=0, atol=2.0 ** -13)
    for name, value, spread in (("dhidden", g @ w.double(), g.abs() @ w.double().abs()),
                                ("dweight", g.T @ h.double(), g.abs().T @ h.double().abs())):
        off = 2.0 ** -8 * (value.abs() + spread) + ref.SMALL * 4 * spread
        assert ((got[name].double() - value).abs() <= off).all(), name


def test_loss_of_more_rows_than_are_taken_at_a_time():
    """A few rows and classes of many, in 64 bits on the GPU.  Forward: rows in pieces of 8192 for so many classes;
    backward: vectors too long to keep gradients in registers, the classes in two pieces."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    def some(rows, classes, dim):
        h = torch.randn(rows, dim, device="cuda", generator=gen).to(BF16)
        w = (torch.randn(classes, dim, device="cuda", generator=gen) * (2 / math.sqrt(dim))).to(BF16)
        return h, w, targets(rows, rows, classes).cuda()

    def logits(h, w):
        """and how far they may be off: dim products summed in 32 bits"""
        z = h.double() @ w.double().T
        off = (h.shape[1] + 8) * 2.0 ** -24 * (h.double().abs() @ w.double().abs().T).amax(1) + 2.0 ** -21 * z.abs().amax(1)
        return z, off

    h, w, t = some(8503, 262100, 264)
    loss, lse = ops.vocabulary_loss_forward(h, w, t)
    at = torch.tensor([0, 1, 4095, 8190, 8191, 8192, 8193, 8447, 8448, 8502], device="cuda")
    z, z_off = logits(h[at], w)
    want = torch.logsumexp(z, 1)
    assert ((lse[at].double() - want).abs() <= z_off + 2.0 ** -13).all()
    has = (t[at] >= 0) & (t[at] < len(w))
    mine = z.gather(1, torch.where(has, t[at], torch.zeros_like(t[at]))[:, None])[:, 0]
    assert ((loss[at].double() - torch.where(has, want - mine, torch.zeros_like(mine))).abs() <= 2 * z_off + 2.0 ** -13).all()

    h, w, t = some(16700, 40001, 232)
    dloss = (0.5 + torch.rand(len(h), device="cuda", generator=gen)) / len(h)
    loss, lse = ops.vocabulary_loss_forward(h, w, t)
    dhidden, dweight = ops.vocabulary_loss_backward(dloss, h, w, t, lse)
    each = torch.where((t >= 0) & (t < len(w)), dloss, torch.zeros_like(dloss)).double()
    for row0 in (0, 8256, 16636):  # all classes
        rows = slice(row0, row0 + 64)
        z, z_off = logits(h[rows], w)
        p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) * each[rows, None]
        g = p - each[rows, None] * (t[rows, None] == torch.arange(len(w), device="cuda"))
        value = g @ w.double()
        g_off = (2.0 ** -8 + ref.SMALL) * g.abs() + (2 * z_off[:, None] + ref.SMALL) * p
        assert ((dhidden[rows].double() - value).abs() <= 2.0 ** -8 * value.abs() + g_off @ w.double().abs()).all()
    for class0 in (0, 31936, 32000, 39937):  # all rows
        classes = slice(class0, class0 + 64)
        z, z_off = logits(h, w[classes])
        p = torch.exp(z - lse.double()[:, None]) * each[:, None]
        g = p - each[:, None] * (t[:, None] == torch.arange(class0, class0 + 64, device="cuda"))
        value = g.T @ h.double()
        g_off = (2.0 ** -8 + ref.SMALL) * g.abs() + (2 * (z_off[:, None] + 2.0 ** -13) + ref.SMALL) * p
        assert ((dweight[classes].double() - value).abs() <= 2.0 ** -8 * value.abs() + g_off.T @ h.double().abs()).all()


@pytest.mark.parametrize("dim", [64, 512])
def test_loss_of_more_elements_than_32_bits_count(dim):
    """A vocabulary of over 2^32 elements: three rows' loss, and the gradients of its first and last classes."""
    rows, classes = 3, 2 ** 32 // dim + 1001
    gen = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(rows, dim, device="cuda", generator=gen).to(BF16)
    w = torch.zeros(classes, dim, dtype=BF16, device="cuda")
    ends = torch.cat([torch.arange(500, device="cuda"), torch.arange(classes - 500, classes, device="cuda")])
    w[ends] = (torch.randn(1000, dim, device="cuda", generator=gen) * (8 / math.sqrt(dim))).to(BF16)
    t = torch.tensor([classes - 7, 3, classes], device="cuda")
    loss, lse = ops.vocabulary_loss_forward(h, w, t)
    dloss = torch.full((rows,), 1000.0, device="cuda")
    dhidden, dweight = ops.vocabulary_loss_backward(dloss, h, w, t, lse)
    # all other logits are 0
    z = h.double() @ w[ends].double().T
    z_off = (dim + 8) * 2.0 ** -24 * (h.double().abs() @ w[ends].double().abs().T).amax(1) + 2.0 ** -21 * z.abs().amax(1) + 2.0 ** -21 * 20
    want = torch.logsumexp(torch.cat([z, torch.full((rows, 1), math.log(classes - 1000), dtype=torch.float64, device="cuda")], 1), 1)
    assert ((lse.double() - want).abs() <= z_off + 2.0 ** -13).all()
    target = torch.tensor([[993], [3]], device="cuda")
    assert ((loss[:2].double() - (want[:2] - z[:2].gather(1, target)[:, 0])).abs() <= 2 * z_off[:2] + 2.0 ** -13).all() and loss[2] == 0
    p = torch.exp(z - want[:, None]) * 1000
    p[2] = 0
    g = p.clone()
    g[[0, 1], target[:, 0]] -= 1000
    g_off = (2.0 ** -8 + ref.SMALL) * g.abs() + (2 * (z_off[:, None] + 2.0 ** -13) + ref.SMALL) * p
    for got, value, off in ((dhidden, g @ w[ends].double(), g_off @ w[ends].double().abs()),
                            (dweight[ends], g.T @ h.double(), g_off.T @ h.double().abs())):
        assert ((got.double() - value).abs() <= 2.0 ** -8 * value.abs() + off).all()
    del w, dweight
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_loss_of_peaked_and_of_tiny_gradients(dtype):
    """Rows whose target has nearly all the weight, logits in the hundreds, and the tiny gradients of a large mean."""
    rows, classes, dim = 200, 700, 64
    h, w = normal(1, rows, dim, dtype=dtype, std=3.0), normal(2, classes, dim, dtype=dtype, std=3.0)
    t = (h.double() @ w.double().T).argmax(1)
    for size in (1.0, 1e-7):
        dloss = torch.rand(rows, generator=torch.Generator().manual_seed(4)) * size
        want, off = ref.vocabulary_loss(h, w, t, dloss)
        check_all(run_loss(h.cuda(), w.cuda(), t.cuda(), dloss.cuda()), want, off, size)


def test_loss_rows_without_a_target_send_nothing_back():
    h, w = normal(1, 50, 32).cuda(), normal(2, 100, 32).cuda()
    h[7] = math.nan
    t = torch.full((50,), 100, device="cuda")
    loss, lse = ops.vocabulary_loss_forward(h, w, t)
    dh, dw = ops.vocabulary_loss_backward(torch.full((50,), math.inf, device="cuda"), h, w, t, lse)
    assert not loss.any() and not dh.any()


def test_loss_without_rows():
    h, w = normal(1, 0, 32).cuda(), normal(2, 100, 32).cuda()
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    loss, lse = ops.vocabulary_loss_forward(h, w, t)
    dh, dw = ops.vocabulary_loss_backward(loss, h, w, t, lse)
    assert loss.shape == (0,) and dh.shape == (0, 32) and dw.shape == (100, 32) and not dw.any()


@pytest.mark.parametrize("dim", [1, 7, 50])
def test_loss_of_odd_vectors_and_orders(dim):
    h, w, t = normal(1, 40, dim), normal(2, 90, dim), targets(3, 40, 90)
    dloss = torch.ones(1).expand(40)
    want, off = ref.vocabulary_loss(h, w, t, dloss)
    got = run_loss(h.cuda(), w.T.contiguous().T.cuda(), t.cuda(), dloss.cuda().expand(40))
    assert got["dhidden"].shape == h.shape and got["dweight"].shape == w.shape
    check_all(got, want, off, dim)


def test_loss_gradients_against_differences():
    rows, classes, dim = 30, 400, 64
    h, w, t = normal(1, rows, dim, dtype=F16), normal(2, classes, dim, dtype=F16, std=0.2), targets(3, rows, classes)
    a, b = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    ops.vocabulary_loss(a, b, t.cuda()).sum().backward()
    step = 2.0 ** -8
    for i, grad in enumerate((a.grad, b.grad)):
        direction = torch.sign(normal(9 + i, *(h, w)[i].shape, dtype=F32)).double()
        value = []
        for sign in (1, -1):
            moved = [h.double(), w.double()]
            moved[i] = moved[i] + sign * step * direction
            z = moved[0] @ moved[1].T
            has = (t >= 0) & (t < classes)
            value.append(float((torch.logsumexp(z, 1)[has] - z[has, t[has]]).sum()))
        slope = (value[0] - value[1]) / (2 * step)
        mine = float((grad.cpu().double() * direction).sum())
        # roundings of 2^-11 of each entry, of random sign here, and the third derivative's share
        off = 2.0 ** -11 * float(grad.cpu().double().abs().sum()) + 2e-3 * abs(slope) + 0.05
        assert abs(mine - slope) <= off, (i, mine, slope)


def test_loss_is_the_same_in_a_graph():
    h, w = normal(1, 300, 64).cuda(), normal(2, 5000, 64, std=0.2).cuda()
    t = targets(3, 300, 5000).to(torch.int32).cuda()
    dloss = torch.full((300,), 1 / 300, device="cuda")

    def step():
        loss, lse = ops.vocabulary_loss_forward(h, w, t)
        return (loss, *ops.vocabulary_loss_backward(dloss, h, w, t, lse))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        for x in got:
            x.zero_()
        h.copy_(h.roll(1, 0))
        want = [x.clone() for x in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_loss_refuses():
    h, w = normal(1, 10, 64).cuda(), normal(2, 30, 64).cuda()
    t = torch.zeros(10, dtype=torch.int64, device="cuda")
    _, lse = ops.vocabulary_loss_forward(h, w, t)

    def refused(match, fn, *args):
        with pytest.raises(NextDoorError, match=match):
            fn(*args)

    forward, backward = ops.vocabulary_loss_forward, ops.vocabulary_loss_backward
    refused("16-bit", forward, h.float(), w.float(), t)
    refused("different types", forward, h, w.half(), t)
    refused("equally long", forward, h, w[:, :32], t)
    refused("one target", forward, h, w, t[:9])
    refused("int32 or int64", forward, h, w, t.float())
    refused("GPU only", forward, h, w, t.cpu())
    refused("classes", forward, h, w[:0], t)
    refused("one value for each row", backward, lse[:9], h, w, t, lse)


# ---- dropout ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (7,), (8,), (9,), (101, 64), (33, 31), (5000, 21), (2, 3, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(shape, dtype, p):
    x, r = normal(1, *shape, dtype=dtype), normal(2, *shape, dtype=dtype)
    seed, step = 0xFEDCBA9876543210, 17
    want, off = ref.dropout(x, p, seed, step)
    got = ops.dropout_forward(x.cuda(), p, seed, step)
    assert ref.close(got, want, off)
    assert torch.equal(got, ops.dropout_backward(x.cuda(), p, seed, step))
    want, off = ref.dropout(x, p, seed, step, r)
    assert ref.close(ops.dropout_forward(x.cuda(), p, seed, step, residual=r.cuda()), want, off)


def test_dropout_uses_the_samplers_stream():
    import nextdoor_amd as nd
    n, seed, step = 10007, 42, 3
    kept = nd.philox_fill_uniform(seed, step, 0, n, 1, step_size=2)[:, 0] >= np.float32(0.3)
    got = ops.dropout_forward(torch.ones(n, device="cuda"), 0.3, seed, step).cpu().numpy()
    assert np.array_equal(got != 0, kept)


def test_dropout_of_more_elements_than_one_row_of_workgroups_has():
    import nextdoor_amd as nd
    n, seed, step = 2 ** 33 + 1003, 42, 3
    x = torch.empty(n, dtype=BF16, device="cuda")
    places = [0, 2 ** 32 - 500, 2 ** 33 - 500, n - 1000]
    for at in places:
        x[at:at + 1000] = 1
    y = ops.dropout_forward(x, 0.3, seed, step)
    for at in places:
        kept = nd.philox_fill_uniform(seed, step, at, 1000, 1, step_size=2)[:, 0] >= np.float32(0.3)
        assert np.array_equal((y[at:at + 1000] != 0).cpu().numpy(), kept), at
    del x, y
    torch.cuda.empty_cache()


def test_dropout_drops_whatever_is_there_and_reads_odd_places():
    x = normal(1, 4001, dtype=F32).cuda()
    kept = ops.dropout_forward(torch.ones_like(x), 0.5, 1, 1) != 0
    bad = torch.where(kept, x, torch.full_like(x, math.nan))
    assert torch.equal(ops.dropout_forward(bad, 0.5, 1, 1), ops.dropout_forward(x, 0.5, 1, 1))
    for dtype in (F32, BF16):
        y = x.to(dtype)
        assert torch.equal(ops.dropout_forward(y[1:], 0.5, 1, 1), ops.dropout_forward(y[1:].clone(), 0.5, 1, 1))
        m = y[:4000].view(50, 80)
        assert torch.equal(ops.dropout_forward(m.T, 0.5, 1, 1), ops.dropout_forward(m.T.contiguous(), 0.5, 1, 1))


def test_dropout_gradients():
    x = normal(1, 77, 33, dtype=F32).cuda().requires_grad_()
    r = normal(2, 77, 33, dtype=F32).cuda().requires_grad_()
    d = normal(3, 77, 33, dtype=F32).cuda()
    ops.dropout(x, 0.2, 9, 5, r).backward(d)
    want, off = ref.dropout(d.cpu(), 0.2, 9, 5)
    assert ref.close(x.grad, want, off) and torch.equal(r.grad, d)


def test_dropout_refuses():
    x = torch.ones(8, device="cuda")
    for args in ((x, -0.1, 1, 1), (x, 1.5, 1, 1), (x, math.nan, 1, 1), (x, 0.5, -1, 1), (x, 0.5, 1 << 64, 1), (x, 0.5, 1, 1 << 31),
                 (x.double(), 0.5, 1, 1), (x.cpu(), 0.5, 1, 1), (x, 0.5, 1, 1, x[:7]), (x, 0.5, 1, 1, x.half())):
        with pytest.raises(NextDoorError):
            ops.dropout_forward(*args)
    assert ops.dropout_forward(x[:0], 0.5, 1, 1).shape == (0,)


# ---- together --------------------------------------------------------------------------------------


def test_a_walk_model_learns():
    """Walks from the engine, packed, through all three operators, forward and backward: the loss falls from that of a guess,
    and the same seeds give the same losses."""
    from nextdoor_amd import Graph, walk_model
    graph = Graph.chung_lu(500, 6000, 2.2, seed=3)
    losses = [walk_model.train(graph, steps=30, walks=400, seed=5, log=None, dropout=0.1)[1] for _ in range(2)]
    assert abs(losses[0][0] - math.log(500)) < 1.0
    assert losses[0][-1] < losses[0][0] - 0.5
    assert losses[0][0] == losses[1][0]


def test_walk_model_gradients_are_those_of_plain_operations():
    """One step of the model in 16 bits against the same model with the definitions in 64 bits."""
    from nextdoor_amd import walk_model
    torch.manual_seed(1)
    n, width = 97, 64
    rng = np.random.default_rng(2)
    samples = rng.integers(0, n, (20, 30)).astype(np.int32)
    for walk in samples[::2]:
        walk[rng.integers(0, 30):] = n
    tokens, targets, starts = walk_model.pack_walks(rng.integers(0, n, 20), samples, n)
    model = walk_model.WalkModel(n, width=width, heads=2, kv_heads=1, layers=1, dropout=0.2).to("cuda", BF16)
    batch = walk_model.batch_of(tokens, targets, starts)
    each = model(*batch[:3], batch[3], 11)
    each.sum().backward()

    exact = walk_model.WalkModel(n, width=width, heads=2, kv_heads=1, layers=1, dropout=0.2).double()
    exact.load_state_dict({k: v.double().cpu() for k, v in model.state_dict().items()})

    def attention(q, k, v, sequences, scale=None):
        of = torch.from_numpy(np.repeat(np.arange(len(starts) - 1), np.diff(starts)))
        at = torch.arange(len(of))
        sees = (of[:, None] == of) & (at[:, None] >= at)
        out = []
        for h in range(q.shape[1]):
            s = (q[:, h] @ k[:, h // (q.shape[1] // k.shape[1])].T / math.sqrt(q.shape[2])).masked_fill(~sees, -math.inf)
            out.append(torch.softmax(s, 1) @ v[:, h // (q.shape[1] // k.shape[1])])
        return torch.stack(out, 1)

    def drop(x, p, seed, step, residual=None):
        kept = torch.from_numpy(ref.uniforms(x.numel(), seed, step) >= np.float32(p)).view(x.shape)
        y = x * kept / (1 - p)
        return y if residual is None else y + residual

    def loss(h, w, t):
        has = (t >= 0) & (t < n)
        z = h @ w.T
        return torch.where(has, torch.logsumexp(z, 1) - z.gather(1, torch.where(has, t, 0).long()[:, None])[:, 0], 0.0)

    kept = ops.packed_attention, ops.dropout, ops.vocabulary_loss
    try:
        ops.packed_attention, ops.dropout, ops.vocabulary_loss = attention, drop, loss
        want = exact(batch[0].cpu(), batch[1].cpu(), batch[2].cpu(), None, 11)
        want.sum().backward()
    finally:
        ops.packed_attention, ops.dropout, ops.vocabulary_loss = kept
    # the model itself works in bfloat16 throughout: a dozen roundings of 2^-9 each on a path, of random sign
    assert abs(float(each.detach().sum()) / float(want.detach().sum()) - 1) < 0.02
    for (name, a), (_, b) in zip(model.named_parameters(), exact.named_parameters()):
        off = float((a.grad.double().cpu() - b.grad).norm() / b.grad.norm())
        assert off < 0.05, (name, off)
