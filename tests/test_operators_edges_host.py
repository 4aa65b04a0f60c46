"""What the training operators' torch functions hand to the kernels, and the sizes they ask for, before a GPU is touched."""
import pytest
import torch

from nextdoor_amd import _capi, ops

BF16 = torch.bfloat16


def filled(*shape):
    return torch.arange(torch.Size(shape).numel(), dtype=torch.float32).view(shape).to(BF16)


@pytest.mark.parametrize("what,make", [
    ("one token of an odd row", lambda: filled(3, 131)[:1, :128].view(1, 2, 64)),
    ("one token, one head, an odd place", lambda: filled(3, 1, 67)[:1, :, 3:]),
    ("one token of rows farther apart than the kernels go", lambda: torch.zeros(16, dtype=BF16).as_strided((1, 2, 8), (1 << 25, 8, 1))),
    ("one head that lies anywhere", lambda: filled(5, 64).as_strided((5, 1, 64), (64, 3, 1))),
    ("several tokens of odd rows", lambda: filled(5, 131)[:, :128].unflatten(1, (2, 64))),
    ("an odd place", lambda: filled(5, 2, 67)[:, :, 3:]),
    ("dim first", lambda: filled(64, 2, 5).permute(2, 1, 0)),
    ("slices of a projection", lambda: filled(5, 6, 64)[:, 4:]),
    ("no token", lambda: filled(5, 2, 67)[:0, :, 3:]),
    ("a broadcast token", lambda: filled(1, 2, 64).expand(5, 2, 64))])
def test_heads_reach_the_kernels_aligned_and_in_order(what, make):
    """What the kernels read: rows of dim side by side at multiples of 16 bytes, the strides given."""
    x = make()
    tokens, heads, dim = x.shape
    y, a, b = ops._heads(what, x, tokens, dim)
    assert a % 8 == 0 and b % 8 == 0 and 0 <= a <= 16777216 and 0 <= b and y.data_ptr() % 16 == 0
    assert torch.equal(y.as_strided(x.shape, (a, b, 1)), x)


def test_slices_that_can_be_read_in_place_are_not_copied():
    qkv = filled(5, 6, 64)
    for x in qkv.split([4, 1, 1], 1):
        assert ops._heads("q", x, 5, 64)[0] is x


@pytest.mark.parametrize("rows,classes,dim", [
    (4096, 131072, 1024), (16700, 40001, 232), (65536, 131072, 4096), (131072, 131072, 4096), (32768, 131072, 8192), (262144, 50000, 65536),
    (1 << 20, 20000, 300), (1 << 21, 20000, 8192), (4194240, 3000, 4096), (4194240, 131072, 264)])
def test_the_loss_keeps_a_few_gib_of_gradients_however_many_rows_there_are(rows, classes, dim):
    """What the backward call asks for beyond the rows themselves in 16 bits (once) and the sums of their gradients: g of one piece of the
    classes, up to 4 GiB, or 1024 classes where that is more, filled up to a multiple of 256."""
    dim = -(-dim // 8) * 8
    size = _capi.lib().nd_vocabulary_loss_workspace(rows, classes, dim, 1)
    padded = -(-rows // 256) * 256
    g = max(4 << 30, 2 * padded * 1024) + 2 * padded * 256
    # (rows that do not fill the GPU leave several sums of dh, and dw's of one piece)
    shares = max(1, 256 // (padded // 256 * -(-dim // 256)))
    assert 0 < size <= g + padded * dim * 2 + shares * rows * dim * 4 + 12 * padded + 4096, (size - g) / 2 ** 30
