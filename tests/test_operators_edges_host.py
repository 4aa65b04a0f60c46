"""What the training operators' torch functions hand to the kernels, and the sizes they ask for, before a GPU is touched."""
import pytest
import torch

from nextdoor_amd import ops

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
