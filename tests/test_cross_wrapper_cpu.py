"""What CrossAttention does around the library's calls, without a GPU."""
import pytest
import torch

from zenyx_amd import kv
from zenyx_amd.train import cross_attention as ca


@pytest.mark.parametrize("strides, group, copied", [
    ((128, 64, 1), 1, False), ((256, 64, 1), 2, False), ((0, 64, 1), 1, False), ((64, 1 << 20, 1), 4, False),
    ((1 << 23, 64, 1), 1, True),            # rows further apart than the kernels' 32-bit offsets go
    ((64, 1 << 26, 1), 8, True), ((64, 1 << 26, 1), 1, False), ((64, 1 << 26, 1), 7, False),
    ((128, 64, 2), 1, True), ((132, 64, 1), 1, True), ((128, 68, 1), 1, True)])
def test_gradients_are_laid_out_as_the_kernels_take_them(strides, group, copied):
    t = torch.empty_strided((2, 2, 64), strides, dtype=torch.bfloat16)
    got = ca._strided(t, group)
    assert torch.equal(got.view(torch.int16), t.contiguous().view(torch.int16))
    assert (got.data_ptr() != t.data_ptr()) == copied
    assert got.is_contiguous() or not copied


@pytest.mark.parametrize("shape, strides", [((1, 2, 64), (5, 64, 1)), ((2, 1, 64), (64, 3, 1)), ((1, 1, 64), (1 << 30, 7, 1))])
def test_strides_of_single_rows_and_heads(shape, strides):
    """Which torch leaves as anything, in tensors that it calls contiguous too."""
    t = torch.empty_strided(shape, strides, dtype=torch.float16)
    got = ca._strided(t, 1)
    assert torch.equal(got.view(torch.int16), t.view(torch.int16))
    assert got.stride() == (shape[1] * 64, 64, 1) and got.data_ptr() % 16 == 0
