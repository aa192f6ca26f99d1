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


def test_errors_can_be_seen(monkeypatch):
    """err reaches the forward pass and the gradients, check the forward pass, with and without autograd."""
    seen = []

    def forward(q, k, v, cu_q, cu_k, return_lse=False, **kw):
        seen.append(("forward", kw["check"], kw["err"]))
        return (torch.zeros_like(q), torch.zeros(q.shape[1], q.shape[0])) if return_lse else torch.zeros_like(q)

    def backward(grad, q, k, v, out, lse, cu_q, cu_k, err=None, **kw):
        seen.append(("backward", False, err))
        return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    monkeypatch.setattr(kv, "cross_attention", forward)
    monkeypatch.setattr(kv, "cross_attention_backward", backward)
    q, k = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32) for n in (3, 5))
    err = torch.zeros(1, dtype=torch.int32)
    attend = ca.CrossAttention()
    for kw, want in (({}, (False, None)), (dict(check=True), (True, None)), (dict(err=err), (False, err)),
                     (dict(err=err, check=True), (True, err))):
        attend(q, k, k, cu_q, cu_k, **kw)
        attend(q.clone().requires_grad_(), k, k, cu_q, cu_k, **kw).sum().backward()
        (a, check, e), (b, check2, e2), (c, _, e3) = seen
        assert (a, b, c) == ("forward", "forward", "backward") and check == check2 == want[0]
        assert e is want[1] and e2 is want[1] and e3 is want[1]
        del seen[:]
