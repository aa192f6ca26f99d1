"""GPU attention to shared pages where a sequence has more rows than the call computes: the rows that are
written are at their own positions (tolerances: test_gpu_shared.py)."""
import pytest
import torch

from test_gpu_shared import Batch

from zenyx_amd import _native as N

pytestmark = pytest.mark.gpu

CASES = [  # groups, own, rows, Hq, Hkv, D
    ([(3, 64)], [20] * 3, [2, 5, 1], 8, 2, 64),
    ([(3, 64)], [20] * 3, [2, 5, 1], 4, 4, 128),
    ([(24, 160)], [30 + i for i in range(24)], [1 + i % 6 for i in range(24)], 8, 2, 128),  # many columns
    ([(2, 128), (2, 0)], [2, 0, 300, 4], [5, 7, 40, 4], 8, 2, 128),  # rows among the shared positions
    ([(3, 48)], [40, 9, 17], [9, 3, 6], 8, 4, 256),
]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("most", [1, 2, 3])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_rows_of_overlong_sequences_see_no_later_tokens(dev, bits, most, case):
    """Row i of n is at position seq_lens[b] - n + i, with n what cu_q says, whatever the bound is."""
    groups, own, rows, Hq, Hkv, D = CASES[case]
    t = Batch(dev, bits, groups, own, rows, Hq, Hkv, D, 16, seed=20 + case)
    whole = t.call(check=True)
    t.check(whole)
    beyond = torch.cat([torch.arange(n) >= most for n in rows]).to(dev)
    for causal in (True, False):
        out = torch.full_like(t.q, 7.0)
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        t.call(max_q_per_seq=most, out=out, err=err, causal=causal)
        assert int(err) == N.ZX_KERR_POS_RANGE and (out[beyond] == 7).all()
        out[beyond] = (whole if causal else t.call(causal=False))[beyond]
        t.check(out, causal=causal)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_rows_that_reach_beyond_q(dev, bits, case):
    """The last sequence claims rows that q does not have: those that it has are at their positions."""
    groups, own, rows, Hq, Hkv, D = CASES[case]
    t = Batch(dev, bits, groups, own, rows[:-1] + [rows[-1] + 3], Hq, Hkv, D, 16, seed=30 + case)
    whole, q = t.call(check=True), t.q
    t.q = q[:-3].contiguous()
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    got = t.call(max_q_per_seq=max(t.rows), err=err)
    assert int(err) == N.ZX_KERR_POS_RANGE and got.shape == t.q.shape
    t.q = q
    t.check(torch.cat([got, whole[-3:]]))
