"""GPU cross attention and its gradients where bounds or cu_q, cu_k leave rows and keys out: what is not
computed is zeros, not what the memory held before (tolerances: test_gpu_cross.py)."""
import pytest
import torch

from test_gpu_cross import TYPES, exact, i32, inputs, near, starts

from zenyx_amd import _native as N
from zenyx_amd import kv
from zenyx_amd.train.cross_attention import CrossAttention

pytestmark = pytest.mark.gpu


@pytest.fixture
def dirty(monkeypatch):
    """Fresh memory holds NaN, workspaces too."""
    empty = torch.empty

    def filled(*a, **kw):
        t = empty(*a, **kw)
        return t.fill_(0xFF) if t.dtype == torch.uint8 else t.fill_(float("nan")) if t.is_floating_point() else t
    monkeypatch.setattr(torch, "empty", filled)


CASES = [  # rows, keys, Hq, Hkv, D, bound of the rows, of the keys
    ([5, 9], [70, 30], 4, 2, 64, 6, 40),
    ([5, 9, 3], [70, 30, 200], 3, 3, 128, 1, 1),
    ([2, 30], [5000, 40], 4, 1, 128, 7, 3001),     # keys cut among blocks
    ([1500], [1100], 2, 2, 128, 900, 700),         # rows cut in dk and dv
    ([40, 2], [600, 300], 2, 1, 64, 0, 500),       # none of the rows
    ([40, 2], [600, 300], 2, 1, 64, 500, 0),       # none of the keys
    ([700, 20, 90], [77, 10, 130], 8, 8, 64, 300, 64),
]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_beyond_the_bounds_are_zeros(dev, dirty, case, kind):
    rows, keys, Hq, Hkv, D, mq, mk = CASES[case]
    t, h, tiny = TYPES[kind]
    q, k, v, g = inputs(dev, t, rows, keys, Hq, Hkv, D, 40 + case)
    cu_q, cu_k = starts(rows, dev), starts(keys, dev)
    kept_q, kept_k = (torch.cat([torch.arange(n) < most for n in count]).to(dev) for count, most in ((rows, mq), (keys, mk)))
    few_q, few_k = [min(n, mq) for n in rows], [min(n, mk) for n in keys]
    want, tol = exact(q[kept_q], k[kept_k], v[kept_k], g[kept_q], few_q, few_k, h, tiny, D ** -0.5)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    bounds = dict(max_q_per_seq=mq, max_k_per_seq=mk)
    out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, return_lse=True, zero_rest=True, err=err, **bounds)
    assert int(err) == N.ZX_KERR_POS_RANGE
    grads = kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k, err=err, **bounds)
    for x, kept, w, e, name in zip((out, *grads), (kept_q, kept_q, kept_k, kept_k), want, tol, ("out", "dq", "dk", "dv")):
        assert (x[~kept] == 0).all(), name
        if kept.any():
            near(x[kept], w, e, name)
    # through autograd, where nobody sees the flag
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    y = CrossAttention()(*leaves, cu_q, cu_k, **bounds)
    assert torch.equal(y, out)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, g), grads))
    assert torch.equal(CrossAttention()(q, k, v, cu_q, cu_k, **bounds), out)


@pytest.mark.parametrize("D, scale", [(64, 1), (128, 1), (128, 40)])
def test_sequences_out_of_order_leave_nothing_unwritten(dev, dirty, D, scale):
    """Flagged, and every value is a number all the same (scale: longer ones, whose keys or rows are cut)."""
    rows, keys = [5 * scale, 9 * scale], [70 * scale, 30 * scale]
    q, k, v, g = inputs(dev, torch.bfloat16, rows, keys, 4, 2, D, 50)
    for cq, ck in (([0, 5, 15], [0, 70, 100]), ([-1, 5, 14], [0, 70, 100]), ([0, 5, 14], [0, 70, 101]), ([0, 9, 5], [0, 70, 100]),
                   ([0, 5, 14], [40, 20, 100]), ([0, 5, 14], [-9, 70, 100]), ([9, 3, 1], [0, 70, 100])):
        cu_q, cu_k = i32([scale * n for n in cq], dev), i32([scale * n for n in ck], dev)
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        bounds = dict(max_q_per_seq=14 * scale, max_k_per_seq=100 * scale, err=err)
        out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, return_lse=True, zero_rest=True, **bounds)
        assert int(err) == N.ZX_KERR_POS_RANGE
        # (log-sum-exp of rows that no call has computed is as good as any)
        lse = torch.where(lse.isnan(), 0.0, lse)
        for x in (out, *kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k, **bounds)):
            assert torch.isfinite(x).all(), (cq, ck)


def test_out_in_memory_that_inputs_have_parts_of(dev):
    """Disjoint parts of one arena are as good as tensors of their own; what overlaps q is refused."""
    q, k, v, _ = inputs(dev, torch.bfloat16, [40], [90], 2, 2, 64, 60)
    cu_q, cu_k = starts([40], dev), starts([90], dev)
    want = kv.cross_attention(q, k, v, cu_q, cu_k)
    arena = torch.cat([x.flatten() for x in (q, k, v)] + [torch.zeros(2 * q.numel(), dtype=q.dtype, device=dev)])
    at = [0, q.numel(), q.numel() + k.numel(), q.numel() + 2 * k.numel()]
    parts = [arena[a:a + x.numel()].view(x.shape) for a, x in zip(at, (q, k, v))]
    out = arena[at[3]:at[3] + q.numel()].view(q.shape)
    assert torch.equal(kv.cross_attention(*parts, cu_q, cu_k, out=out), want)
    assert torch.equal(parts[0], q)
    for shift in (8, q.numel() - 8):  # over the last rows of q, and of v
        with pytest.raises(ValueError, match="memory"):
            kv.cross_attention(*parts, cu_q, cu_k, out=arena[at[3] - shift:][:q.numel()].view(q.shape))
        with pytest.raises(ValueError, match="memory"):
            kv.cross_attention(parts[0], k, v, cu_q, cu_k, out=arena[shift:][:q.numel()].view(q.shape))
    # q's memory in another order
    wide = torch.zeros((40, 4, 64), dtype=q.dtype, device=dev)
    with pytest.raises(ValueError, match="memory"):
        kv.cross_attention(wide[:, :2], k, v, cu_q, cu_k, out=wide.flatten()[:q.numel()].view(q.shape))
    assert torch.equal(kv.cross_attention(parts[0], k, v, cu_q, cu_k, out=parts[0]), want)


def test_cross_attention_module_reports_bounds(dev):
    q, k, v, g = inputs(dev, torch.bfloat16, [5, 9], [70, 30], 4, 2, 64, 61)
    cu_q, cu_k = starts([5, 9], dev), starts([70, 30], dev)
    attend, leaf = CrossAttention(), q.clone().requires_grad_()
    for x in (q, leaf):
        assert attend(x, k, v, cu_q, cu_k, check=True).shape == q.shape
        with pytest.raises(ValueError, match="position"):
            attend(x, k, v, cu_q, cu_k, max_q_per_seq=6, max_k_per_seq=70, check=True)
        with pytest.raises(ValueError, match="err"):
            attend(x, k, v, cu_q, cu_k, err=torch.zeros(1, device=dev))
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    y = attend(leaf, k, v, cu_q, cu_k, max_q_per_seq=9, max_k_per_seq=69, err=err)
    assert int(err) == N.ZX_KERR_POS_RANGE
    err.zero_()
    y.backward(g)
    assert int(err) == N.ZX_KERR_POS_RANGE
    err.zero_()
    attend(leaf, k, v, cu_q, cu_k, max_q_per_seq=9, max_k_per_seq=70, err=err).backward(g)
    assert int(err) == 0
