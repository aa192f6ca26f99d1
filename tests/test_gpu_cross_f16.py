"""GPU gradients of cross attention in fp16 over its range: small gradients, whose scores' gradients would
be subnormal in fp16, and ones whose scores' gradients are above its largest value.

dS is rounded to fp16 times a power of two that brings the largest of a row's (for dk: of a key's) so far to
2^7 or more, so a value is off by 2^-11 of itself or 2^-25 / 2^7 of the largest, whatever the gradient's size."""
import math

import pytest
import torch

from test_gpu_cross import inputs, starts

from zenyx_amd import kv

pytestmark = pytest.mark.gpu
H = 2.0 ** -11
F = 2.0 ** -24
TINY = 2.0 ** -25

SHAPES = [  # rows, keys, Hq, Hkv, D
    ([30, 5], [1500, 700], 2, 2, 64), ([9], [8000], 4, 2, 64), ([40], [1500], 2, 1, 128), ([200, 33], [77, 128], 2, 2, 64),
    ([700], [600], 2, 1, 128), ([3], [5000], 2, 2, 128),
]


def grads_of(q, k, v, g, rows, keys, sm=None):
    cu_q, cu_k = starts(rows, q.device), starts(keys, q.device)
    out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, sm_scale=sm, return_lse=True, check=True)
    return kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k, sm_scale=sm, check=True)


def exact(q, k, v, g, rows, keys):
    """(dq, dk, dv) in float64 and their tolerances (test_gpu_cross.py's, dS as above)."""
    n_q, Hq, D = q.shape
    grp, sm = Hq // k.shape[1], D ** -0.5
    dq, t_q = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    dk, dv, t_k, t_v = (torch.zeros(k.shape, dtype=torch.float64, device=q.device) for _ in range(4))
    a = c = 0
    for n, m in zip(rows, keys):
        for j in range(k.shape[1]):
            K, V = k[c:c + m, j].double(), v[c:c + m, j].double()
            parts = []
            for i in range(j * grp, (j + 1) * grp):
                Q, G = q[a:a + n, i].double(), g[a:a + n, i].double()
                p = torch.softmax(Q @ K.t() * sm, -1)
                e = 2 * ((D + 4) * F * (Q.abs() @ K.abs().t()) * sm + 2.0 ** -21 + (m / 64 + 64) * F)
                e_p = p * (e + H) + 2.0 ** -32
                o = p @ V
                t_o = e_p @ V.abs() + (m / 64 + 64) * F * (p @ V.abs()) + H * o.abs() + TINY
                dp = G @ V.t()
                ds = p * (dp - (G * o).sum(-1, keepdim=True))
                e_delta = (G.abs() * t_o).sum(-1, keepdim=True) + D * F * (G * o).abs().sum(-1, keepdim=True)
                e_s = ds.abs() * (e + H) + p * (D * F * (G.abs() @ V.abs().t()) + e_delta) * (1 + e)
                more = (max(n * grp, m) / 64 + 64) * F
                dq[a:a + n, i] = sm * ds @ K
                t_q[a:a + n, i] = sm * ((e_s + 2.0 ** -32 * ds.abs().amax(-1, keepdim=True) + more * ds.abs()) @ K.abs())
                parts.append((ds, e_s + more * ds.abs(), Q))
                dv[c:c + m, j] += p.t() @ G
                t_v[c:c + m, j] += e_p.t() @ G.abs() + more * (p.t() @ G.abs())
            most = torch.stack([ds.abs().amax(0) for ds, _, _ in parts]).amax(0)  # of a key's, over the group's heads
            for ds, e_s, Q in parts:
                dk[c:c + m, j] += sm * ds.t() @ Q
                t_k[c:c + m, j] += sm * ((e_s + 2.0 ** -32 * most).t() @ Q.abs())
        a += n
        c += m
    for x, t in ((dq, t_q), (dk, t_k), (dv, t_v)):
        t += H * (x.abs() + t) + TINY
    return (dq, dk, dv), (t_q, t_k, t_v)


def factor(shape, which, size):
    """A power of two for the keys (and one over it for the queries), or the reverse, that brings dq's (dk's)
    values near 2^-6 or above: dP is about sqrt(D) size, a weight 1 / keys, and D^-1/2 is the scale."""
    rows, keys, Hq, Hkv, _ = SHAPES[shape]
    about = size / max(keys) ** 0.5 if which == 0 else size * (max(rows) * Hq // Hkv) ** 0.5 / max(keys)
    return 2.0 ** min(12, max(0, math.ceil(math.log2(2.0 ** -6 / about))))


def scaled(dev, shape, which, size, seed):
    rows, keys, Hq, Hkv, D = SHAPES[shape]
    q, k, v, g = inputs(dev, torch.float16, rows, keys, Hq, Hkv, D, seed)
    by = factor(shape, which, size) ** (-1 if which == 0 else 1)
    return q * by, k / by, v, g


@pytest.mark.parametrize("size", [1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_small_gradients_keep_their_bits(dev, shape, size):
    """Beside the tolerance: dS and the result are each rounded once, by errors whose root mean square is
    2^-11 / sqrt 3 of the value at most and which do not know each other: 2^-11 sqrt(2/3) in all, and not
    more than 2^-11 with what fp32 adds."""
    rows, keys, _, _, _ = SHAPES[shape]
    for which in (0, 1):
        q, k, v, g = scaled(dev, shape, which, size, 60 + shape)
        g = (g.float() * size).half()
        got = grads_of(q, k, v, g, rows, keys)
        want, tol = exact(q, k, v, g, rows, keys)
        for x, w, e in zip(got, want, tol):
            bad = (x.double() - w).abs() / e
            assert torch.isfinite(x).all() and bad.max() <= 1, (which, float(bad.max()))
        normal = want[which].abs() > 2.0 ** -14  # (below it fp16 has no relative accuracy)
        if normal.sum() < 1000:
            continue
        x, w = got[which].double()[normal], want[which][normal]
        off = float(((x - w).square().sum() / w.square().sum()).sqrt())
        assert off <= H, (which, off / H)


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_gradients_are_linear_in_the_outputs(dev, shape):
    """Output gradients times a power of two give dq and dk the same bits at that power, where both are normal
    numbers (dv, whose weights do not depend on the gradient, always had them)."""
    rows, keys, _, _, _ = SHAPES[shape]
    for which in (0, 1):
        q, k, v, g = scaled(dev, shape, which, 2.0 ** -10, 70 + shape)
        g = torch.where(g.abs() < 2.0 ** -4, torch.full_like(g, 0.25), g)  # normal numbers at 2^-10 too
        want = grads_of(q, k, v, g, rows, keys)[which]
        for power in (-10, -5, 4):
            got = grads_of(q, k, v, g * 2.0 ** power, rows, keys)[which]
            there = want.double() * 2.0 ** power
            normal = (want.abs() >= 2.0 ** -14) & (there.abs() >= 2.0 ** -14) & (there.abs() < 65504)
            assert normal.double().mean() > 0.5
            assert torch.equal(got.double()[normal], there[normal]), (which, power)


@pytest.mark.parametrize("rows, keys, D", [([5], [4], 64), ([40, 3], [4, 200], 64), ([33], [130], 128)])
def test_large_gradients_of_scores(dev, rows, keys, D):
    """Scores' gradients above fp16's largest value, whose dq and dk are within its range."""
    q, k, v, g = inputs(dev, torch.float16, rows, keys, 2, 2, D, 80)
    q, k, v, g = q / 1024, k / 1024, v * 1024, g * 2048
    got = grads_of(q, k, v, g, rows, keys)
    want, tol = exact(q, k, v, g, rows, keys)
    # (scores are near zero: a weight is 1 / keys)
    assert float((g[:rows[0], 0].double() @ v[:keys[0], 0].double().t()).abs().max()) / keys[0] > 2 * 65504
    for x, w, e in zip(got, want, tol):
        assert w.abs().max() < 60000 and torch.isfinite(x).all() and ((x.double() - w).abs() <= e).all()


def test_gradients_that_grow_along_the_sequence(dev):
    """Rows (for dk) and keys (for dq) whose scores' gradients rise, or fall, by 2^16 and more from first to
    last: the factor follows, and what was summed before keeps its place."""
    rows, keys, D = [300], [300], 64
    for way in (1, -1):
        q, k, v, g = inputs(dev, torch.float16, rows, keys, 2, 1, D, 90)
        ramp = torch.linspace(-12, 12, 300, device=dev) * way
        ramp = torch.exp2(ramp.round())
        g = (g.float() * ramp.clamp(max=2.0 ** 9)[:, None, None]).half()
        v = (v.float() * ramp.clamp(max=2.0 ** 4)[:, None, None]).half()
        q, k = q / 8, k / 8
        got = grads_of(q, k, v, g, rows, keys)
        want, tol = exact(q, k, v, g, rows, keys)
        for x, w, e in zip(got, want, tol):
            fits = w.abs() < 65000
            assert fits.any() and ((x.double() - w).abs() <= e)[fits].all()


def test_gradients_with_infinities_and_nan(dev):
    """An output gradient that overflowed or is NaN makes its own row's dq and every key's dk not finite, and
    the other rows' dq as they were."""
    rows, keys, D = [70], [150], 64
    q, k, v, g = inputs(dev, torch.float16, rows, keys, 2, 2, D, 95)
    want = grads_of(q, k, v, g, rows, keys)
    for bad in (float("inf"), float("nan")):
        x = g.clone()
        x[33, 1, 7] = bad
        dq, dk, _ = grads_of(q, k, v, x, rows, keys)
        assert not torch.isfinite(dq[33, 1]).any() and not torch.isfinite(dk[:, 1]).any()
        dq[33, 1] = want[0][33, 1]
        assert torch.equal(dq, want[0]) and torch.equal(dk[:, 0], want[1][:, 0])
