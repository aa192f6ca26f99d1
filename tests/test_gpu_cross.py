"""GPU cross attention and its gradients against float64.

Tolerances, elementwise, each from the steps that round (h: half a step of the type relative to a
value, 2^-8 in bf16 and 2^-11 in fp16; fp16 has subnormal values, off by 2^-25 at most):

* scores: a sum of D products in fp32 and its scaling are off by at most (D + 4) 2^-24 sum|q k|, the
  exponential by 2^-22 of a weight, and log-sum-exp (of the same scores) by as much once more: a weight p
  by e p with e = 2 ((D + 4) 2^-24 |sm| sum|q k| + 2^-21 + (n / 64 + 64) 2^-24) over n keys;
* a weight is rounded to the type: h p more (fp16 holds it times 2^7: 2^-32 at least);
* out: sum of p |v| times that, and h of the value for the last rounding;
* dv: sum over rows of p |dO| times that;
* dS = p (dP - D): dP a sum of D products, off by D 2^-24 sum|dO v|; D_r = sum dO out from the rounded
  out, off by sum |dO| (out's error) + D 2^-24 sum|dO out|; rounded to the type: so
  |dS| (e + h) + p (those two) + 2^-25, and dq and dk the sums of that times |k| and |q|;
* sums over n rows or keys in fp32: n / 64 + 64 additions follow each other, 2^-24 of the sum of
  magnitudes each.
"""
import pytest
import torch

from zenyx_amd import _native as N
from zenyx_amd import kv
from zenyx_amd.train.cross_attention import CrossAttention

pytestmark = pytest.mark.gpu
TYPES = {"bf16": (torch.bfloat16, 2.0 ** -8, 0.0), "f16": (torch.float16, 2.0 ** -11, 2.0 ** -25)}


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def starts(counts, dev, first=0):
    return i32([first + sum(counts[:i]) for i in range(len(counts) + 1)], dev)


def exact(q, k, v, g, rows, keys, h, tiny, sm, k_at=None):
    """(out, dq, dk, dv) in float64 and their tolerances; rows and keys per sequence, packed; k_at: where a
    sequence's keys begin (default: packed)."""
    n_q, Hq, D = q.shape
    Hkv = k.shape[1]
    grp = Hq // Hkv
    zq, zk = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(k.shape, dtype=torch.float64, device=q.device)
    out, dq, dk, dv = zq.clone(), zq.clone(), zk.clone(), zk.clone()
    t_out, t_q, t_k, t_v = zq.clone(), zq.clone(), zk.clone(), zk.clone()
    a = c = 0
    f = 2.0 ** -24
    for b, (n, m) in enumerate(zip(rows, keys)):
        c = c if k_at is None else k_at[b]
        for i in range(Hq):
            if n == 0 or m == 0:
                break
            Q, K, V, G = q[a:a + n, i].double(), k[c:c + m, i // grp].double(), v[c:c + m, i // grp].double(), g[a:a + n, i].double()
            s = Q @ K.t() * sm
            p = torch.softmax(s, -1)
            size = (Q.abs() @ K.abs().t()) * abs(sm)
            e = 2 * ((D + 4) * f * size + 2.0 ** -21 + (m / 64 + 64) * f)
            e_p = p * (e + h) + (2.0 ** -32 if tiny else 0.0)
            o = p @ V
            out[a:a + n, i] = o
            t_o = e_p @ V.abs() + (m / 64 + 64) * f * (p @ V.abs()) + h * o.abs() + tiny
            t_out[a:a + n, i] = t_o
            dp = G @ V.t()
            delta = (G * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            e_dp = D * f * (G.abs() @ V.abs().t())
            e_delta = (G.abs() * t_o).sum(-1, keepdim=True) + D * f * (G * o).abs().sum(-1, keepdim=True)
            e_s = ds.abs() * (e + h) + p * (e_dp + e_delta) * (1 + e) + tiny
            more = 1 + (max(n * grp, m) / 64 + 64) * f
            dq[a:a + n, i] = sm * ds @ K
            t_q[a:a + n, i] = abs(sm) * (e_s @ K.abs() + (more - 1) * (ds.abs() @ K.abs()))
            dk[c:c + m, i // grp] += sm * ds.t() @ Q
            t_k[c:c + m, i // grp] += abs(sm) * (e_s.t() @ Q.abs() + (more - 1) * (ds.abs().t() @ Q.abs()))
            dv[c:c + m, i // grp] += p.t() @ G
            t_v[c:c + m, i // grp] += e_p.t() @ G.abs() + (more - 1) * (p.t() @ G.abs())
        a += n
        c += m
    for x, t in ((dq, t_q), (dk, t_k), (dv, t_v)):
        t += h * (x.abs() + t) + tiny + 1e-30
    return (out, dq, dk, dv), (t_out + 1e-30, t_q, t_k, t_v)


def near(got, want, tol, name):
    bad = (got.double() - want).abs() / tol
    assert torch.isfinite(got).all() and bad.max() <= 1, (name, float(bad.max()), int((bad > 1).sum()))


CASES = [  # rows, keys, Hq, Hkv, D
    ([1], [1], 1, 1, 64), ([1], [1], 2, 1, 128), ([3, 1], [2, 65], 2, 2, 64), ([64], [64], 1, 1, 128),
    ([33, 1, 100], [129, 64, 7], 4, 2, 64), ([0, 5, 17], [4, 0, 31], 3, 3, 128), ([1] * 9, [300] * 9, 8, 2, 64),
    ([1] * 5, [1500, 3, 64, 65, 700], 4, 4, 128), ([130, 257], [200, 77], 2, 2, 128), ([700], [77], 3, 3, 64),
    ([600, 20], [1000, 1300], 2, 1, 64), ([515], [640], 2, 1, 128), ([40], [3000], 8, 1, 128), ([5], [5000], 2, 2, 64),
    ([90, 3], [100, 50], 12, 4, 64), ([7, 9], [40, 33], 71, 71, 64), ([2000], [10], 1, 1, 64),
]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_float64(dev, case, kind):
    rows, keys, Hq, Hkv, D = CASES[case]
    t, h, tiny = TYPES[kind]
    gen = torch.Generator(device=dev).manual_seed(case)
    q = torch.randn((sum(rows), Hq, D), generator=gen, device=dev).to(t)
    kvp = torch.randn((sum(keys), 2, Hkv, D), generator=gen, device=dev).to(t)
    k, v = kvp[:, 0], kvp[:, 1]
    g = torch.randn(q.shape, generator=gen, device=dev).to(t)
    cu_q, cu_k = starts(rows, dev), starts(keys, dev)
    want, tol = exact(q, k, v, g, rows, keys, h, tiny, D ** -0.5)
    out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, return_lse=True, check=True)
    near(out, want[0], tol[0], "out")
    got = kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k, check=True)
    for x, w, e, name in zip(got, want[1:], tol[1:], ("dq", "dk", "dv")):
        near(x, w, e, name)
