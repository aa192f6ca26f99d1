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


def inputs(dev, t, rows, keys, Hq, Hkv, D, seed=0, width=1):
    """q, k, v, grad; width > 1: rows that lie in wider ones."""
    gen = torch.Generator(device=dev).manual_seed(seed)

    def make(n, H):
        x = torch.randn((n, H, D * width), generator=gen, device=dev).to(t)
        return x[..., D * (width - 1):]
    return make(sum(rows), Hq), make(sum(keys), Hkv), make(sum(keys), Hkv), make(sum(rows), Hq)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("sm", [-0.07, 0.0, 0.5])
@pytest.mark.parametrize("D, rows, keys", [(64, [70, 5], [90, 40]), (128, [4], [900])])
def test_other_scales(dev, kind, sm, D, rows, keys):
    t, h, tiny = TYPES[kind]
    q, k, v, g = inputs(dev, t, rows, keys, 4, 2, D, 1)
    cu_q, cu_k = starts(rows, dev), starts(keys, dev)
    want, tol = exact(q, k, v, g, rows, keys, h, tiny, sm)
    out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, sm_scale=sm, return_lse=True, check=True)
    near(out, want[0], tol[0], "out")
    for x, w, e, name in zip(kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k, sm_scale=sm), want[1:], tol[1:],
                             ("dq", "dk", "dv")):
        near(x, w, e, name)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D, Hq, Hkv", [(64, 6, 2), (128, 4, 4)])
def test_padded_states_and_rows_in_no_sequence(dev, kind, D, Hq, Hkv):
    """k_lens over padding that holds NaN and infinities; rows and keys before the first sequence and behind
    the last."""
    t, h, tiny = TYPES[kind]
    rows, lens, S = [9, 0, 200, 1, 33], [70, 12, 129, 0, 200], 200
    q, k, v, g = inputs(dev, t, [7 + sum(rows) + 600], [3 + S * 5 + 70], Hq, Hkv, D, 2)
    keep = torch.zeros(len(k), dtype=torch.bool, device=dev)
    at = [3 + S * b for b in range(5)]
    for a, n in zip(at, lens):
        keep[a:a + n] = True
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device=dev, dtype=t)
    k[~keep] = bad[torch.arange(int((~keep).sum()), device=dev) % 3][:, None, None]
    v[~keep] = bad[0]
    cu_q, cu_k, k_lens = starts(rows, dev, 7), i32([*at, 3 + S * 5], dev), i32(lens, dev)
    clean = [torch.where(keep[:, None, None], x, torch.zeros_like(x)) for x in (k, v)]
    mid = slice(7, 7 + sum(rows))
    want, tol = exact(q[mid], *clean, g[mid], rows, lens, h, tiny, D ** -0.5, at)
    out = torch.full_like(q, 5.0)
    got, lse = kv.cross_attention(q, k, v, cu_q, cu_k, k_lens, out=out, return_lse=True, check=True)
    assert got is out and (out[:7] == 5).all() and (out[7 + sum(rows):] == 5).all()
    near(out[mid], want[0], tol[0], "out")
    no_key = mid.start + sum(rows[:3])
    assert (out[no_key] == 0).all() and (lse[:, no_key] == -torch.inf).all()
    zero = kv.cross_attention(q, k, v, cu_q, cu_k, k_lens, zero_rest=True)
    assert torch.equal(zero[mid], out[mid]) and (zero[:7] == 0).all() and (zero[mid.stop:] == 0).all()
    # what rows in no sequence hold, and their gradients, reach nothing
    for x in (q, g):
        x[:7], x[mid.stop:] = float("nan"), float("inf")
    grads = kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k, k_lens, check=True)
    assert (grads[0][:7] == 0).all() and (grads[0][mid.stop:] == 0).all()
    near(grads[0][mid], want[1], tol[1], "dq")
    for x, w, e, name in zip(grads[1:], want[2:], tol[2:], ("dk", "dv")):
        near(x, w, e, name)
        assert (x[~keep] == 0).all()
    # gradients that overflowed do not reach the padding's either
    g[mid] = float("inf")
    for x in kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k, k_lens)[1:]:
        assert (x[~keep] == 0).all()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_lse_and_large_scores(dev, kind):
    """Scores of some hundreds, falling and rising along the keys: log-sum-exp to fp32's accuracy."""
    t = TYPES[kind][0]
    for rows, keys, D in (([40], [500], 64), ([3], [2000], 128)):
        q, k, v, _ = inputs(dev, t, rows, keys, 2, 1, D, 3)
        k *= torch.linspace(-9, 9, keys[0], device=dev, dtype=t)[:, None, None]
        q *= 4
        out, lse = kv.cross_attention(q, k, v, starts(rows, dev), starts(keys, dev), sm_scale=0.25, return_lse=True)
        s = torch.einsum("rhd,td->hrt", q.double(), k[:, 0].double()) * 0.25
        want = torch.logsumexp(s, -1) / torch.log(torch.tensor(2.0, dtype=torch.float64))
        size = torch.einsum("rhd,td->hrt", q.double().abs(), k[:, 0].double().abs()).amax(-1) * 0.25 * 1.4427
        assert ((lse - want).abs() <= size * (D + 4) * 2.0 ** -24 + want.abs() * 2.0 ** -23 + 1e-5).all()
        assert torch.isfinite(out).all()


def test_strided_inputs(dev):
    """The parts of fused projections, rows of wider ones, one KV head for all by a stride of 0, and rows so
    far apart that their offsets pass 2^32 bytes."""
    t, h, tiny = TYPES["bf16"]
    rows, keys, D = [33, 4], [80, 130], 64
    for Hq, Hkv, width in ((4, 4, 1), (8, 2, 3)):
        q, k, v, g = inputs(dev, t, rows, keys, Hq, Hkv, D, 4, width)
        flat = [x.contiguous() for x in (q, k, v, g)]
        cu_q, cu_k = starts(rows, dev), starts(keys, dev)
        want = kv.cross_attention(*flat[:3], cu_q, cu_k, return_lse=True)
        grads = kv.cross_attention_backward(flat[3], *flat[:3], *want, cu_q, cu_k)

        def same(q, k, v, g):
            got = kv.cross_attention(q, k, v, cu_q, cu_k, return_lse=True, check=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            got = kv.cross_attention_backward(g, q, k, v, *got, cu_q, cu_k, check=True)
            assert all(torch.equal(a, b) for a, b in zip(got, grads))
        same(q, k, v, g)
        head_major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in flat]
        same(*head_major)
        fused = torch.cat([flat[1], flat[2]], 1)
        same(q, fused[:, :Hkv], fused[:, Hkv:], g)
        fused = torch.empty((len(flat[1]), Hkv, 2 * D), dtype=t, device=dev)
        fused[..., :D], fused[..., D:] = flat[1], flat[2]
        same(q, fused[..., :D], fused[..., D:], g)
    one = flat[1][:, :1].expand(-1, 2, -1)
    got = kv.cross_attention(flat[0], one, one, cu_q, cu_k)
    assert torch.equal(got, kv.cross_attention(flat[0], one.contiguous(), one.contiguous(), cu_q, cu_k))
    far = torch.zeros((1100, 1 << 22), dtype=t, device=dev)  # 8.6 GiB
    rows = keys = [500, 600]
    q, k, v, g = inputs(dev, t, rows, keys, 2, 2, D, 5)
    cu = starts(rows, dev)
    out, lse = kv.cross_attention(q, k, v, cu, cu, return_lse=True)
    grads = kv.cross_attention_backward(g, q, k, v, out, lse, cu, cu)
    views = []
    for i, x in enumerate((q, k, v, g)):
        view = far[:, i * 2 * D:(i + 1) * 2 * D].unflatten(1, (2, D))
        view.copy_(x)
        views.append(view)
    a, b = kv.cross_attention(*views[:3], cu, cu, return_lse=True)
    assert torch.equal(a, out) and torch.equal(b, lse)
    for x, w in zip(kv.cross_attention_backward(views[3], *views[:3], a, b, cu, cu), grads):
        assert torch.equal(x, w)


def test_bounds_are_flagged(dev):
    t = torch.bfloat16
    rows, keys = [5, 9], [70, 30]
    q, k, v, g = inputs(dev, t, rows, keys, 4, 2, 64, 6)
    cu_q, cu_k = starts(rows, dev), starts(keys, dev)
    whole = kv.cross_attention(q, k, v, cu_q, cu_k)
    out = torch.full_like(q, 3.0)
    with pytest.raises(ValueError, match="position"):
        kv.cross_attention(q, k, v, cu_q, cu_k, max_q_per_seq=6, out=out, check=True)
    assert torch.equal(out[:11], whole[:11]) and (out[11:] == 3).all()
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    got, lse = kv.cross_attention(q, k, v, cu_q, cu_k, max_k_per_seq=40, return_lse=True, err=err)
    assert int(err) == N.ZX_KERR_POS_RANGE
    assert torch.equal(got, kv.cross_attention(q, k, v, cu_q, cu_k, i32([40, 30], dev)))
    for cq, ck in (([0, 5, 15], [0, 70, 100]), ([-1, 5, 14], [0, 70, 100]), ([0, 5, 14], [0, 70, 101]), ([0, 9, 5], [0, 70, 100]),
                   ([0, 5, 14], [40, 20, 100]), ([0, 5, 14], [-9, 70, 100]), ([0, 1 << 30, 14], [0, 1 << 30, 100])):
        for f in (lambda: kv.cross_attention(q, k, v, i32(cq, dev), i32(ck, dev), max_q_per_seq=14, max_k_per_seq=100,
                                             check=True),
                  lambda: kv.cross_attention_backward(g, q, k, v, got, lse, i32(cq, dev), i32(ck, dev), max_q_per_seq=14,
                                                      max_k_per_seq=100, check=True)):
            with pytest.raises(ValueError, match="position"):
                f()
    # k_lens beyond a sequence's keys and below 0: all of them, none
    got = kv.cross_attention(q, k, v, cu_q, cu_k, i32([1 << 30, -4], dev), check=True)
    assert torch.equal(got[:5], whole[:5]) and (got[5:] == 0).all()


@pytest.mark.parametrize("D, rows, keys, Hq, Hkv", [(64, [300, 40], [500, 900], 4, 2), (128, [2, 3], [5000, 40], 4, 1),
                                                    (128, [1500], [1100], 2, 2)])
def test_captured_and_repeated(dev, D, rows, keys, Hq, Hkv):
    """The same bits from call to call; a captured forward and backward on other inputs and lengths, with
    eager work between the replays; two streams at once."""
    q, k, v, g = inputs(dev, torch.bfloat16, rows, keys, Hq, Hkv, D, 7)
    cu_q, cu_k, k_lens = starts(rows, dev), starts(keys, dev), i32(keys, dev)
    mq, mk = max(rows), max(keys)

    def step():
        out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, k_lens, max_q_per_seq=mq, max_k_per_seq=mk, return_lse=True,
                                      zero_rest=True)
        return (out, *kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k, k_lens, max_q_per_seq=mq,
                                                  max_k_per_seq=mk))
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(), first))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        q.mul_(-1.0), g.mul_(0.5 if i % 2 else 2.0)
        cut = [max(0, n - 37 * i) for n in keys]
        k_lens.copy_(i32(cut, dev))
        cu_q.copy_(starts([max(0, n - i) for n in rows], dev))
        for x in held:
            x.fill_(9.0)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))
    torch.cuda.synchronize()
    want, got = step(), []
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x in got for a, b in zip(x, want))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_gradients_against_differences(dev, kind):
    """<dq, x> and the like against the forward's own central difference along x.  The step e is exact in
    the type for the direction's values of +-1 and inputs on a grid of 1/8 below 4; the forward is off by
    tol per element at each end, the difference by 2 |g| tol / 2 e, its third-order term by
    (e^2 / 6) |f'''|, which halving e would show: the bound takes a quarter of f(2e)'s difference from f(e)'s."""
    t, h, tiny = TYPES[kind]
    rows, keys, D = [6, 3], [20, 9], 64
    gen = torch.Generator(device=dev).manual_seed(8)
    q, k, v, g = (torch.randint(-8, 9, (n, H, D), generator=gen, device=dev).to(t) / 8
                  for n, H in ((9, 4), (29, 2), (29, 2), (9, 4)))
    cu_q, cu_k = starts(rows, dev), starts(keys, dev)

    def f(q, k, v):
        out = kv.cross_attention(q, k, v, cu_q, cu_k)
        _, tol = exact(q, k, v, g, rows, keys, h, tiny, D ** -0.5)
        return (out.double() * g.double()).sum(), (tol[0] * g.double().abs()).sum()
    out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, return_lse=True)
    grads = kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k)
    _, tol = exact(q, k, v, g, rows, keys, h, tiny, D ** -0.5)
    xs = [q, k, v]
    for i in range(3):
        for trial in range(3):
            way = torch.randint(0, 2, xs[i].shape, generator=gen, device=dev).to(t) * 2 - 1
            diff, noise = [], []
            for e in (0.125, 0.25):
                (hi, n1), (lo, n2) = (f(*[x + s * e * way if j == i else x for j, x in enumerate(xs)]) for s in (1, -1))
                diff.append((hi - lo) / (2 * e))
                noise.append((n1 + n2) / (2 * e))
            got = (grads[i].double() * way.double()).sum()
            bound = noise[0] + noise[1] + (tol[i + 1] * 1.0).sum() + (diff[1] - diff[0]).abs()
            assert (got - diff[0]).abs() <= bound, (i, trial, float(got), float(diff[0]), float(bound))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_cross_attention_module(dev, kind):
    """Through autograd: leaves that are views and broadcast, gradients as autograd lays them out, inputs
    that need none, no grad, other bounds; and what it refuses."""
    t, h, tiny = TYPES[kind]
    rows, keys, D = [20, 1, 50], [64, 7, 300], 64
    q, k, v, g = inputs(dev, t, rows, keys, 4, 2, D, 9)
    cu_q, cu_k = starts(rows, dev), starts(keys, dev)
    attend = CrossAttention()
    out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, return_lse=True)
    want = kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k)
    fused = torch.stack([k, v], 1).requires_grad_()  # [n, 2, H, D]
    ql = q.clone().requires_grad_()
    y = attend(ql, fused[:, 0], fused[:, 1], cu_q, cu_k)
    assert torch.equal(y, out)
    y.backward(g)
    assert torch.equal(ql.grad, want[0]) and torch.equal(fused.grad, torch.stack(want[1:], 1))
    # gradients that are expanded, transposed or not aligned
    for give in (torch.ones((), dtype=t, device=dev).expand(q.shape), g.transpose(0, 2).contiguous().transpose(0, 2),
                 torch.empty(g.numel() + 1, dtype=t, device=dev)[1:].view(g.shape).copy_(g)):
        ql.grad = None
        attend(ql, k, v, cu_q, cu_k).backward(give)
        assert torch.equal(ql.grad, kv.cross_attention_backward(give.contiguous().clone(), q, k, v, out, lse, cu_q, cu_k)[0])
    # one head's states for both: their gradients come together, in the type
    one = k[:, :1].clone().requires_grad_()
    attend(q, one.expand(-1, 2, -1), v, cu_q, cu_k).backward(g)
    both = one.detach().expand(-1, 2, -1).contiguous()
    o1, l1 = kv.cross_attention(q, both, v, cu_q, cu_k, return_lse=True)
    assert torch.equal(one.grad, kv.cross_attention_backward(g, q, both, v, o1, l1, cu_q, cu_k)[1].sum(1, keepdim=True))
    with torch.no_grad():
        z = attend(ql, k, v, cu_q, cu_k)
    assert not z.requires_grad and torch.equal(z, out)
    assert not attend(q, k, v, cu_q, cu_k).requires_grad
    y = attend(ql, k, v, cu_q, cu_k, max_q_per_seq=71, max_k_per_seq=371)
    (d,) = torch.autograd.grad(y, ql, g, create_graph=True)
    with pytest.raises(RuntimeError):  # once, in reverse mode
        torch.autograd.grad(d.float().sum(), ql)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            attend(torch.autograd.forward_ad.make_dual(q, torch.ones_like(q)), k, v, cu_q, cu_k)
    for bad in ((q.float(), k, v), (q, k[:, :, :32], v), (q[:, :3], k, v), (q, k[:5], v), (q, k.cpu(), v), (q, k, v.half().bfloat16() if
                kind == "f16" else v.half()), (q[..., ::2], k, v), (q[0], k, v)):
        with pytest.raises(ValueError):
            attend(*bad, cu_q, cu_k)
    for cq, ck, kl in ((cu_q.long(), cu_k, None), (cu_q, cu_k[:3], None), (cu_q, cu_k, cu_k), (cu_q[:1], cu_k[:1], None),
                       (cu_q, cu_k, cu_k[:3].long()), (cu_q.cpu(), cu_k, None)):
        with pytest.raises(ValueError):
            attend(q, k, v, cq, ck, kl)
    for kw in (dict(out=q.float()), dict(out=q[:3]), dict(out=q.transpose(0, 1)), dict(err=torch.zeros(1, device=dev))):
        with pytest.raises(ValueError):
            kv.cross_attention(q, k, v, cu_q, cu_k, **kw)
    for i, x in ((0, g.float()), (0, g[:3]), (4, out.float()), (5, lse.double()), (5, lse[:1]), (0, g.cpu())):
        args = [g, q, k, v, out, lse]
        args[i] = x
        with pytest.raises(ValueError):
            kv.cross_attention_backward(*args, cu_q, cu_k)


def test_captured_training_step(dev):
    """Forward and backward through autograd in one graph, replayed with other inputs."""
    rows, keys, D = [64, 30], [200, 77], 128
    q, k, v, g = inputs(dev, torch.bfloat16, rows, keys, 4, 2, D, 10)
    cu_q, cu_k = starts(rows, dev), starts(keys, dev)
    for x in (q, k, v):
        x.requires_grad_()
    attend = CrossAttention()

    def step():
        out = attend(q, k, v, cu_q, cu_k, max_q_per_seq=64, max_k_per_seq=200)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), g))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        with torch.no_grad():
            q.mul_(0.5 if i else -1.0), v.add_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_no_rows_no_keys(dev):
    for n, m in ((0, 5), (5, 0), (0, 0)):
        q = torch.randn((n, 4, 64), device=dev).bfloat16().requires_grad_()
        k = torch.randn((m, 2, 64), device=dev).bfloat16().requires_grad_()
        y = CrossAttention()(q, k, k, i32([0, n], dev), i32([0, m], dev))
        assert y.shape == q.shape and (y == 0).all()
        y.backward(torch.ones_like(y))
        assert (q.grad == 0).all() and (k.grad == 0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows, keys", [([40, 9], [1, 1]), ([3], [100])])
def test_one_key_has_no_gradient(dev, D, rows, keys):
    """Where all of a row's weight is on one key (the others, if any, at scores 40 below in log2), dS is
    p (dP - p dP): p is 1 within 2^-20 (scores and log-sum-exp as the tolerances above), nothing else rounds."""
    q, k, v, g = inputs(dev, torch.bfloat16, rows, keys, 2, 2, D, 11)
    q, k = q.abs(), k.abs()
    if keys[0] > 1:
        k[1:] = 0
        k[0] = 8
        q = torch.ones_like(q) * 4
    cu_q, cu_k = starts(rows, dev), starts(keys, dev)
    out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, return_lse=True)
    dq, dk, _ = kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k)
    most = float((g.double().abs().sum(-1).max() * v.abs().max()))  # |dP|
    size = float((q.double().abs().sum(-1).max() * k.abs().max())) * D ** -0.5
    off = most * 2 * (2 * (D + 4) * 2.0 ** -24 * size + 2.0 ** -20)
    assert dq.abs().max() <= off * float(k.abs().max()) * D ** -0.5 * sum(keys)
    assert dk.abs().max() <= off * float(q.abs().max()) * D ** -0.5 * sum(rows)


def test_out_in_place(dev):
    """out may be q itself (a block reads its rows before it writes them), but not lie in k or v."""
    for rows, keys in (([300, 40], [500, 900]), ([2, 3], [5000, 40])):
        q, k, v, _ = inputs(dev, torch.bfloat16, rows, keys, 4, 2, 64, 12)
        cu_q, cu_k = starts(rows, dev), starts(keys, dev)
        want = kv.cross_attention(q, k, v, cu_q, cu_k)
        assert torch.equal(kv.cross_attention(q, k, v, cu_q, cu_k, out=q), want)
    both = torch.zeros((2, 10, 2, 64), dtype=torch.bfloat16, device=dev)
    cu = starts([10], dev)
    with pytest.raises(ValueError, match="memory"):
        kv.cross_attention(both[0].clone(), both[0], both[1], cu, cu, out=both[0])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("D, Hq, Hkv", [(64, 3, 1), (128, 2, 2)])
def test_around_the_tiles_ends(dev, kind, D, Hq, Hkv):
    """Keys around one and two tiles, by themselves and as the first ones of longer padded states; rows
    around a wave's and a block's columns."""
    t, h, tiny = TYPES[kind]
    lens = [63, 64, 65, 127, 128, 129, 1, 0, 192]
    rows = [31, 32, 33, 127, 128, 129, 2, 5, 1]
    q, k, v, g = inputs(dev, t, rows, lens, Hq, Hkv, D, 13)
    cu_q, cu_k = starts(rows, dev), starts(lens, dev)
    want, tol = exact(q, k, v, g, rows, lens, h, tiny, D ** -0.5)
    out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, return_lse=True, check=True)
    near(out, want[0], tol[0], "out")
    grads = kv.cross_attention_backward(g, q, k, v, out, lse, cu_q, cu_k, check=True)
    for x, w, e, name in zip(grads, want[1:], tol[1:], ("dq", "dk", "dv")):
        near(x, w, e, name)
    S = 200
    pk, pv = (torch.full((S * len(lens), Hkv, D), float("nan"), dtype=t, device=dev) for _ in range(2))
    at = 0
    for b, n in enumerate(lens):
        pk[b * S:b * S + n], pv[b * S:b * S + n] = k[at:at + n], v[at:at + n]
        at += n
    cu_p, k_lens = starts([S] * len(lens), dev), i32(lens, dev)
    o, e = kv.cross_attention(q, pk, pv, cu_q, cu_p, k_lens, return_lse=True, check=True)
    near(o, want[0], tol[0], "padded out")
    dq, dk, dv = kv.cross_attention_backward(g, q, pk, pv, o, e, cu_q, cu_p, k_lens, check=True)
    near(dq, want[1], tol[1], "padded dq")
    at = 0
    for b, n in enumerate(lens):
        near(dk[b * S:b * S + n], want[2][at:at + n], tol[2][at:at + n], "padded dk") if n else None
        near(dv[b * S:b * S + n], want[3][at:at + n], tol[3][at:at + n], "padded dv") if n else None
        assert (dk[b * S + n:(b + 1) * S] == 0).all() and (dv[b * S + n:(b + 1) * S] == 0).all()
        at += n
