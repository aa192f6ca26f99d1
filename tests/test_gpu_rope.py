"""GPU rotary positions (zx_rope, zx_rope_table) and the FP8 append that rotates the keys
(zx_kv_rope_append).

The rotation is fixed to the bit: both products and their sum are rounded to float32, then the
result once to the tensor's type, so kernels are compared with a numpy evaluation in float32
exactly, and with float64 within what those roundings allow: 3 roundings of 2^-24 of the
products' magnitudes, and half a step (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) of the result (fp16:
2^-25 absolute below its normal range).  The append is compared to the bit with the rotation
followed by the append that takes rotated keys."""
import warnings

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from oracle import kv4 as R
from zenyx_amd import _native as N
from zenyx_amd import kv
from zenyx_amd.train.rotary import RotaryPositions, rotary_frequencies

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def table64(n_pos, rot, dev, base=10000.0, scale=1.0):
    f = rotary_frequencies(rot, base)[0]
    return kv.rope_table(f.to(dev), n_pos, scale)


def rows(x, table, positions, interleaved, transpose=False):
    """numpy float32 [n, H, D]: the rotation before its last rounding."""
    t = table.cpu().numpy()[positions.cpu().numpy()]
    h = t.shape[1] // 2
    s = t[:, h:]
    return R.rotate_f32(x.float().cpu().numpy(), t[:, :h], -s if transpose else s, interleaved)


def same_bits(a: torch.Tensor, b: torch.Tensor) -> bool:
    i = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.contiguous().view(i), b.contiguous().view(i))


@pytest.mark.parametrize("rot, n_pos, scale", [(128, 131072, 1.0), (16, 3, 1.25), (64, 1, 1.0)])
def test_table(dev, rot, n_pos, scale):
    """cos / sin of 64-bit angles, rounded once: within half a step of float32 of the value plus
    what 64 bits leave open (2^-50), also at the far end, where an angle in float32 would be
    2^-8 off."""
    freq = rotary_frequencies(rot)[0]
    t = table64(n_pos, rot, dev, scale=scale).cpu().double().numpy()
    at = np.unique(np.concatenate([np.arange(min(n_pos, 500)), np.arange(max(0, n_pos - 500), n_pos)]))
    angle = at[:, None].astype(np.float64) * freq.numpy()
    want = np.concatenate([np.cos(angle), np.sin(angle)], 1) * scale
    assert np.all(np.abs(t[at] - want) <= np.abs(want) * 2.0 ** -24 + 2.0 ** -36)  # an angle of 2^17 has 2^-36


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n, H, D, rot", [(1, 1, 16, 16), (5, 3, 64, 64), (1000, 32, 128, 128), (77, 71, 72, 48),
                                          (33, 8, 256, 64), (300, 12, 64, 32), (2, 1, 128, 128), (9000, 8, 128, 96),
                                          (13, 5, 88, 80)])
def test_rotation_bits(dev, dtype, interleaved, n, H, D, rot):
    g = torch.Generator().manual_seed(n * H + D)
    x = torch.randn((n, H, D), generator=g).to(dtype).to(dev)
    positions = torch.randint(0, 5000, (n,), generator=g, dtype=torch.int32).to(dev)
    table = table64(5000, rot, dev)
    for transpose in (False, True):
        got = kv.rope(x, table, positions, interleaved=interleaved, transpose=transpose)
        want32 = rows(x, table, positions, interleaved, transpose)
        assert same_bits(got, torch.from_numpy(want32).to(dtype).to(dev))
        # against 64 bits
        t = table.cpu().numpy()[positions.cpu().numpy()].astype(np.float64)
        c, s = t[:, None, :rot // 2], t[:, None, rot // 2:] * (-1 if transpose else 1)
        x64 = x.double().cpu().numpy()
        a = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
        b = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
        want, mag = x64.copy(), np.abs(x64)
        want[..., a], want[..., b] = x64[..., a] * c - x64[..., b] * s, x64[..., b] * c + x64[..., a] * s
        mag[..., a] = np.abs(x64[..., a] * c) + np.abs(x64[..., b] * s)
        mag[..., b] = np.abs(x64[..., b] * c) + np.abs(x64[..., a] * s)
        e32 = 3 * 2.0 ** -24 * mag
        tol = e32 + HALF_STEP[dtype] * (np.abs(want) + e32) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol)


def test_views_and_in_place(dev):
    """The queries of a fused projection are turned where they lie; nothing else changes."""
    n, Hq, Hkv, D = 50, 4, 2, 64
    qkv = torch.randn((n, Hq + 2 * Hkv, D), device=dev).to(torch.bfloat16)
    before = qkv.clone()
    table, positions = table64(100, D, dev), torch.arange(n, dtype=torch.int32, device=dev)
    q = qkv[:, :Hq]
    want = kv.rope(q.contiguous(), table, positions)
    fresh = kv.rope(q, table, positions)  # a strided input
    assert same_bits(fresh, want) and torch.equal(qkv, before)
    assert kv.rope(q, table, positions, out=q) is q
    assert same_bits(q, want) and torch.equal(qkv[:, Hq:], before[:, Hq:])
    # heads last: [H, n, D] seen as [n, H, D], into a part of a larger output
    y = torch.randn((Hq, n, D), device=dev)
    room = torch.full((n, 2 * Hq, D), 7.0, device=dev)
    out = room[:, Hq:]
    kv.rope(y.transpose(0, 1), table, positions, interleaved=True, out=out)
    assert same_bits(out, kv.rope(y.transpose(0, 1).contiguous(), table, positions, interleaved=True))
    assert torch.all(room[:, :Hq] == 7)
    # one head broadcast to several: the input may be a stride-0 view
    one = torch.randn((n, 1, D), device=dev)
    assert same_bits(kv.rope(one.expand(n, 3, D), table, positions),
                     kv.rope(one, table, positions).expand(n, 3, D).contiguous())


def test_partial_in_place_leaves_the_rest(dev):
    x = torch.randn((7, 3, 128), device=dev)
    table, positions = table64(64, 32, dev), torch.randint(0, 64, (7,), dtype=torch.int32, device=dev)
    want = kv.rope(x, table, positions)
    rest = x[..., 32:].clone()
    kv.rope(x, table, positions, out=x)
    assert same_bits(x, want) and same_bits(x[..., 32:], rest)


@pytest.mark.parametrize("in_place", [False, True])
def test_positions_that_the_table_does_not_have(dev, in_place):
    x = torch.randn((6, 2, 64), device=dev).to(torch.float16)
    table = table64(10, 32, dev)
    positions = torch.tensor([0, -1, 9, 10, 2 ** 31 - 1, 5], dtype=torch.int32, device=dev)
    good = torch.tensor([True, False, True, False, False, True], device=dev)
    want = kv.rope(x, table, positions.clamp(0, 9))
    want[~good] = x[~good]
    y = x.clone()
    got = kv.rope(y, table, positions, out=y if in_place else None)
    assert same_bits(got, want)
    with pytest.raises(ValueError, match="position"):
        kv.rope(x, table, positions, check=True)
    kv.rope(x[good], table, positions[good], check=True)


def test_non_finite_values_stay_in_their_pair(dev):
    x = torch.ones((1, 1, 64), device=dev)
    x[0, 0, 3], x[0, 0, 20] = float("nan"), float("inf")
    y = kv.rope(x, table64(8, 64, dev), torch.tensor([5], dtype=torch.int32, device=dev))
    bad = ~torch.isfinite(y[0, 0])
    assert torch.nonzero(bad).flatten().tolist() == [3, 20, 35, 52]


def test_refusals(dev):
    table, p = table64(16, 64, dev), torch.zeros(4, dtype=torch.int32, device=dev)
    x = torch.zeros((4, 2, 64), device=dev)
    for bad in (lambda: kv.rope(x.double(), table, p), lambda: kv.rope(x[0], table, p),
                lambda: kv.rope(x, table.half(), p), lambda: kv.rope(x, table, p.long()),
                lambda: kv.rope(x, table, p[:3]), lambda: kv.rope(x[..., :32], table, p),
                lambda: kv.rope(x.transpose(1, 2), table[:, :16].contiguous(), p),
                lambda: kv.rope(torch.zeros((4, 2, 66), device=dev)[..., 1:65], table, p),
                lambda: kv.rope(x.cpu(), table, p), lambda: kv.rope(x, table.cpu(), p),
                lambda: kv.rope(x, table, p, out=torch.zeros((4, 2, 64), device=dev, dtype=torch.float16)),
                lambda: kv.rope(x, table, p, out=torch.zeros((4, 1, 64), device=dev).expand(4, 2, 64)),
                lambda: kv.rope(torch.zeros((4, 2, 100), device=dev), table, p),  # 100 channels
                lambda: kv.rope(torch.zeros((4, 2, 72), device=dev), torch.zeros((3, 24), device=dev), p),
                lambda: RotaryPositions(64, 16, rotary_dim=24), lambda: RotaryPositions(64, 0),
                lambda: RotaryPositions(64, 16, rotary_dim=80),
                lambda: RotaryPositions(64, 16, scaling={"type": "other", "factor": 2}),
                lambda: RotaryPositions(64, 16, scaling={"type": "yarn", "factor": 2}),
                lambda: kv.rope_table(torch.ones(4, device=dev), 3)):
        with pytest.raises(ValueError):
            bad()
    big = torch.zeros((8, 2, 64), device=dev)
    with pytest.raises(ValueError, match="overlap"):  # a shifted view of the same memory
        kv.rope(big[:4], table, p, out=big[2:6])
    assert kv.rope(x[:0], table, p[:0]).shape == (0, 2, 64)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scaling", [None, {"type": "yarn", "factor": 4, "original_positions": 32}])
def test_gradient(dev, interleaved, scaling):
    """The gradient is the transposed rotation: against the formula's matrix and differences."""
    rope = RotaryPositions(32, 200, rotary_dim=16, interleaved=interleaved, scaling=scaling)
    n, H, D = 6, 3, 32
    x = torch.randn((n, H, D), device=dev, requires_grad=True)
    p = torch.randint(0, 200, (n,), dtype=torch.int32, device=dev)
    g = torch.randn((n, H, D), device=dev)
    rope(x, p).backward(g)
    t = rope.table.double()[p.long()]
    want = torch.zeros((n, H, D), dtype=torch.float64, device=dev)
    for i in range(n):  # rows of the rotation's matrix
        m = torch.eye(D, dtype=torch.float64, device=dev)
        for k in range(8):
            a, b = (2 * k, 2 * k + 1) if interleaved else (k, k + 8)
            m[a, a], m[a, b], m[b, a], m[b, b] = t[i, k], -t[i, 8 + k], t[i, 8 + k], t[i, k]
        want[i] = g[i].double() @ m
    assert torch.all((x.grad.double() - want).abs() <= 4 * 2.0 ** -24 * (2 * g.abs().max() * rope.table.abs().max()))
    # differences: the map is linear, so a step of 1 has no truncation error
    with torch.no_grad():
        f0 = (rope(x, p).double() * g).sum()
        for at in [(0, 0, 0), (1, 2, 9), (5, 1, 31), (3, 0, 15)]:
            y = x.detach().clone()
            y[at] += 1
            d = (rope(y, p).double() * g).sum() - f0
            big = (x.abs().max() + 1) * g.abs().max() * rope.table.abs().max()
            assert abs(d - x.grad[at]) <= 32 * 2.0 ** -24 * big  # 4 changed values, 4 roundings each, both sides


def test_gradient_of_the_gradient(dev):
    """Second derivatives of sum(sin(R x)) along v: -R^T (sin(R x) * R v).  R x and R v are off by 3
    roundings of their largest sum, the sine by as much and 4 steps of 2^-24, product and R^T by
    four more."""
    rope = RotaryPositions(32, 50)
    x = torch.randn((5, 2, 32), device=dev, requires_grad=True)
    v = torch.randn((5, 2, 32), device=dev)
    p = torch.randint(0, 50, (5,), dtype=torch.int32, device=dev)
    first, = torch.autograd.grad(rope(x, p).sin().sum(), x, create_graph=True)
    got, = torch.autograd.grad((first * v).sum(), x)
    c, s = (t[:, None] for t in rope.table.double()[p.long()].split(16, -1))

    def turn(a, sign):
        a1, a2 = a.detach().double().split(16, -1)
        return torch.cat([a1 * c - sign * a2 * s, a2 * c + sign * a1 * s], -1)
    want = -turn(turn(x, 1).sin() * turn(v, 1), -1)
    mx, mv = 2 * x.abs().max(), 2 * v.abs().max()
    assert torch.all((got.double() - want).abs() <= 2 * mv * (3 * mx + 12) * 2.0 ** -24)
    # a second use of the same keys adds up
    x.grad = None
    (rope(x, p).sum() + rope(x, p).sum()).backward()
    once, = torch.autograd.grad(rope(x, p).sum(), x)
    assert torch.equal(x.grad, 2 * once)


def test_rotations_compose_and_keep_distances(dev):
    """Scores depend on distances only: q at m against k at n as q at m + s against k at n + s."""
    rope = RotaryPositions(128, 131072)
    q, k = torch.randn((2, 1, 1, 128), device=dev)
    def at(x, p):
        return rope(x, torch.tensor([p], dtype=torch.int32, device=dev)).double().flatten()
    a, b = at(q, 1000) @ at(k, 990), at(q, 131000) @ at(k, 130990)
    # table entries are off by 2^-25 each, products and sums as in the bits' test
    assert abs(a - b) <= 2 * 8 * 2.0 ** -24 * (q.abs().double().flatten() @ k.abs().double().flatten() * 2 + 64)


def test_another_stream_and_a_graph(dev):
    rope = RotaryPositions(64, 50)
    x = torch.randn((9, 4, 64), device=dev)
    p = torch.randint(0, 50, (9,), dtype=torch.int32, device=dev)
    want = rope(x, p)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rope(x, p)
    torch.cuda.current_stream().wait_stream(s)
    assert same_bits(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rope(x, p)
    for i in range(4):
        x.copy_(torch.randn((9, 4, 64), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert same_bits(y, rope(x, p))


# ------------------------------------------------------------------ the FP8 append

def paged(lens, old, P, extra, dev, seed):
    g = torch.Generator().manual_seed(seed)
    need = [-(-(a + b) // P) for a, b in zip(lens, old)]
    n_pages = sum(need) + extra
    perm = torch.randperm(n_pages, generator=g).to(torch.int32)
    bt = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    k = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[k:k + n]
        k += n
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32)
    return bt.to(dev), cu.to(dev), torch.tensor(old, dtype=torch.int32, device=dev), n_pages


CASES = [  # lens, old, L, H, D, P, rot, padded rows
    ([1], [0], 1, 1, 64, 1, 64, 0), ([1, 1, 1], [5, 0, 33], 3, 8, 128, 16, 128, 0), ([0, 7, 0, 40], [3, 0, 9, 1], 2, 3, 64, 24, 32, 5),
    ([300, 5, 129], [0, 100, 17], 1, 8, 128, 16, 64, 0), ([17], [0], 2, 1, 256, 16, 256, 3), ([64, 31], [0, 0], 2, 5, 128, 3, 112, 1),
    ([2500, 1, 1700], [0, 4000, 11], 4, 8, 128, 16, 128, 2), ([9000], [0], 1, 12, 64, 32, 64, 0)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("mode", ["dynamic", "single", "two", "static", "saturate"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_append_equals_rotation_then_append(dev, interleaved, mode, case):
    lens, old, L, H, D, P, rot, pad = CASES[case]
    T = sum(lens)
    bt, cu, start, n_pages = paged(lens, old, P, 3, dev, case)
    g = torch.Generator(device=dev).manual_seed(case)
    x = torch.randn((L, T + pad, 2, H, D), generator=g, device=dev).to(torch.bfloat16)
    x[:, :, 0, H // 2] *= 30
    if pad:
        x[:, T:] = 1e4  # rows behind the last sequence count for nothing
    table = table64(max(a + b for a, b in zip(lens, old)) + 1, rot, dev)
    positions = torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in zip(old, lens)]).to(dev)
    turned = x[:, :T].clone()
    for layer in range(L):
        turned[layer, :, 0] = kv.rope(x[layer, :T, 0].contiguous(), table, positions, interleaved=interleaved)
    pool = torch.randint(0, 256, (L, n_pages, 2, H, P, D), generator=g, device=dev, dtype=torch.uint8)
    want_pool = pool.clone()
    scales = None
    dynamic = mode in ("dynamic", "single", "two")
    if not dynamic:
        scales = torch.rand((L, 2, H), generator=g, device=dev) * 0.02 + 0.01
        scales[0, 0, 0] = -0.03
    want_err, err = torch.zeros(1, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    kw = dict(start_pos=start, static_scales=not dynamic, saturate=mode == "saturate")
    want = kv.kv_quant_append(turned, cu, bt, want_pool, scales=None if scales is None else scales.clone(), err=want_err,
                              **kw)
    got = kv.kv_rope_append(x, table, cu, bt, pool, scales=scales, interleaved=interleaved, err=err,
                            single_pass=mode == "single", two_pass=mode == "two", **kw)
    assert same_bits(got, want) and torch.equal(pool, want_pool)
    assert err.item() == want_err.item()


def test_append_that_the_rule_sends_through_one_pass(dev):
    """A batch large enough that the call takes the cooperative pass by itself, in several parts:
    many sequences, rows behind them, a share that nearly fills the registers."""
    L, H, D, P, rot = 2, 8, 128, 16, 128
    rng = np.random.default_rng(3)
    lens = rng.integers(100, 1900, 70).tolist()
    bt, cu, start, n_pages = paged(lens, [0] * 70, P, 2, dev, 7)
    T = sum(lens)
    x = torch.randn((L, T + 50, 2, H, D), device=dev).to(torch.bfloat16)
    x[:, T:] = 1e4
    table = table64(2000, rot, dev)
    a, b = (torch.zeros((L, n_pages, 2, H, P, D), dtype=torch.uint8, device=dev) for _ in range(2))
    sa = kv.kv_rope_append(x, table, cu, bt, a, check=True)
    sb = kv.kv_rope_append(x, table, cu, bt, b, check=True, two_pass=True)
    assert same_bits(sa, sb) and torch.equal(a, b)


def test_append_into_a_pool_beyond_2_gib(dev):
    """Pages whose offsets pass 31 bits, both passes and one, static scales."""
    H, D, P = 8, 128, 16
    n_pages = 140_000  # 32 KiB each
    table = table64(300, D, dev)
    bt = torch.tensor([[n_pages - 1, 3, 70_000, 65_535, 65_536]], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 70], dtype=torch.int32, device=dev)
    x = torch.randn((1, 70, 2, H, D), device=dev).to(torch.bfloat16)
    small = torch.zeros((1, 5, 2, H, P, D), dtype=torch.uint8, device=dev)
    want = kv.kv_rope_append(x, table, cu, torch.arange(5, dtype=torch.int32, device=dev)[None], small)
    pool = torch.empty((1, n_pages, 2, H, P, D), dtype=torch.uint8, device=dev)
    for kw in (dict(two_pass=True), dict(single_pass=True), dict(static_scales=True, scales=want)):
        pool[0, bt[0].long()] = 0
        got = kv.kv_rope_append(x, table, cu, bt, pool, check=True, **kw)
        assert same_bits(got, want) and torch.equal(pool[0, bt[0].long()], small[0]), kw


def test_append_gives_up_waiting_then_recovers(dev):
    """A bound of zero makes the single pass's first wait without progress take the release path:
    every wave exits, the call is flagged, and with the bound restored the bits are right."""
    H, D, P = 8, 128, 16
    bt, cu, start, n_pages = paged([700, 333, 1201], [0, 0, 0], P, 1, dev, 2)
    table = table64(1300, D, dev)
    x = torch.randn((2, 2234, 2, H, D), device=dev).to(torch.bfloat16)
    pools = [torch.zeros((2, n_pages, 2, H, P, D), dtype=torch.uint8, device=dev) for _ in range(2)]
    kv.set_wait_bound_us(0)
    try:
        with pytest.raises(ValueError, match="wait"):
            kv.kv_rope_append(x, table, cu, bt, pools[0], check=True, single_pass=True)
    finally:
        kv.set_wait_bound_us(None)
    a = kv.kv_rope_append(x, table, cu, bt, pools[0], check=True, single_pass=True)
    b = kv.kv_rope_append(x, table, cu, bt, pools[1], check=True, two_pass=True)
    assert same_bits(a, b) and torch.equal(*pools)


def test_append_bad_pages_and_positions(dev):
    L, H, D, P = 2, 2, 64, 16
    bt = torch.tensor([[0, 99, 2], [3, -1, 4]], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 48, 96], dtype=torch.int32, device=dev)
    x = torch.randn((L, 96, 2, H, D), device=dev).to(torch.bfloat16)
    for n_pos, bits in ((48, N.ZX_KERR_PAGE_RANGE), (40, N.ZX_KERR_PAGE_RANGE | N.ZX_KERR_POS_RANGE)):
        table = table64(n_pos, D, dev)
        pool = torch.full((L, 5, 2, H, P, D), 9, dtype=torch.uint8, device=dev)
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        scales = torch.full((L, 2, H), 0.01, device=dev)
        kv.kv_rope_append(x, table, cu, bt, pool, scales=scales, static_scales=True, saturate=True, err=err)
        assert err.item() & ~N.ZX_KERR_OVERFLOW == bits
        assert torch.all(pool[:, 1] == 9)  # no table entry names it
        wrote = (pool != 9).any(-1)  # [L, page, 2, H, P]
        assert wrote[:, 0].float().mean() > 0.99 and wrote[:, 3].float().mean() > 0.99
        last = min(16, n_pos - 32)
        for page in (2, 4):
            assert wrote[:, page, :, :, :last].float().mean() > 0.99 and not wrote[:, page, :, :, last:].any()
    with pytest.raises(ValueError, match="block table"):
        kv.kv_rope_append(x, table64(48, D, dev), cu, bt, pool, check=True)


def test_append_non_finite(dev):
    """A NaN or an infinity in a pair reaches its slab's scale as it does after a rotation."""
    H, D, P = 2, 64, 16
    bt, cu, start, n_pages = paged([20], [0], P, 0, dev, 0)
    table = table64(20, D, dev)
    for bad, one in ((float("nan"), False), (float("inf"), False), (float("nan"), True), (float("inf"), True)):
        x = torch.randn((1, 20, 2, H, D), device=dev).to(torch.bfloat16)
        x[0, 3, 0, 1, 5] = bad
        turned = x.clone()
        turned[0, :, 0] = kv.rope(x[0, :, 0].contiguous(), table, torch.arange(20, dtype=torch.int32, device=dev))
        a, b = (torch.zeros((1, n_pages, 2, H, P, D), dtype=torch.uint8, device=dev) for _ in range(2))
        sa, sb = kv.kv_rope_append(x, table, cu, bt, a, single_pass=one), kv.kv_quant_append(turned, cu, bt, b)
        assert torch.equal(sa.isnan(), sb.isnan()) and torch.equal(a, b)


def test_append_of_nothing_and_refusals(dev):
    H, D, P = 2, 64, 16
    bt, cu = torch.zeros((1, 2), dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    pool = torch.zeros((1, 3, 2, H, P, D), dtype=torch.uint8, device=dev)
    table = table64(8, D, dev)
    x = torch.zeros((1, 4, 2, H, D), dtype=torch.bfloat16, device=dev)
    s = kv.kv_rope_append(x[:, :0], table, cu, bt, pool)
    assert torch.equal(s, kv.kv_quant_append(x[:, :0], cu, bt, pool))
    for bad in (lambda: kv.kv_rope_append(x, table, cu, bt, pool[..., :32]), lambda: kv.kv_rope_append(x.float(), table, cu, bt, pool),
                lambda: kv.kv_rope_append(x, table.double(), cu, bt, pool),
                lambda: kv.kv_rope_append(x, torch.zeros((8, 128), device=dev), cu, bt, pool),
                lambda: kv.kv_rope_append(x, table, cu.long(), bt, pool), lambda: kv.kv_rope_append(x, table, cu, bt[0], pool),
                lambda: kv.kv_rope_append(x, table, cu, bt, pool, static_scales=True),
                lambda: kv.kv_rope_append(x, table, cu, bt, pool, saturate=True),
                lambda: kv.kv_rope_append(x, table, cu, bt, pool, start_pos=torch.zeros(2, dtype=torch.int32, device=dev)),
                lambda: kv.kv_rope_append(x, table, cu.cpu(), bt, pool)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("single", [False, True])
def test_append_in_a_graph(dev, single):
    """Captured appends (two graphs, each with its own workspace) replay to the eager bits."""
    H, D, P, L = 4, 128, 16, 2
    lens, old = [40, 3], [0, 20]
    bt, cu, start, n_pages = paged(lens, old, P, 0, dev, 1)
    table = table64(64, D, dev)
    x = torch.randn((L, 43, 2, H, D), device=dev).to(torch.bfloat16)
    kv.kv_rope_append(x, table, cu, bt, torch.zeros((L, n_pages, 2, H, P, D), dtype=torch.uint8, device=dev), start_pos=start,
                      single_pass=single)
    pools = [torch.zeros((L, n_pages, 2, H, P, D), dtype=torch.uint8, device=dev) for _ in range(2)]
    scales = [torch.zeros((L, 2, H), device=dev) for _ in range(2)]
    graphs = []
    for pool, sc in zip(pools, scales):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv.kv_rope_append(x, table, cu, bt, pool, scales=sc, start_pos=start, single_pass=single)
        graphs.append(g)
    for i in range(3):
        x.copy_(torch.randn(x.shape, device=dev))
        for g in graphs:
            g.replay()
        want = torch.zeros_like(pools[0])
        s = kv.kv_rope_append(x, table, cu, bt, want, start_pos=start)
        torch.cuda.synchronize()
        for pool, sc in zip(pools, scales):
            assert torch.equal(pool, want) and same_bits(sc, s)


@pytest.mark.parametrize("n, H, D, row, head", [
    (2, 3, 16, 64, 48), (3, 2, 16, 16, 64), (2, 3, 16, 16, 32), (1, 4, 16, 0, 16), (4, 1, 16, 16, 0), (7, 5, 32, 32, 7 * 32),
    (2, 2, 32, 36, 72), (3, 3, 16, 116, 40)])
def test_an_out_whose_rows_lie_between_each_other(dev, n, H, D, row, head):
    """Any strides whose rows do not overlap are written, and nothing between the rows is."""
    x = torch.randn((n, H, D), device=dev)
    table, p = table64(9, 16, dev), torch.randint(0, 9, (n,), dtype=torch.int32, device=dev)
    room = torch.full(((n - 1) * row + (H - 1) * head + D + 4,), 7.0, device=dev)
    out = room.as_strided((n, H, D), (row, head, 1))
    want = torch.full_like(room, 7.0)
    want.as_strided((n, H, D), (row, head, 1)).copy_(kv.rope(x, table, p))
    assert kv.rope(x, table, p, out=out) is out
    assert same_bits(room, want)


def test_an_out_whose_rows_overlap_is_refused(dev):
    x = torch.randn((4, 2, 64), device=dev)
    table, p = table64(9, 64, dev), torch.zeros(4, dtype=torch.int32, device=dev)
    room = torch.zeros(1000, device=dev)
    for row, head in ((64, 64), (72, 64), (64, 72), (64, 128)):
        with pytest.raises(ValueError, match="overlap"):
            kv.rope(x, table, p, out=room.as_strided((4, 2, 64), (row, head, 1)))
    assert not room.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_at_any_alignment(dev, dtype):
    """A gradient arrives as autograd lays it out: at an odd offset, expanded, with other strides."""
    rope = RotaryPositions(32, 20, rotary_dim=16)
    x = torch.randn((5, 2, 32), device=dev).to(dtype).requires_grad_()
    p = torch.randint(0, 20, (5,), dtype=torch.int32, device=dev)
    g = torch.randn(320 + 7, device=dev).to(dtype)

    def back(t):
        return kv.rope(t.contiguous().clone(), rope.table, p, transpose=True)
    for lead in (0, 1, 3, 7):
        got, = torch.autograd.grad(torch.cat([g[:lead], rope(x, p).flatten()]), x, g[:320 + lead])
        assert same_bits(got, back(g[lead:320 + lead].view(5, 2, 32))), lead
    got, = torch.autograd.grad(rope(x, p).sum(), x)
    assert same_bits(got, back(torch.ones((5, 2, 32), device=dev, dtype=dtype)))
    got, = torch.autograd.grad(rope(x, p).transpose(0, 2).contiguous(), x, g[:320].view(32, 2, 5))
    assert same_bits(got, back(g[:320].view(32, 2, 5).transpose(0, 2)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forward_mode_derivative(dev, dtype):
    """The tangent turns with the values, to the bit, alone and where a gradient is asked for too; a
    trace holds the kernel."""
    rope = RotaryPositions(64, 50, rotary_dim=32, interleaved=True)
    p = torch.randint(0, 50, (9,), dtype=torch.int32, device=dev)
    x, v = torch.randn((2, 9, 4, 64), device=dev).to(dtype)
    for primal in (x, x.clone().requires_grad_()):
        with fwAD.dual_level():
            out = fwAD.unpack_dual(rope(fwAD.make_dual(primal, v), p))
            assert same_bits(out.primal.detach(), rope(x, p)) and same_bits(out.tangent.detach(), rope(v, p))
    leaf, u = x.clone().requires_grad_(), torch.randn(x.shape, device=dev).to(dtype)
    with fwAD.dual_level():  # the gradient's own tangent: d/de <u, (R (x + e v))^2> = R^T (2 u R v)
        g, = torch.autograd.grad((rope(fwAD.make_dual(leaf, v), p).square() * u).sum(), leaf)
        got = fwAD.unpack_dual(g).tangent
    rv = rope(v, p).double()
    want, near = 2 * u.double() * rv, 2 * u.double().abs() * rv.abs()
    c, s = (t[:, None] for t in rope.table.double()[p.long()].split(16, 1))
    a, b = want[..., 0:32:2].clone(), want[..., 1:32:2].clone()
    want[..., 0:32:2], want[..., 1:32:2] = a * c + b * s, b * c - a * s
    a, b = near[..., 0:32:2].clone(), near[..., 1:32:2].clone()
    near[..., 0:32:2], near[..., 1:32:2] = a + b, a + b
    # six roundings to the type on the way at most: the square's derivative (2), its tangent (2), their
    # sum with u, the rotation
    assert torch.all((got.double() - want).abs() <= 6 * HALF_STEP[dtype] * 1.05 * near + 1e-30)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(lambda t: rope(t, p), (x,))
    assert same_bits(traced(v), rope(v, p))
