"""GPU attention for batches whose sequences share pages, FP8 and 4 bits, against float64 over each
sequence's own block table.

Tolerance, elementwise, beside half a bf16 step of the value (2^-8 of it) for the last rounding:

* weights: FP8 rounds them to fp16 (half a step, 2^-11 of a weight; below 2^-21 of the largest, where
  fp16 is subnormal, 2^-32 of it at most), 4 bits carries them as bf16 hi + lo (2^-16); a row is a
  weighted mean, so weights off by e move it by at most 2 e max|V|, n of them off by 2^-32 of the
  largest by 2 n 2^-32 max|V|;
* scores: a sum of D products in fp32 and its scaling are off by at most (D + 4) 2^-24 sum|q k|, the
  exponential by 2^-22 of a weight: each weight by (D + 4) 2^-24 |sm| sum|q k| + 2^-21;
* sums over keys in fp32: at most (n / 32 + 64) additions follow each other in an accumulator and its
  merges, 2^-24 each, on numerator and denominator: 2 (n / 32 + 64) 2^-24 max|V|.
"""
import numpy as np
import pytest
import torch

from zenyx_amd import _native as N
from zenyx_amd import kv

pytestmark = pytest.mark.gpu
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def i32(v, dev):
    return torch.as_tensor(np.asarray(v, np.int32), device=dev)


class Batch:
    """Groups of (sequences, shared positions) over a shuffled pool; own: tokens of each sequence
    beyond what its group shares; loose: sequences in no group, after the others."""

    def __init__(self, dev, bits, groups, own, rows, Hq, Hkv, D, P, seed=0, loose=(), behind=0):
        rng = np.random.default_rng(seed)
        self.bits, self.Hq, self.Hkv, self.D, self.P, self.dev = bits, Hq, Hkv, D, P, dev
        n_group = sum(n for n, _ in groups)
        lens, share = [], []
        for g, (n, s) in enumerate(groups):
            share += [s] * n
        share += [0] * len(loose)
        own = list(own) + list(loose)
        self.lens = [s + o for s, o in zip(share, own)]
        need = [-(-t // P) for t in self.lens]
        self.n_pages = sum(need) + 5
        perm = rng.permutation(self.n_pages)
        bt = np.full((len(own), max(max(need), 1) + 1), -1, np.int64)
        at, b = 0, 0
        for n, s in groups:
            lead = None
            for _ in range(n):
                k = s // P  # whole pages are the same ones
                if lead is None:
                    lead = perm[at:at + -(-s // P)]
                    at += len(lead)
                bt[b, :len(lead)] = lead
                fresh = need[b] - k
                # a page that is shared in part is a copy
                bt[b, k:need[b]] = perm[at:at + fresh]
                at += fresh
                b += 1
        for _ in loose:
            bt[b, :need[b]] = perm[at:at + need[b]]
            at += need[b]
            b += 1
        self.bt_np, self.groups = bt, groups
        g = torch.Generator(device=dev).manual_seed(seed)
        if bits == 8:
            x = torch.randn((self.n_pages, 2, Hkv, P, D), generator=g, device=dev) * 60
            self.pool = x.to(torch.float8_e4m3fn).view(torch.uint8)
            self.scales = (torch.rand((2, Hkv), generator=g, device=dev) + 0.5) / 60
        else:
            self.pool = torch.randint(0, 256, (self.n_pages, 2, Hkv, P // 16, 17 * D // 2), generator=g, device=dev,
                                      dtype=torch.uint8)
            self.pool[..., 8 * D:] = torch.randint(124, 128, self.pool[..., 8 * D:].shape, generator=g, device=dev,
                                                   dtype=torch.uint8)
            self.scales = None
        self.copy_partial()
        self.rows = list(rows)
        self.q = torch.randn((sum(rows) + behind, Hq, D), generator=g, device=dev).mul_(1.5).to(torch.bfloat16)
        self.cu_q = i32(np.concatenate([[0], np.cumsum(rows)]), dev)
        self.cu_group = i32(np.concatenate([[0], np.cumsum([n for n, _ in groups])]), dev)
        self.shared = i32([s for _, s in groups], dev)
        self.bt, self.seq_lens = i32(bt, dev), i32(self.lens, dev)

    def copy_partial(self):
        """Every sequence's copy of a page that its group shares in part holds what the first one's does."""
        b = 0
        for n, s in self.groups:
            k = s // self.P
            if s % self.P:
                for i in range(1, n):
                    self.pool[self.bt_np[b + i, k]] = self.pool[self.bt_np[b, k]]
            b += n

    def call(self, cu_q=True, **kw):
        args = [self.q, self.pool] + ([self.scales] if self.bits == 8 else []) + [self.bt, self.seq_lens, self.cu_group,
                                                                                  self.shared]
        f = kv.paged_attention_shared if self.bits == 8 else kv.paged_attention4_shared
        return f(*args, cu_q=self.cu_q if cu_q else None, **kw)

    def cached(self, b):
        """(K, V) float64 [Hkv, len, D] of sequence b."""
        n, D = self.lens[b], self.D
        t = self.pool[torch.as_tensor(self.bt_np[b, :-(-n // self.P)], device=self.dev)]
        if self.bits == 8:
            v = t.view(torch.float8_e4m3fn).double() * self.scales.double()[:, :, None, None]
        else:
            c = t[..., :8 * D].unflatten(-1, (D // 32, 16, 16))
            both = torch.stack([c & 15, c >> 4], -1).flatten(-2)
            p = t[..., 8 * D:].unflatten(-1, (D // 32, 16)).double()
            power = torch.where(p == 255, torch.nan, torch.exp2(p - 127))
            v = torch.tensor(E2M1, dtype=torch.float64, device=self.dev)[both.int()] * power[..., None]
            v = v.transpose(-3, -2).flatten(-2).flatten(-3, -2)
        v = v.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]
        return v[0], v[1]

    def check(self, got, causal=True, sm=None, exact_nan=True):
        sm = self.D ** -0.5 if sm is None else sm
        grp = self.Hq // self.Hkv
        e_w = 2.0 ** -11 if self.bits == 8 else 2.0 ** -16
        at = 0
        worst = 0.0
        for b, (n, r) in enumerate(zip(self.lens, self.rows)):
            q = self.q[at:at + r].double().view(r, self.Hkv, grp, self.D).permute(1, 2, 0, 3)  # [H, grp, r, D]
            g = got[at:at + r].double().view(r, self.Hkv, grp, self.D).permute(1, 2, 0, 3)
            at += r
            if n == 0:
                assert (g == 0).all()
                continue
            k, v = self.cached(b)
            s = torch.matmul(q, k.transpose(-1, -2)[:, None]) * sm
            size = torch.matmul(q.abs(), k.abs().transpose(-1, -2)[:, None]) * abs(sm)
            hide = torch.zeros((r, n), dtype=torch.bool, device=self.dev)
            if causal:
                hide = torch.arange(n, device=self.dev) > n - r + torch.arange(r, device=self.dev)[:, None]
            s = s.masked_fill(hide, -torch.inf)
            empty = hide.all(-1)
            p = torch.softmax(s, -1)
            p = torch.where(hide | empty[:, None], 0.0, p)
            live = torch.where((p > 0)[..., None], v[:, None, None], 0.0) if v.isnan().any() else v[:, None]
            want = (p[..., None] * live).sum(-2) if v.isnan().any() else torch.matmul(p, live)
            vmax = v.nan_to_num(0.0).abs().amax((1, 2))[:, None, None, None]
            e = e_w + ((self.D + 4) * 2.0 ** -24 * size.nan_to_num(0.0).amax(-1, keepdim=True) + 2.0 ** -21)
            tol = 2.0 ** -8 * want.abs() + (2 * e + 2 * n * 2.0 ** -32 + 2 * (n / 32 + 64) * 2.0 ** -24) * vmax
            nan = want.isnan()
            assert torch.equal(g.isnan(), nan), (b, int(g.isnan().sum()), int(nan.sum()))
            bad = ((g - want).abs() > tol) & ~nan
            assert not bad.any(), (b, n, r, float(((g - want).abs() / tol)[~nan].max()))
            worst = max(worst, float(((g - want).abs() / tol)[~nan].max()) if (~nan).any() else 0.0)
        return worst


SHAPES = [  # groups, own, rows, Hq, Hkv, D, P
    ([(2, 32)], [1, 5], [1, 1], 8, 2, 128, 16),
    ([(3, 48)], [0, 17, 130], [1, 1, 1], 4, 4, 64, 16),
    ([(1, 16)], [0], [1], 1, 1, 64, 16),
    ([(5, 333)], [10, 200, 1, 64, 31], [1] * 5, 32, 8, 128, 16),
    ([(4, 1000), (1, 64), (2, 0), (7, 250)], list(range(1, 15)), [1] * 14, 12, 12, 64, 32),
    ([(40, 700)], [3 * i for i in range(40)], [1] * 40, 32, 8, 128, 16),
    ([(70, 100), (0, 40), (33, 513)], [i % 50 for i in range(103)], [1] * 103, 8, 1, 128, 64),
    ([(3, 100)], [40, 7, 300], [1] * 3, 16, 4, 256, 16),
    ([(2, 64)], [9, 90], [1, 1], 40, 2, 64, 16),
    ([(2, 64)], [9, 90], [1, 1], 19, 1, 128, 48),
    # several rows
    ([(3, 96)], [8, 30, 100], [8, 3, 1], 8, 2, 128, 16),
    ([(6, 400), (2, 33)], [20, 20, 5, 9, 100, 64, 4, 3], [5, 8, 1, 0, 3, 2, 4, 3], 32, 8, 128, 16),
    ([(2, 160)], [70, 45], [70, 40], 4, 2, 64, 16),
    ([(3, 64)], [33, 20, 5], [3, 2, 5], 8, 8, 256, 32),
    # rows that reach back into the shared positions, and sequences shorter than what is shared
    ([(2, 128)], [2, 0], [5, 7], 8, 2, 128, 16),
]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_against_float64(dev, bits, shape):
    groups, own, rows, Hq, Hkv, D, P = SHAPES[shape]
    t = Batch(dev, bits, groups, own, rows, Hq, Hkv, D, P, seed=shape)
    one = all(r == 1 for r in rows)
    t.check(t.call(cu_q=not one, check=True))
    if one:
        t.check(t.call(cu_q=True, max_q_per_seq=1, check=True))
    else:
        t.check(t.call(causal=False, check=True), causal=False)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("groups, loose, rows", [
    ([(300, 64)], [], 1),                                # more sequences than the kernel keeps in LDS
    ([(1, 16)] * 280 + [(30, 128)], [5] * 7, 1),         # and more groups
    ([(150, 80), (120, 48)], [200, 0, 3], 2)])
def test_many_sequences(dev, bits, groups, loose, rows):
    n = sum(c for c, _ in groups)
    own = [rows + i % 37 for i in range(n)]
    r = [rows if i % 3 else 1 for i in range(n + len(loose))]
    t = Batch(dev, bits, groups, own, r, 8, 2, 64, 16, seed=3, loose=loose)
    t.check(t.call(check=True))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D, loose", [(128, [40, 0, 300]), (64, [1])])
def test_sequences_in_no_group(dev, bits, D, loose):
    t = Batch(dev, bits, [(3, 128)], [5, 60, 200], [1] * (3 + len(loose)), 8, 2, D, 16, loose=loose)
    want = t.call(cu_q=False, check=True)
    t.check(want)
    # no groups at all: attention over each sequence's own table
    t.cu_group, t.shared = i32([0], dev), i32([], dev)
    t.check(t.call(cu_q=False, check=True))
    # a group of which nothing is shared, one of each alone, and all that one has in common
    for cu, s in (([0, 3], [0]), ([0, 1, 2, 3], [128, 128, 128]), ([0, 2, 3], [128, 0]), ([0, 3], [100]), ([0, 3], [15])):
        t.cu_group, t.shared = i32(cu, dev), i32(s, dev)
        t.check(t.call(cu_q=False, check=True))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("sm", [-0.11, 0.0, 1.0])
def test_other_scales(dev, bits, sm):
    for rows in ([1] * 6, [2, 1, 5, 3, 1, 4]):
        t = Batch(dev, bits, [(6, 192)], [9, 30, 5, 70, 6, 20], rows, 16, 4, 128, 16, seed=5)
        t.check(t.call(sm_scale=sm, check=True), sm=sm)


@pytest.mark.parametrize("n", [20, 6])
def test_negative_fp8_scales(dev, n):
    t = Batch(dev, 8, [(n, 160)], list(range(n)), [1] * n, 16, 4, 128, 16, seed=6)
    t.scales[0, 1] *= -1
    t.scales[1, 2] *= -1
    t.check(t.call(cu_q=False, check=True))


def nan_at(t, b, pos, head, ch, kv_):
    """Makes channel ch (4 bits: its block) of position pos of sequence b a NaN."""
    page = int(t.bt_np[b, pos // t.P])
    if t.bits == 8:
        t.pool[page, kv_, head, pos % t.P, ch] = 0xFF
    else:
        t.pool[page, kv_, head, (pos % t.P) // 16, 8 * t.D + 16 * (ch // 32) + pos % 16] = 255


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D, n", [(64, 3), (128, 3), (128, 18)])
def test_nan_values_reach_the_rows_that_see_them(dev, bits, D, n):
    """Of the shared keys and of a sequence's own, at positions that some rows do not see; behind the last
    position of a sequence they reach none."""
    rows = [8, 3, 1] + [2] * (n - 3)
    t = Batch(dev, bits, [(n, 96)], [8, 37, 5] + [10] * (n - 3), rows, 8, 2, D, 16, seed=9)
    nan_at(t, 0, 40, 0, 5, 1)               # everyone's
    nan_at(t, 0, 96 + 4, 1, 33, 1)          # seen by rows 4 .. of sequence 0
    nan_at(t, 1, 96 + 36, 0, D - 1, 1)      # by the last row of sequence 1
    for pos in range(96 + 5, 112):          # behind sequence 2's last position, on its page
        nan_at(t, 2, pos, 1, 0, 1)
        nan_at(t, 2, pos, 0, 3, 0)
    t.check(t.call(check=True))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n", [2, 24])
def test_nan_keys(dev, bits, n):
    t = Batch(dev, bits, [(n, 64)], [20] * n, [1] * n, 8, 2, 128, 16, seed=10)
    nan_at(t, 1, 64 + 3, 1, 7, 0)  # a key of sequence 1 alone: its rows of that KV head
    got = t.call(cu_q=False, check=True)
    bad = got.isnan().view(n, 2, 4, 128)
    assert bad[1, 1].all() and not bad[1, 0].any() and not bad[0].any()
    nan_at(t, 0, 9, 0, 7, 0)  # a shared one: every row of the other
    bad = t.call(cu_q=False, check=True).isnan().view(n, 2, 4, 128)
    assert bad[:, 0].all() and not bad[0, 1].any()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n", [2, 24])
def test_bad_pages_are_left_out_and_flagged(dev, bits, n):
    t = Batch(dev, bits, [(n, 128)], [40] * n, [1] * n, 8, 2, 128, 16, seed=11)
    good = t.call(cu_q=False, check=True)
    for b, col, bad in ((0, 3, -1), (0, 3, t.n_pages), (1, 8, -7), (1, 8, 1 << 30)):
        keep = int(t.bt[b, col])
        t.bt[b, col] = bad
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        got = t.call(cu_q=False, err=err)
        assert int(err) == N.ZX_KERR_PAGE_RANGE and torch.isfinite(got).all()
        with pytest.raises(ValueError, match="block table"):
            t.call(cu_q=False, check=True)
        touched = (got != good).flatten(1).any(1)
        assert touched.all() if b == 0 else touched.tolist() == [i == 1 for i in range(n)]
        t.bt[b, col] = keep
    assert torch.equal(t.call(cu_q=False, check=True), good)


@pytest.mark.parametrize("bits", [8, 4])
def test_what_groups_and_lengths_flag(dev, bits):
    t = Batch(dev, bits, [(4, 64), (3, 32)], [5] * 7, [1] * 7, 8, 2, 64, 16, seed=12)
    for cu, lens in (([0, 5, 4], None), ([-1, 4, 7], None), ([0, 4, 9], None), ([0, 6, 2], None), ([3, 0, 7], None),
                     ([0, 4, 7], 1 << 20)):
        t.cu_group = i32(cu, dev)
        s = t.seq_lens.clone()
        if lens:
            s[2] = lens
        args = [t.q, t.pool] + ([t.scales] if bits == 8 else []) + [t.bt, s, t.cu_group, t.shared]
        with pytest.raises(ValueError, match="position"):
            (kv.paged_attention_shared if bits == 8 else kv.paged_attention4_shared)(*args, check=True)
    # rows beyond max_q_per_seq: not computed, left as they are
    t = Batch(dev, bits, [(3, 64)], [20] * 3, [2, 5, 1], 8, 2, 64, 16, seed=13)
    out = torch.full_like(t.q, 7.0)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    t.call(max_q_per_seq=3, out=out, err=err)
    assert int(err) == N.ZX_KERR_POS_RANGE
    assert (out[5:7] == 7).all() and (out[:5] != 7).any(-1).any(-1).all() and (out[7] != 7).any()


@pytest.mark.parametrize("bits", [8, 4])
def test_rows_in_no_sequence_are_left(dev, bits):
    t = Batch(dev, bits, [(3, 64)], [20] * 3, [2, 0, 3], 8, 2, 64, 16, seed=14, behind=4)
    out = torch.full_like(t.q, 7.0)
    t.call(out=out, check=True)
    t.check(out)
    assert (out[5:] == 7).all()
    empty = torch.empty((0, 8, 64), dtype=torch.bfloat16, device=dev)
    t.q, t.cu_q = empty, i32([0, 0, 0, 0], dev)
    assert t.call(check=True).shape == empty.shape


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n, D", [(3, 64), (30, 128)])
def test_captured_replays_follow_the_lengths(dev, bits, n, D):
    """One captured call on other lengths, groups and pages, with eager work between the replays, and on
    another stream; twice at once on streams of their own."""
    t = Batch(dev, bits, [(n, 640)], [64] * n, [1] * n, 8, 2, D, 16, seed=15)
    out = torch.empty_like(t.q)
    t.call(cu_q=False, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.call(cu_q=False, out=out)
    for k, (own, shared, cu) in enumerate(((64, 640, [0, n]), (3, 640, [0, n]), (50, 48, [0, n]), (64, 0, [0, n]),
                                           (17, 320, [0, n - 1]), (64, 640, [0, n]))):
        t.lens = [640 + own - i % 3 for i in range(n)]
        t.seq_lens.copy_(i32(t.lens, dev))
        t.shared.copy_(i32([shared], dev))
        t.cu_group.copy_(i32(cu, dev))
        t.q.mul_(-1.0)
        out.zero_()
        graph.replay()
        t.check(out)
        assert torch.equal(out, t.call(cu_q=False))  # the same launch: the same sums in the same order
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    want = out.clone()
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(t.call(cu_q=False))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_pools_beyond_4_gib(dev):
    """Pages whose bytes lie beyond 2^32, FP8 and 4 bits, of wide and narrow groups."""
    for bits, D, n in ((8, 128, 20), (8, 64, 3), (4, 128, 3)):
        t = Batch(dev, bits, [(n, 96)], [20] * n, [1] * n, 8, 2, D, 16, seed=16)
        page = t.pool[0].numel()
        far = torch.zeros((5 * 2 ** 30 // page, *t.pool.shape[1:]), dtype=torch.uint8, device=dev)
        shift = far.shape[0] - t.n_pages
        far[shift:] = t.pool
        want = t.call(cu_q=False)
        t.pool, t.bt = far, torch.where(t.bt >= 0, t.bt + shift, t.bt)
        assert torch.equal(t.call(cu_q=False, check=True), want)
        del far, t


def test_wrappers_refuse(dev):
    t = Batch(dev, 8, [(2, 32)], [5, 5], [1, 1], 8, 2, 128, 16)
    f = Batch(dev, 4, [(2, 32)], [5, 5], [1, 1], 8, 2, 128, 16)
    ok = [t.q, t.pool, t.scales, t.bt, t.seq_lens, t.cu_group, t.shared]
    bad = {0: [t.q.float(), t.q[:1], t.q[..., :64].contiguous(), t.q[:, :3].contiguous(), t.q.cpu()],
           1: [t.pool.int(), t.pool[:, :, :, :, :96].contiguous(), t.pool[0], f.pool],
           2: [None, t.scales.half(), t.scales[:1]], 3: [t.bt.long(), t.bt[0], t.bt[:1].contiguous()],
           4: [t.seq_lens.long(), t.seq_lens[:1]], 5: [t.cu_group.long(), t.cu_group[:1]],
           6: [t.shared.long(), t.shared[None], torch.cat([t.shared] * 3)]}
    for i, values in bad.items():
        for v in values:
            with pytest.raises(ValueError):
                kv.paged_attention_shared(*(ok[:i] + [v] + ok[i + 1:]))
    for kw in (dict(cu_q=t.cu_q.long()), dict(cu_q=t.cu_q[:2]), dict(out=t.q.float()), dict(out=t.q[:1]),
               dict(err=torch.zeros(1, device=dev)), dict(err=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            kv.paged_attention_shared(*ok, **kw)
    with pytest.raises(ValueError):
        kv.paged_attention4_shared(f.q, t.pool, f.bt, f.seq_lens, f.cu_group, f.shared)
    # pages of other sizes belong to the usual decode
    pool = torch.zeros((9, 2, 2, 8, 128), dtype=torch.uint8, device=dev)
    with pytest.raises(ValueError, match="multiple of 16"):
        kv.paged_attention_shared(t.q, pool, t.scales, t.bt, t.seq_lens, t.cu_group, t.shared)


@pytest.mark.parametrize("bits", [8, 4])
def test_rows_out_of_order_are_flagged(dev, bits):
    """cu_q or groups that go back: flagged, no access outside what there is (rows that lie before their
    group's first take no part of it), and a good call afterwards is as before."""
    t = Batch(dev, bits, [(6, 96)], [20] * 6, [2] * 6, 8, 2, 128, 16, seed=17)
    want = t.call(check=True)
    for cu in ([0, 10, 5, 12, 12, 12, 12], [0, 9, 1, 9, 1, 9, 12], [12, 10, 8, 6, 4, 2, 0]):
        for groups, shared in (([0, 6], [96]), ([0, 1, 6], [0, 96]), ([0, 6, 2, 6], [96, 96, 96])):
            cu_q, t.cu_q, t.cu_group, t.shared = t.cu_q, i32(cu, dev), i32(groups, dev), i32(shared, dev)
            err = torch.zeros(1, dtype=torch.int32, device=dev)
            t.call(max_q_per_seq=12, err=err)
            assert int(err) & N.ZX_KERR_POS_RANGE
            t.cu_q, t.cu_group, t.shared = cu_q, i32([0, 6], dev), i32([96], dev)
    assert torch.equal(t.call(check=True), want)
