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
