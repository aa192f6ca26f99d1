"""GPU 4-bit KV pages: append and gather to the bit against the oracle's search for the nearest
code, decode and prefill attention against float64 on the decoded pages.

Attention's tolerance, elementwise, beside half a bf16 step of the value (2^-8 of it) for the last
rounding:

* weights: hi + lo of bf16 carry a weight to 2^-16 of it, one bf16 to 2^-8; a row is a weighted
  mean, so weights off by e move it by at most 2 e max|V|;
* scores: a sum of D products in fp32 and its scaling by sm_scale log2(e) are off by at most
  (D + 4) 2^-24 sum|q k|, the exponential by 2^-22 of a weight: each weight by
  e = (D + 4) 2^-24 |sm| sum|q k| + 2^-21 (subtracting the maximum adds 2^-24 of a score, in it);
* sums over keys in fp32: at most (n / 32 + 64) additions follow each other in an accumulator
  and its merges, 2^-24 each, on numerator and denominator: 2 (n / 32 + 64) 2^-24 max|V|.
"""
import numpy as np
import pytest
import torch

from oracle import kv4 as R
from zenyx_amd import _native as N
from zenyx_amd import kv
from zenyx_amd.train.fp8_kv_quantization import PagedFP4KVCache, PagedFP8KVCache, QuantizedRingAttention
from zenyx_amd.train.rotary import RotaryPositions, rotary_frequencies

pytestmark = pytest.mark.gpu


def bits(t):
    return t.detach().cpu().contiguous().view(torch.int16).numpy()


def tables(total, P, extra, seed):
    rng = np.random.default_rng(seed)
    need = [-(-t // P) for t in total]
    n_pages = sum(need) + extra
    perm = rng.permutation(n_pages).astype(np.int32)
    bt = np.full((len(total), max(max(need), 1)), -1, np.int32)
    k = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[k:k + n]
        k += n
    return bt, n_pages


def i32(v, dev):
    return torch.as_tensor(np.ascontiguousarray(v, np.int32), device=dev)


# ------------------------------------------------------------------ codes

def special_blocks():
    """bf16 bit patterns [n, 32] that visit every power, the ties and what is not finite."""
    rng = np.random.default_rng(0)
    blocks = []
    for e in list(range(0, 12)) + list(range(118, 136)) + list(range(244, 256)):  # exponent fields of the largest
        for m in (0, 1, 63, 64, 65, 95, 96, 97, 127):
            top = (e << 7) | m
            other = rng.integers(0, top + 1, 31) if top else np.zeros(31, np.int64)
            blocks.append(np.concatenate([[top], other]) | (rng.integers(0, 2, 32) << 15))
    # every tie and its neighbours at several powers
    for e in (-120, -3, 0, 5, 100):
        for p in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1, 6):
            v = np.float32(p * 2.0 ** e)
            b = int(v.view(np.uint32)) >> 16
            row = np.array([b, b - 1, b + 1, b | 0x8000, 0, 0x8000] + [b] * 26)
            row[6] = int(np.float32(6 * 2.0 ** e).view(np.uint32)) >> 16
            blocks.append(row)
    for bad in (0x7F80, 0xFF80, 0x7FC0, 0xFFFF, 0x7F81):
        row = rng.integers(0, 0x4100, 32)
        row[rng.integers(32)] = bad
        blocks.append(row)
    return np.array(blocks, np.uint16)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_codes_of_special_blocks(dev, D):
    b = special_blocks()
    b = b[:len(b) // (D // 32) * (D // 32)].reshape(-1, D)
    T, P, H = len(b), 32, 1
    x = torch.from_numpy(np.stack([b, b[::-1]], 1).astype(np.int16).copy()).view(torch.bfloat16)  # [T, 2, D]
    bt, n_pages = tables([T], P, 1, 0)
    pool = kv.kv4_pool(1, n_pages, H, P, D)
    kv.kv4_append(x[None, :, :, None].contiguous().to(dev), i32([0, T], dev), i32(bt, dev), pool, check=True)
    want = np.zeros(pool.shape, np.uint8)
    for kv_ in range(2):
        vals = x[:, kv_].float().numpy()
        for t in range(T):
            R.store(want[0], bt[0, t // P], kv_, 0, t % P, vals[t])
    assert np.array_equal(pool.cpu().numpy(), want)
    k, v = kv.kv4_gather_dequant(pool[0], i32(bt, dev), i32([T], dev), T, check=True)
    for got, kv_ in ((k, 0), (v, 1)):
        w, ok = R.load(want[0], bt[0], T, kv_)
        g = got[0].float().cpu().numpy()
        assert ok.all() and np.array_equal(np.isnan(g), np.isnan(w))
        assert np.array_equal(g[~np.isnan(g)], w[~np.isnan(w)].astype(np.float32))


CASES = [  # lens, old, L, H, D, P, rot, rows behind the last sequence
    ([1], [0], 1, 1, 64, 16, 0, 0), ([1, 1, 1], [5, 0, 33], 3, 8, 128, 16, 128, 0), ([0, 7, 0, 40], [3, 0, 9, 1], 2, 3, 64, 48, 32, 5),
    ([70, 5, 33], [0, 100, 17], 1, 2, 128, 16, 64, 0), ([17], [0], 2, 1, 256, 16, 256, 3), ([64, 31], [0, 0], 1, 5, 128, 32, 112, 1),
    ([20], [3], 1, 2, 256, 32, 16, 0), ([2500, 1, 1700], [0, 90, 11], 4, 8, 128, 16, 128, 2), ([9000], [0], 1, 12, 64, 64, 64, 0),
    ([37], [0], 1, 71, 128, 16, 96, 0)]


def oracle_append(x, bt, lens, old, pool):
    """x [L, T, 2, H, D] torch bf16 (rotated) into pool (numpy): vectorised over tokens."""
    L, _, _, H, D = x.shape
    P = pool.shape[4] * 16
    seq = np.repeat(np.arange(len(lens)), lens)
    pos = np.concatenate([np.arange(a, a + n) for a, n in zip(old, lens)]) if sum(lens) else np.zeros(0, int)
    page, row = bt[seq, pos // P], pos % P
    f = x[:, :len(seq)].float().cpu().numpy()
    for layer in range(L):
        code, byte = R.encode_block(f[layer].reshape(len(seq), 2, H, D // 32, 32))
        packed = code[..., 0::2] | (code[..., 1::2] << 4)  # [T, 2, H, D / 32, 16]
        tiles = pool[layer][..., :8 * D].reshape(*pool.shape[1:5], D // 32, 16, 16).copy()
        tiles[page, :, :, row // 16, :, row % 16] = packed
        pw = pool[layer][..., 8 * D:].reshape(*pool.shape[1:5], D // 32, 16).copy()
        pw[page, :, :, row // 16, :, row % 16] = byte
        pool[layer][..., :8 * D] = tiles.reshape(*pool.shape[1:5], -1)
        pool[layer][..., 8 * D:] = pw.reshape(*pool.shape[1:5], -1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_append_and_gather(dev, case, interleaved):
    lens, old, L, H, D, P, rot, pad = CASES[case]
    interleaved = interleaved and rot > 0
    T = sum(lens)
    total = [a + b for a, b in zip(lens, old)]
    bt, n_pages = tables(total, P, 3, case)
    g = torch.Generator(device=dev).manual_seed(case)
    x = torch.randn((L, T + pad, 2, H, D), generator=g, device=dev).to(torch.bfloat16)
    x *= torch.exp2(torch.randint(-6, 7, (1, 1, 1, 1, D), generator=g, device=dev).float()).to(torch.bfloat16)
    cu, start = i32(np.concatenate([[0], np.cumsum(lens)]), dev), i32(old, dev)
    turned, table = x, None
    if rot:
        table = kv.rope_table(rotary_frequencies(rot)[0].to(dev), max(total) + 1)
        p = i32(np.concatenate([np.arange(a, a + n) for a, n in zip(old, lens)] + [np.zeros(pad)]), dev)
        turned = x.clone()
        for layer in range(L):
            turned[layer, :, 0] = kv.rope(x[layer, :, 0].contiguous(), table, p, interleaved=interleaved)
    pool = torch.randint(0, 256, tuple(kv.kv4_pool(L, n_pages, H, P, D).shape), generator=g, device=dev, dtype=torch.uint8)
    want = pool.cpu().numpy()
    oracle_append(turned, bt, lens, old, want)
    kv.kv4_append(x, cu, i32(bt, dev), pool, start_pos=start, table=table, interleaved=interleaved, check=True)
    assert np.array_equal(pool.cpu().numpy(), want)
    # back: the whole sequences of the last layer, short of them and beyond them
    layer = L - 1
    for out_len in sorted({1, max(total) // 2 + 1, max(total) + 37}):
        k, v = kv.kv4_gather_dequant(pool[layer], i32(bt, dev), i32(total, dev), out_len)
        for got, kv_ in ((k, 0), (v, 1)):
            got = got.float().cpu().numpy()
            for b, n in enumerate(total):
                m = min(n, out_len)
                w, _ = R.load(want[layer], bt[b], m, kv_)
                with np.errstate(over="ignore"):  # (random power bytes: 6 x 2^127 is an infinity in bf16 too)
                    w = w.astype(np.float32)
                np.testing.assert_array_equal(got[b, :, :m], w)
                assert not got[b, :, m:].any()


def test_append_bad_pages_and_positions(dev):
    H, D, P = 2, 64, 16
    bt = np.array([[0, 99, 2], [3, -1, 4]], np.int32)
    x = torch.randn((2, 120, 2, H, D), device=dev).to(torch.bfloat16)
    cu = i32([0, 60, 120], dev)  # 12 positions past each table
    pool = torch.full((2, 5, 2, H, 1, 544), 3, dtype=torch.uint8, device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    kv.kv4_append(x, cu, i32(bt, dev), pool, err=err)
    assert err.item() == N.ZX_KERR_PAGE_RANGE | N.ZX_KERR_POS_RANGE
    assert torch.all(pool[:, 1] == 3)
    good = torch.full_like(pool, 3)
    for b, col, page in ((0, 0, 0), (0, 2, 2), (1, 0, 3), (1, 2, 4)):
        one = x[:, 60 * b + 16 * col:60 * b + 16 * col + 16].contiguous()
        kv.kv4_append(one, i32([0, 16], dev), i32([[page]], dev), good, check=True)
    assert torch.equal(pool, good)
    with pytest.raises(ValueError, match="block table"):
        kv.kv4_append(x, cu, i32(bt, dev), pool, check=True)
    # negative start positions and a table shorter than the sequence
    kv.kv4_append(x[:, :4].contiguous(), i32([0, 4], dev), i32([[1]], dev), pool, start_pos=i32([-2], dev), err=err.zero_())
    assert err.item() == N.ZX_KERR_POS_RANGE
    table = kv.rope_table(rotary_frequencies(64)[0].to(dev), 5)
    before = pool.clone()
    kv.kv4_append(x[:, :9].contiguous(), i32([0, 9], dev), i32([[1]], dev), pool, table=table, err=err.zero_())
    assert err.item() == N.ZX_KERR_POS_RANGE
    changed = (pool != before)[:, 1, ..., :512].reshape(2, 2, H, 2, 16, 16).any(-1)
    assert changed[:, :, :, :, :5].float().mean() > 0.9 and not changed[:, :, :, :, 5:].any()


def test_gather_bad_pages(dev):
    pool = torch.randint(0, 120, (4, 2, 3, 1, 1088), device=dev, dtype=torch.uint8)
    bt = i32([[1, 7, 2], [0, 3, -1]], dev)
    err_free = kv.kv4_gather_dequant(pool, i32([[1, 1, 2], [0, 3, 3]], dev), i32([48, 40], dev), 64)
    k, v = kv.kv4_gather_dequant(pool, bt, i32([48, 40], dev), 64)
    for got, want in zip((k, v), err_free):
        want = want.clone()
        want[0, :, 16:32] = 0
        want[1, :, 32:] = 0
        assert torch.equal(got, want)
    with pytest.raises(ValueError, match="block table"):
        kv.kv4_gather_dequant(pool, bt, i32([48, 40], dev), 64, check=True)
    with pytest.raises(ValueError, match="position"):
        kv.kv4_gather_dequant(pool, i32([[0, 1]], dev), i32([40], dev), 48, check=True)


# ------------------------------------------------------------------ attention

def random_pool(n_pages, H, P, D, seed, spread=3):
    rng = np.random.default_rng(seed)
    pool = rng.integers(0, 256, (n_pages, 2, H, P // 16, 17 * D // 2), dtype=np.uint8)
    pool[..., 8 * D:] = rng.integers(126 - spread, 127, pool[..., 8 * D:].shape)
    return pool


def check_rows(got, want, qk, vm, n, D, sm, weight):
    """got / want [rows, D], qk [rows], vm [D]; n keys; weight: what a weight's rounding costs."""
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    e = (weight + (D + 4) * 2.0 ** -24 * abs(sm) * qk[:, None] + 2.0 ** -21 + (n / 32 + 64) * 2.0 ** -24)
    with np.errstate(invalid="ignore"):
        tol = 2.0 ** -8 * np.abs(want) + 2.1 * e * vm[None] + 2.0 ** -133
        bad = ~nan & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (got[bad][:4], want[bad][:4], np.broadcast_to(tol, got.shape)[bad][:4])


def check_attention(got, q, pool, bt, lens, sm, weight, rows=None, pos0=None, causal=False):
    """got [n_q, Hq, D] against float64; rows[b] rows of sequence b from pos0[b] (decode: one)."""
    n_pages, _, H, tiles, nb = pool.shape
    D, P = nb * 2 // 17, tiles * 16
    got, q = got.double().cpu().numpy(), q.double().cpu().numpy()
    at = 0
    for b, n in enumerate(lens):
        r = 1 if rows is None else rows[b]
        n = max(0, min(int(n), bt.shape[1] * P))
        k, ok = R.load(pool, bt[b], n, 0)
        v, _ = R.load(pool, bt[b], n, 1)
        seen = np.broadcast_to(ok, (r, n))
        if causal:
            seen = seen & (np.arange(n) <= pos0[b] + np.arange(r)[:, None])
        grp = q.shape[1] // H
        for hq in range(q.shape[1]):
            want, qk, vm = R.attend(q[at:at + r, hq], k[hq // grp], v[hq // grp], seen, sm)
            check_rows(got[at:at + r, hq], want, qk, vm, n, D, sm, weight)
        at += r


DECODE = [  # lens, Hq, Hkv, D, P, spare table columns
    ([1], 1, 1, 64, 16, 0), ([0, 5, 16], 8, 2, 128, 16, 1), ([15, 17, 31, 32, 33], 6, 2, 128, 16, 0),
    ([127, 128, 129, 1, 0, 300], 32, 8, 128, 16, 40), ([700], 32, 8, 128, 16, 200), ([2000, 3], 17, 1, 64, 48, 0),
    ([90, 1000], 71, 1, 64, 16, 3), ([333, 64], 12, 12, 64, 32, 0), ([500, 77, 1], 16, 2, 256, 16, 9), ([250] * 5, 3, 1, 256, 64, 0),
    (list(range(1, 100)), 4, 2, 64, 16, 0), ([40] * 70 + [0, 3000], 4, 2, 128, 16, 5), ([4100], 8, 8, 128, 112, 0)]


@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(dev, case):
    lens, Hq, H, D, P, spare = DECODE[case]
    bt, n_pages = tables(lens, P, 2, case)
    bt = np.concatenate([bt, np.full((len(lens), spare), -1, np.int32)], 1)
    pool = random_pool(n_pages, H, P, D, case)
    # beyond a sequence's end a page holds what is not a number: it must not be seen
    for b, n in enumerate(lens):
        if n % 16:
            tile = pool[bt[b, n // P], :, :, (n % P) // 16]
            tile[..., 8 * D:].reshape(2, H, D // 32, 16)[..., n % 16:] = 255
    q = torch.randn((len(lens), Hq, D), device=dev).mul(1.5).to(torch.bfloat16)
    pd, btd, ld = torch.from_numpy(pool).to(dev), i32(bt, dev), i32(lens, dev)
    got = kv.paged_attention4_decode(q, pd, btd, ld, check=True)
    check_attention(got, q, pool, bt, lens, D ** -0.5, 2.0 ** -16)
    out = torch.full_like(q, 3.0)
    assert kv.paged_attention4_decode(q, pd, btd, ld, sm_scale=-0.3, out=out) is out
    check_attention(out, q, pool, bt, lens, -0.3, 2.0 ** -16) if case < 4 else None
    again = kv.paged_attention4_decode(q, pd, btd, ld)
    assert np.array_equal(bits(again), bits(got))


def test_decode_equals_the_gathered_pages(dev):
    """The kernel reads what the gather writes: its error against the gathered bf16 is the same."""
    lens = [100, 37]
    bt, n_pages = tables(lens, 16, 0, 3)
    pool = random_pool(n_pages, 2, 16, 128, 3)
    pd = torch.from_numpy(pool).to(dev)
    k, v = kv.kv4_gather_dequant(pd, i32(bt, dev), i32(lens, dev), 112)
    q = torch.randn((2, 4, 128), device=dev).to(torch.bfloat16)
    got = kv.paged_attention4_decode(q, pd, i32(bt, dev), i32(lens, dev)).double().cpu()
    for b, n in enumerate(lens):
        for hq in range(4):
            s = (q[b, hq].double().cpu() @ k[b, hq // 2, :n].double().cpu().T) * 128 ** -0.5
            want = torch.softmax(s, -1) @ v[b, hq // 2, :n].double().cpu()
            assert torch.all((got[b, hq] - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * 6)


def test_decode_nan_and_bad_pages(dev):
    H, Hq, D, P = 2, 4, 128, 16
    lens = [40, 33, 20, 60]
    bt, n_pages = tables(lens, P, 1, 5)
    pool = random_pool(n_pages, H, P, D, 5)
    pool[bt[0, 1], 0, 0, 0, 8 * D + 3] = 255       # a key's block of (sequence 0, head 0)
    pool[bt[1, 0], 1, 1, 0, 8 * D + 16 * 2 + 5] = 255  # channels 64..96 of a value of (1, head 1)
    bt[2, :] = [n_pages, -1, -7, 2 ** 31 - 1][:1] * bt.shape[1]  # no good page: as an empty sequence
    bt[3, 1] = -1
    q = torch.randn((4, Hq, D), device=dev).to(torch.bfloat16)
    args = (q, torch.from_numpy(pool).to(dev), i32(bt, dev), i32(lens, dev))
    got = kv.paged_attention4_decode(*args)
    assert not got[2].any() and torch.isnan(got[0, :2]).all() and not torch.isnan(got[0, 2:]).any()
    n = torch.isnan(got[1])
    assert n[2:, 64:96].all() and n.sum() == 2 * 32
    with pytest.raises(ValueError, match="block table"):
        kv.paged_attention4_decode(*args, check=True)
    keep = [3]
    check_attention(got[keep], q[keep], pool, bt[keep], [60], D ** -0.5, 2.0 ** -16)
    with pytest.raises(ValueError, match="position"):
        kv.paged_attention4_decode(q[:1], args[1], i32([[0, 1]], dev), i32([33], dev), check=True)
    # a single NaN key makes its row NaN, not zero
    pool[:, 0, :, :, 8 * D:] = 255
    got = kv.paged_attention4_decode(q[:1], torch.from_numpy(pool).to(dev), i32(bt[:1], dev), i32([1], dev))
    assert torch.isnan(got).all()


@pytest.mark.parametrize("Hq, H, D", [(17, 1, 64), (8, 2, 128), (16, 2, 256)])
def test_attention_repeats_to_the_bit(dev, Hq, H, D):
    """Every call gives the same bits, decode and prefill (a product's result read before it is
    complete would now and then change a running maximum, and with it the last bits)."""
    lens, rows, P = [2000, 3, 700], [40, 3, 5], 16
    bt, n_pages = tables(lens, P, 0, 5)
    pool = torch.from_numpy(random_pool(n_pages, H, P, D, 5)).to(dev)
    btd, ld = i32(bt, dev), i32(lens, dev)
    q = torch.randn((sum(rows), Hq, D), device=dev).mul(2).to(torch.bfloat16)
    cu, pos0 = i32(np.concatenate([[0], np.cumsum(rows)]), dev), i32([n - r for n, r in zip(lens, rows)], dev)

    def both(precision):
        return (kv.paged_attention4_decode(q[:3], pool, btd, ld),
                kv.paged_attention4_prefill(q, cu, pos0, pool, btd, ld, max_q_per_seq=40, precision=precision),
                kv.paged_attention4_prefill(q[:2], i32([0, 2, 2, 2], dev), pos0, pool, btd, ld, max_q_per_seq=2))
    for precision in ("bf16", "exact"):
        want = both(precision)
        for _ in range(30):
            assert all(torch.equal(a, b) for a, b in zip(both(precision), want))


PREFILL = [  # rows, tokens before, Hq, Hkv, D, P, causal
    ([1], [0], 1, 1, 64, 16, True), ([3, 0, 5], [10, 4, 0], 4, 2, 128, 16, True), ([4, 1, 2], [500, 1000, 31], 32, 8, 128, 16, True),
    ([40, 17], [0, 90], 4, 1, 128, 32, True), ([130], [60], 8, 8, 64, 16, True), ([33, 64], [100, 0], 6, 2, 256, 16, True),
    ([20, 7], [40, 200], 4, 2, 128, 16, False), ([100, 3], [3, 900], 17, 1, 64, 48, True), ([8], [3000], 8, 1, 128, 16, True),
    ([70, 1], [0, 0], 71, 1, 64, 16, True), ([5], [1500], 4, 4, 256, 16, False), ([200], [0], 3, 1, 128, 112, True)]


@pytest.mark.parametrize("precision", ["bf16", "exact"])
@pytest.mark.parametrize("case", range(len(PREFILL)))
def test_prefill(dev, case, precision):
    rows, old, Hq, H, D, P, causal = PREFILL[case]
    lens = [a + b for a, b in zip(rows, old)]
    bt, n_pages = tables(lens, P, 2, case + 50)
    pool = random_pool(n_pages, H, P, D, case)
    for b, n in enumerate(lens):
        if n % 16:
            tile = pool[bt[b, n // P], :, :, (n % P) // 16]
            tile[..., 8 * D:].reshape(2, H, D // 32, 16)[..., n % 16:] = 255
    pad = 3  # rows behind the last sequence
    q = torch.randn((sum(rows) + pad, Hq, D), device=dev).mul(1.5).to(torch.bfloat16)
    cu = i32(np.concatenate([[0], np.cumsum(rows)]), dev)
    args = (q, cu, i32(old, dev), torch.from_numpy(pool).to(dev), i32(bt, dev), i32(lens, dev))
    out = torch.full_like(q, 5.0)
    kv.paged_attention4_prefill(*args, causal=causal, precision=precision, out=out, check=True)
    assert torch.all(out[sum(rows):] == 5)
    weight = 2.0 ** -16 if precision == "exact" else 2.0 ** -8
    check_attention(out[:sum(rows)], q, pool, bt, lens, D ** -0.5, weight, rows, old, causal)
    # a loose bound on the rows changes tiles, not results; nor does running uncut
    loose = torch.full_like(q, 5.0)
    kv.paged_attention4_prefill(*args, causal=causal, precision=precision, out=loose, max_q_per_seq=max(rows) + 100, check=True)
    check_attention(loose[:sum(rows)], q, pool, bt, lens, D ** -0.5, weight, rows, old, causal)
    uncut = torch.full_like(q, 5.0)
    lib = N.load()
    N.check(lib.zx_paged_attention4_prefill(
        q.data_ptr(), q.shape[0], cu.data_ptr(), args[2].data_ptr(), Hq, args[3].data_ptr(), n_pages, H, D, P,
        args[4].data_ptr(), bt.shape[1], args[5].data_ptr(), len(rows), max(rows), int(causal), D ** -0.5,
        N.ZX_PREFILL_EXACT_P if precision == "exact" else 0, uncut.data_ptr(), None, None, 0, N.stream_ptr(dev)), "uncut")
    check_attention(uncut[:sum(rows)], q, pool, bt, lens, D ** -0.5, weight, rows, old, causal)
    assert torch.all(uncut[sum(rows):] == 5)


def test_prefill_rows_without_keys_and_errors(dev):
    H, Hq, D, P = 2, 4, 64, 16
    bt, n_pages = tables([64, 64, 64], P, 0, 9)
    pool = random_pool(n_pages, H, P, D, 9)
    q = torch.randn((30, Hq, D), device=dev).to(torch.bfloat16)
    cu, pd, btd = i32([0, 10, 20, 30], dev), torch.from_numpy(pool).to(dev), i32(bt, dev)
    # positions below 0 see nothing, a sequence without keys neither; rows past the keys see them all
    pos0, lens = [-5, 0, 100], [40, 0, 30]
    got = kv.paged_attention4_prefill(q, cu, i32(pos0, dev), pd, btd, i32(lens, dev), check=True)
    assert not got[:5].any() and not got[10:20].any() and got[5:10].any()
    check_attention(got, q, pool, bt, lens, D ** -0.5, 2.0 ** -8, [10, 10, 10], pos0, True)
    out = torch.full_like(q, 5.0)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    kv.paged_attention4_prefill(q, cu, i32([20, 20, 20], dev), pd, btd, i32([30, 30, 30], dev), max_q_per_seq=8, out=out, err=err)
    assert err.item() == N.ZX_KERR_POS_RANGE  # two rows of each sequence are not computed
    rows = out.view(3, 10, Hq, D)
    assert torch.all(rows[:, 8:] == 5) and not (rows[:, :8] == 5).all(-1).any()
    bad = bt.copy()
    bad[1, 1] = n_pages
    with pytest.raises(ValueError, match="block table"):
        kv.paged_attention4_prefill(q, cu, i32([20] * 3, dev), pd, i32(bad, dev), i32([30] * 3, dev), check=True)
    with pytest.raises(ValueError, match="position"):
        kv.paged_attention4_prefill(q, cu, i32([60] * 3, dev), pd, btd, i32([70] * 3, dev), check=True)
    empty = kv.paged_attention4_prefill(q[:0], i32([0, 0, 0, 0], dev), i32(pos0, dev), pd, btd, i32(lens, dev))
    assert empty.shape == (0, Hq, D)


def test_prefill_nan_reaches_only_rows_that_see_it(dev):
    """A NaN key or value at position 25 of 40: rows before it are as without it."""
    H, Hq, D, P, n = 1, 2, 128, 16, 40
    bt, n_pages = tables([n], P, 0, 4)
    clean = random_pool(n_pages, H, P, D, 4)
    q = torch.randn((n, Hq, D), device=dev).to(torch.bfloat16)

    def run(pool):
        return kv.paged_attention4_prefill(q, i32([0, n], dev), i32([0], dev), torch.from_numpy(pool).to(dev), i32(bt, dev),
                                           i32([n], dev), precision="exact")
    want = run(clean)
    for kv_ in range(2):
        pool = clean.copy()
        pool[bt[0, 1], kv_, 0, 0, 8 * D + 16 * 3 + 9] = 255  # block 3 (channels 96..128) of position 25
        got = run(pool)
        assert torch.isnan(got[25:]).any(-1).all() and torch.equal(got[:25], want[:25])
        if kv_:  # in its channels only
            assert torch.equal(got[..., :96], want[..., :96]) and torch.isnan(got[25:, :, 96:]).all()


@pytest.mark.parametrize("precision", ["bf16", "exact"])
@pytest.mark.parametrize("rows, old, Hq, H, D", [([70], [9], 4, 2, 128), ([130], [40], 2, 2, 64), ([50], [3], 1, 1, 256),
                                                 ([3, 2], [40, 17], 6, 2, 128), ([20], [0], 8, 4, 64)])
def test_prefill_nan_values(dev, rows, old, Hq, H, D, precision):
    """NaN blocks in every tenth position's values: NaN in the rows that see them, in their
    channels, and the oracle's numbers everywhere else."""
    P = 16
    lens = [a + b for a, b in zip(rows, old)]
    bt, n_pages = tables(lens, P, 0, D)
    pool = random_pool(n_pages, H, P, D, D)
    rng = np.random.default_rng(D)
    for b, n in enumerate(lens):
        for pos in range(n - min(rows[b], 40), n, 7):
            pool[bt[b, pos // P], 1, rng.integers(H), 0, 8 * D + 16 * rng.integers(D // 32) + pos % 16] = 255
    q = torch.randn((sum(rows), Hq, D), device=dev).to(torch.bfloat16)
    cu = i32(np.concatenate([[0], np.cumsum(rows)]), dev)
    got = kv.paged_attention4_prefill(q, cu, i32(old, dev), torch.from_numpy(pool).to(dev), i32(bt, dev), i32(lens, dev),
                                      precision=precision).double().cpu().numpy()
    qn, at = q.double().cpu().numpy(), 0
    for b, n in enumerate(lens):
        k, v = R.load(pool, bt[b], n, 0)[0], R.load(pool, bt[b], n, 1)[0]
        for r in range(rows[b]):
            see = old[b] + r + 1
            for hq in range(Hq):
                vh = v[hq * H // Hq][:see]
                bad = np.isnan(vh).any(0)
                assert np.array_equal(np.isnan(got[at + r, hq]), bad), (b, r, hq)
                want, qk, vm = R.attend(qn[at + r:at + r + 1, hq], k[hq * H // Hq][:see], np.nan_to_num(vh),
                                        np.ones((1, see), bool), D ** -0.5)
                ok = ~bad
                check_rows(got[at + r:at + r + 1, hq][:, ok], want[:, ok], qk, vm[ok], see, D, D ** -0.5,
                           2.0 ** -16 if precision == "exact" else 2.0 ** -8)
        at += rows[b]


@pytest.mark.parametrize("precision", ["bf16", "exact"])
@pytest.mark.parametrize("Hq, H, D, P", [(16, 16, 64, 16), (30, 15, 128, 32), (8, 8, 256, 16)])
def test_prefill_of_many_tiles_with_few_keys(dev, Hq, H, D, P, precision):
    """So many tiles of so few steps (at most 4) that every wave takes one by itself; with NaN
    values in one sequence, rows without keys, and rows behind the last."""
    rng = np.random.default_rng(D)
    rows = rng.integers(50, 90, 24).tolist()
    rows[5], rows[9] = 0, 1
    old = [int(rng.integers(0, 120 - r)) for r in rows]
    old[3] = -7  # its first rows see nothing
    lens = [a + b for a, b in zip(rows, old)]
    lens[7] = 0
    bt, n_pages = tables(lens, P, 1, 4)
    pool = random_pool(n_pages, H, P, D, 4)
    b, pos = 11, lens[11] - 20
    pool[bt[b, pos // P], 1, 2, pos % P // 16, 8 * D + pos % 16] = 255  # block 0 of kv head 2
    q = torch.randn((sum(rows) + 2, Hq, D), device=dev).to(torch.bfloat16)
    out = torch.full_like(q, 5.0)
    cu = np.concatenate([[0], np.cumsum(rows)])
    kv.paged_attention4_prefill(q, i32(cu, dev), i32(old, dev), torch.from_numpy(pool).to(dev), i32(bt, dev),
                                i32(lens, dev), precision=precision, out=out, check=True)
    assert torch.all(out[sum(rows):] == 5) and not out[cu[7]:cu[8]].any() and not out[cu[3]:cu[3] + 7].any()
    weight = 2.0 ** -16 if precision == "exact" else 2.0 ** -8
    hit = out[cu[b]:cu[b + 1]]
    grp = Hq // H
    seen = torch.isnan(hit)
    first = pos - old[b]
    assert seen[first:, 2 * grp:3 * grp, :32].all() and seen.sum() == (rows[b] - first) * grp * 32
    check = [i for i in range(24) if i != b]
    keep = torch.cat([torch.arange(cu[i], cu[i + 1]) for i in check]).to(dev)
    check_attention(out[keep], q[keep], pool, bt[check], [lens[i] for i in check], D ** -0.5, weight,
                    [rows[i] for i in check], [old[i] for i in check], True)


def test_prefill_flags_of_sequences_without_rows(dev):
    """A sequence that computes no row but claims more keys than its table holds is flagged
    wherever its tiles fall (one tile per sequence and head, a wave each)."""
    H, D, P = 1, 64, 16
    pool = kv.kv4_pool(1, 64, H, P, D)
    bt = torch.arange(64, dtype=torch.int32, device=dev)[:, None].contiguous()
    for rows_of, bad in ((70, 1), (70, 2), (70, 3), (70, 62)):
        rows = [0 if b == bad else rows_of for b in range(63)]
        q = torch.zeros((sum(rows), 1, D), dtype=torch.bfloat16, device=dev)
        lens = [17 if b == bad else 16 for b in range(63)]
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        kv.paged_attention4_prefill(q, i32(np.concatenate([[0], np.cumsum(rows)]), dev), i32([0] * 63, dev), pool[0],
                                    bt[:63], i32(lens, dev), max_q_per_seq=rows_of, err=err)
        assert err.item() == N.ZX_KERR_POS_RANGE, bad


def test_prefill_of_many_short_sequences(dev):
    """More than 64 sequences of 0 to 6 rows: dealt by a table, in runs and whole."""
    H, Hq, D, P = 2, 8, 128, 16
    rng = np.random.default_rng(2)
    for n_seqs, longest in ((70, 900), (65, 60)):
        rows = rng.integers(0, 7, n_seqs).tolist()
        old = rng.integers(0, longest, n_seqs).tolist()
        lens = [a + b for a, b in zip(rows, old)]
        bt, n_pages = tables(lens, P, 0, 1)
        pool = random_pool(n_pages, H, P, D, 1)
        q = torch.randn((sum(rows) + 1, Hq, D), device=dev).to(torch.bfloat16)
        out = torch.full_like(q, 5.0)
        cu = i32(np.concatenate([[0], np.cumsum(rows)]), dev)
        kv.paged_attention4_prefill(q, cu, i32(old, dev), torch.from_numpy(pool).to(dev), i32(bt, dev), i32(lens, dev),
                                    precision="exact", out=out, check=True)
        assert torch.all(out[-1] == 5)
        check_attention(out, q, pool, bt, lens, D ** -0.5, 2.0 ** -16, rows, old, True)


@pytest.mark.parametrize("n_seqs, most, Hq, H, D", [(66, 60, 2, 2, 128), (66, 90, 2, 1, 64), (260, 2, 16, 16, 128),
                                                    (70, 20, 1, 1, 256), (130, 3, 32, 32, 64)])
def test_prefill_of_more_than_64_sequences_in_tiles(dev, n_seqs, most, Hq, H, D):
    """Several tiles per sequence, or so many of one that they are not dealt in runs."""
    rng = np.random.default_rng(n_seqs + D)
    rows = rng.integers(0, most + 1, n_seqs).tolist()
    rows[1] = most
    old = rng.integers(0, 40, n_seqs).tolist()
    lens = [a + b for a, b in zip(rows, old)]
    bt, n_pages = tables(lens, 16, 0, 1)
    pool = random_pool(n_pages, H, 16, D, 1)
    q = torch.randn((sum(rows) + 1, Hq, D), device=dev).to(torch.bfloat16)
    out = torch.full_like(q, 5.0)
    cu = i32(np.concatenate([[0], np.cumsum(rows)]), dev)
    kv.paged_attention4_prefill(q, cu, i32(old, dev), torch.from_numpy(pool).to(dev), i32(bt, dev), i32(lens, dev),
                                precision="exact", out=out, max_q_per_seq=most, check=True)
    assert torch.all(out[-1] == 5)
    check_attention(out, q, pool, bt, lens, D ** -0.5, 2.0 ** -16, rows, old, True)


@pytest.mark.parametrize("sm", [0.0, -0.3, 1e-6, 4.0])
def test_prefill_scales(dev, sm):
    for rows, old, Hq, H, D in (([3, 1], [90, 20], 4, 2, 128), ([60], [10], 4, 4, 64)):
        lens = [a + b for a, b in zip(rows, old)]
        bt, n_pages = tables(lens, 16, 0, 3)
        pool = random_pool(n_pages, H, 16, D, 3)
        q = torch.randn((sum(rows), Hq, D), device=dev).to(torch.bfloat16)
        cu = i32(np.concatenate([[0], np.cumsum(rows)]), dev)
        got = kv.paged_attention4_prefill(q, cu, i32(old, dev), torch.from_numpy(pool).to(dev), i32(bt, dev),
                                          i32(lens, dev), sm_scale=sm, precision="exact", check=True)
        check_attention(got, q, pool, bt, lens, sm, 2.0 ** -16, rows, old, True)


@pytest.mark.parametrize("n, most, Hq, H", [(70, 50, 4, 4), (70, 70, 4, 1), (6, 4, 8, 2)])
def test_prefill_computes_no_other_rows(dev, n, most, Hq, H):
    """Rows beyond max_q_per_seq, and rows that cu_q claims and q does not have."""
    D, P = 128, 16
    bt, n_pages = tables([n + 30], P, 0, 6)
    pool = random_pool(n_pages, H, P, D, 6)
    back = torch.randn((n + 40, Hq, D), device=dev).to(torch.bfloat16)
    for claimed in (n, n + 30):
        out = torch.full_like(back, 5.0)
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        kv.paged_attention4_prefill(back[:n], i32([0, claimed], dev), i32([20], dev), torch.from_numpy(pool).to(dev),
                                    i32(bt, dev), i32([n + 20], dev), max_q_per_seq=most, out=out[:n], err=err)
        assert torch.all(out[most:] == 5) and err.item() == (N.ZX_KERR_POS_RANGE if claimed > most else 0)
        check_attention(out[:most], back, pool, bt, [n + 20], D ** -0.5, 2.0 ** -8, [most], [20], True)


def test_a_pool_beyond_2_gib(dev):
    """Pages whose offsets pass 31 and 32 bits: append, gather and both attentions."""
    H, Hq, D, P, n = 8, 8, 128, 16, 90
    n_pages = 260_000  # 17 KiB each
    ids = [n_pages - 1, 0, 123_361, 123_362, 246_723, 246_724]
    x = torch.randn((1, n, 2, H, D), device=dev).to(torch.bfloat16)
    q = torch.randn((n, Hq, D), device=dev).to(torch.bfloat16)
    cu, lens, zero = i32([0, n], dev), i32([n], dev), i32([0], dev)

    def run(pool, bt):
        kv.kv4_append(x, cu, bt, pool, check=True)
        return (*kv.kv4_gather_dequant(pool[0], bt, lens, n, check=True),
                kv.paged_attention4_decode(q[:1], pool[0], bt, lens, check=True),
                kv.paged_attention4_prefill(q, cu, zero, pool[0], bt, lens, max_q_per_seq=n, check=True),
                kv.paged_attention4_prefill(q[:2], i32([0, 2], dev), i32([n - 2], dev), pool[0], bt, lens, max_q_per_seq=2))
    want = run(kv.kv4_pool(1, 6, H, P, D), i32([list(range(6))], dev))
    got = run(torch.empty((1, n_pages, 2, H, 1, 17 * D // 2), dtype=torch.uint8, device=dev), i32([ids], dev))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_append_of_nothing(dev):
    pool = kv.kv4_pool(1, 2, 2, 16, 64)
    x = torch.zeros((1, 0, 2, 2, 64), dtype=torch.bfloat16, device=dev)
    kv.kv4_append(x, i32([0, 0], dev), i32([[0, 1]], dev), pool, check=True)
    assert not pool.any()
    k, v = kv.kv4_gather_dequant(pool[0], i32([[0, 1]], dev), i32([0], dev), 0)
    assert k.shape == v.shape == (1, 2, 0, 64)


def test_two_calls_at_once(dev):
    """Calls on two streams, workspaces and all, do not meet."""
    Hq, H, D, P = 32, 8, 128, 16
    made = []
    for seed in range(2):
        lens = [3000 + 500 * seed, 100]
        bt, n_pages = tables(lens, P, 0, seed)
        pool = random_pool(n_pages, H, P, D, seed)
        q = torch.randn((2, Hq, D), device=dev).to(torch.bfloat16)
        made.append((q, torch.from_numpy(pool).to(dev), i32(bt, dev), i32(lens, dev)))
    want = [kv.paged_attention4_decode(*a) for a in made]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in made], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kv.paged_attention4_decode(*made[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for w, many in zip(want, got) for g in many)


def test_refusals(dev):
    pool, bt, lens = kv.kv4_pool(1, 4, 2, 16, 64), i32([[0, 1]], dev), i32([5], dev)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=dev)
    x = torch.zeros((1, 5, 2, 2, 64), dtype=torch.bfloat16, device=dev)
    cu = i32([0, 5], dev)
    table = kv.rope_table(rotary_frequencies(128)[0].to(dev), 5)
    for bad in (lambda: kv.kv4_pool(1, 4, 2, 24, 64), lambda: kv.kv4_pool(1, 4, 2, 16, 96), lambda: kv.kv4_pool(1, 4, 2, 0, 64),
                lambda: kv.kv4_append(x.half(), cu, bt, pool), lambda: kv.kv4_append(x, cu, bt, pool[..., :500]),
                lambda: kv.kv4_append(x, cu, bt, kv.kv4_pool(1, 4, 3, 16, 64)), lambda: kv.kv4_append(x, cu, bt, pool, table=table),
                lambda: kv.kv4_append(x, cu, bt, pool, interleaved=True), lambda: kv.kv4_append(x, cu.long(), bt, pool),
                lambda: kv.kv4_append(x, cu, bt.cpu(), pool), lambda: kv.kv4_append(x[..., :32], cu, bt, pool),
                lambda: kv.kv4_gather_dequant(pool, bt, lens), lambda: kv.kv4_gather_dequant(pool[0], bt, lens.long()),
                lambda: kv.kv4_gather_dequant(pool[0], bt, i32([1, 2], dev)),
                lambda: kv.paged_attention4_decode(q.float(), pool[0], bt, lens),
                lambda: kv.paged_attention4_decode(q[:, :3], pool[0], bt, lens),
                lambda: kv.paged_attention4_decode(q[..., :32], pool[0], bt, lens),
                lambda: kv.paged_attention4_decode(q, pool[0], bt, i32([1, 2], dev)),
                lambda: kv.paged_attention4_decode(q, pool[0], bt, lens, out=q.float()),
                lambda: kv.paged_attention4_prefill(q, cu, lens, pool[0], bt, lens, precision="f16"),
                lambda: kv.paged_attention4_prefill(q, lens, lens, pool[0], bt, lens),
                lambda: kv.paged_attention4_prefill(q, cu, lens.long(), pool[0], bt, lens),
                lambda: PagedFP4KVCache(1, 2, 64, 4, page_size=8), lambda: PagedFP4KVCache(1, 2, 80, 4)):
        with pytest.raises(ValueError):
            bad()


def test_streams_and_graphs(dev):
    """On another stream, and two captured graphs replayed in turn with eager work between."""
    lens, Hq, H, D, P = [700, 20, 333], 8, 2, 128, 16
    bt, n_pages = tables(lens, P, 0, 8)
    pd, btd, ld = torch.from_numpy(random_pool(n_pages, H, P, D, 8)).to(dev), i32(bt, dev), i32(lens, dev)
    q = torch.randn((3, Hq, D), device=dev).to(torch.bfloat16)
    cu, pos0 = i32([0, 1, 2, 3], dev), i32([n - 1 for n in lens], dev)

    def both():
        return (kv.paged_attention4_decode(q, pd, btd, ld),
                kv.paged_attention4_prefill(q, cu, pos0, pd, btd, ld, max_q_per_seq=1))
    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(np.array_equal(bits(a), bits(b)) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both())
        graphs.append(g)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=dev))
        for g in graphs:
            g.replay()
        want = both()
        torch.cuda.synchronize()
        for o in outs:
            assert all(np.array_equal(bits(a), bits(b)) for a, b in zip(o, want))


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("interleaved, rot", [(False, 128), (True, 64)])
def test_a_cache_that_rotates(dev, four, interleaved, rot):
    """Prompts, a chunk on top, decode steps, a freed sequence: keys rotated while stored and
    queries on their way, against the same cache given rotated keys and queries."""
    L, H, Hq, D = 2, 2, 8, 128
    rope = RotaryPositions(D, 400, rotary_dim=rot, interleaved=interleaved)
    make = (lambda r: PagedFP4KVCache(L, H, D, 60, rope=r)) if four else (lambda r: PagedFP8KVCache(L, H, D, 60, rope=r))
    cache, plain = make(rope), make(None)
    att, ref = QuantizedRingAttention(cache, ring_degree=2), QuantizedRingAttention(plain, ring_degree=2)
    g = torch.Generator(device=dev).manual_seed(rot)

    def step(seqs, lens, decode):
        x = torch.randn((L, sum(lens), 2, H, D), generator=g, device=dev).clamp(-3, 3).to(torch.bfloat16)
        start = [cache.lengths.get(s, 0) for s in seqs]
        p = torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in zip(start, lens)]).to(dev)
        turned = x.clone()
        for layer in range(L):
            turned[layer, :, 0] = rope(x[layer, :, 0].contiguous(), p)
        if four:
            cache.append(x, seqs, lens, check=True)
            plain.append(turned, seqs, lens, check=True)
        else:
            cache.overflow = plain.overflow = "saturate"
            cache.append(x, seqs, lens, check=True)
            plain.append(turned, seqs, lens, check=True)
        assert torch.equal(cache.pool, plain.pool)
        q = torch.randn((sum(lens), Hq, D), generator=g, device=dev).to(torch.bfloat16)
        for layer in range(L):
            got = att.decode(q, layer, seqs) if decode else att(q, layer, seqs, lens)
            want = ref.decode(rope(q, p), layer, seqs) if decode else ref(rope(q, p), layer, seqs, lens)
            assert np.array_equal(bits(got), bits(want))
    step(["a", "b"], [100, 33], False)
    step(["b"], [50], False)
    for _ in range(3):
        step(["b", "a"], [1, 1], True)
    cache.free("a")
    plain.free("a")
    step(["c", "b"], [1, 17], False)
    k, v = cache.gather(1, ["b", "c"])
    assert k.shape == (2, H, cache.lengths["b"], D) and not k[1, :, 1:].any()
    with pytest.raises(ValueError, match="positions"):
        cache.append(torch.zeros((L, 400, 2, H, D), dtype=torch.bfloat16, device=dev), ["c"], [400])
    assert cache.lengths["c"] == 1


def test_4_bit_attention_against_float64_end_to_end(dev):
    """Append, then attend: every row against float64 on what the oracle says the pages hold."""
    L, H, Hq, D = 1, 2, 6, 64
    cache = PagedFP4KVCache(L, H, D, 20, page_size=32)
    att = QuantizedRingAttention(cache, precision="exact")
    x = torch.randn((L, 150, 2, H, D), device=dev).to(torch.bfloat16)
    cache.append(x, [0, 1], [100, 50], check=True)
    q = torch.randn((150, Hq, D), device=dev).to(torch.bfloat16)
    got = att(q, 0, [0, 1], [100, 50])
    code, byte = R.encode_block(x[0].float().cpu().numpy().reshape(150, 2, H, 2, 32))
    held = R.decode_block(code, byte).reshape(150, 2, H, D)
    for lo, hi in ((0, 100), (100, 150)):
        n = hi - lo
        seen = np.arange(n) <= np.arange(n)[:, None]
        for hq in range(Hq):
            want, qk, vm = R.attend(q[lo:hi, hq].double().cpu().numpy(), held[lo:hi, 0, hq // 3], held[lo:hi, 1, hq // 3], seen,
                                    D ** -0.5)
            check_rows(got[lo:hi, hq].double().cpu().numpy(), want, qk, vm, n, D, D ** -0.5, 2.0 ** -16)
    one = att.decode(q[:2], 0, [1, 0])
    assert one.shape == (2, Hq, D) and torch.isfinite(one).all()
    with pytest.raises(ValueError):
        cache.append(x, [0], [10])


def test_prefill_keeps_its_weights_unless_told(dev):
    """The default, and what QuantizedRingAttention's precisions become: "f16" and "exact" the weights to
    2^-17, "bf16" those of one rounding."""
    H, Hq, D, n = 2, 8, 128, 90
    cache = PagedFP4KVCache(1, H, D, 20)
    cache.append(torch.randn((1, n, 2, H, D), device=dev).to(torch.bfloat16), [0], [n], check=True)
    q = torch.randn((n, Hq, D), device=dev).mul(3).to(torch.bfloat16)
    pool, bt, lens = cache.pool[0], cache._tables([0]), cache._lengths([0])
    args = (q, i32([0, n], dev), i32([0], dev), pool, bt, lens)
    exact, one = (kv.paged_attention4_prefill(*args, max_q_per_seq=n, precision=p) for p in ("exact", "bf16"))
    assert not torch.equal(exact, one)
    check_attention(exact, q, pool.cpu().numpy(), bt.cpu().numpy(), [n], D ** -0.5, 2.0 ** -16, [n], [0], True)
    assert torch.equal(kv.paged_attention4_prefill(*args, max_q_per_seq=n), exact)
    for precision, want in (("f16", exact), ("exact", exact), ("bf16", one)):
        assert torch.equal(QuantizedRingAttention(cache, precision=precision)(q, 0, [0], [n]), want), precision
    assert torch.equal(QuantizedRingAttention(cache)(q, 0, [0], [n]), exact)


@pytest.mark.parametrize("other", [40, 1000])  # the other sequence's keys: sequences are taken whole, or in runs
@pytest.mark.parametrize("n_seqs", [2, 70])
@pytest.mark.parametrize("claim", [2, 3, 9])
def test_flags_of_sequences_without_keys(dev, other, n_seqs, claim):
    """A few rows per sequence, dealt in runs: a sequence without keys that claims rows beyond
    max_q_per_seq (2), or rows that q does not have, is flagged as any other, and its two rows are zeros."""
    H, Hq, D, P = 2, 4, 64, 16
    bt, n_pages = tables([1024] * 2 + [16] * (n_seqs - 2), P, 0, 1)
    bt[1, other // P + 1:] = -1
    pool = torch.from_numpy(random_pool(n_pages, H, P, D, 1)).to(dev)
    for empty, length in ((0, 0), (1, -3), (n_seqs - 1, 0)):
        lens = [other] + [16] * (n_seqs - 1)
        lens[empty] = length
        rows = [2] * n_seqs
        rows[empty] = claim
        cu = np.concatenate([[0], np.cumsum(rows)])
        n_q = int(cu[-1])
        missing = claim == 9 and empty == n_seqs - 1  # rows that q does not have
        q = torch.randn((n_q - 7 if missing else n_q, Hq, D), device=dev).to(torch.bfloat16)
        out = torch.full_like(q, 5.0)
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        kv.paged_attention4_prefill(q, i32(cu, dev), i32([2000] * n_seqs, dev), pool, i32(bt, dev), i32(lens, dev),
                                    max_q_per_seq=2, out=out, err=err)
        assert err.item() == (N.ZX_KERR_POS_RANGE if claim > 2 else 0), (empty, length)
        at = int(cu[empty])
        assert not out[at:at + 2].any() and torch.all(out[at + 2:int(cu[empty + 1])] == 5)
        assert torch.isfinite(out).all() and not (out[:2] == 5).any()


@pytest.mark.parametrize("sm", [-0.3, 0.0, 0.7, -1e-6])
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode_scales_into_the_callers_buffer(dev, case, sm):
    """Every shape's values under scales of either sign and zero (then each sequence's mean), in a buffer
    that held something else."""
    lens, Hq, H, D, P, spare = DECODE[case]
    bt, n_pages = tables(lens, P, 2, case)
    bt = np.concatenate([bt, np.full((len(lens), spare), -1, np.int32)], 1)
    pool = random_pool(n_pages, H, P, D, case + 100)
    q = torch.randn((len(lens), Hq, D), device=dev).mul(1.5).to(torch.bfloat16)
    out = torch.full_like(q, 3.0)
    got = kv.paged_attention4_decode(q, torch.from_numpy(pool).to(dev), i32(bt, dev), i32(lens, dev), sm_scale=sm,
                                     out=out, check=True)
    assert got is out
    check_attention(out, q, pool, bt, lens, sm, 2.0 ** -16)


@pytest.mark.parametrize("n_seqs", [255, 256, 257, 258, 700])
@pytest.mark.parametrize("longest", [1, 40])
def test_append_of_many_sequences(dev, n_seqs, longest):
    """Either side of the 256 sequences whose table fits the kernels' LDS, few tokens (found in the append
    itself) and more (found by a launch before it), empty sequences among them, rotating."""
    L, H, D, P, rot = 2, 2, 64, 16, 32
    rng = np.random.default_rng(n_seqs + longest)
    lens = rng.integers(0, longest + 1, n_seqs)
    lens[[0, -1]] = 0, longest
    old = rng.integers(0, 30, n_seqs)
    T = int(lens.sum())
    bt, n_pages = tables(lens + old, P, 2, 1)
    x = torch.randn((L, T + 1, 2, H, D), device=dev).to(torch.bfloat16)
    table = kv.rope_table(rotary_frequencies(rot)[0].to(dev), int((lens + old).max()) + 1)
    pos = i32(np.concatenate([np.arange(a, a + n) for a, n in zip(old, lens)]), dev)
    turned = x.clone()
    for layer in range(L):
        turned[layer, :T, 0] = kv.rope(x[layer, :T, 0].contiguous(), table, pos)
    cu, start = i32(np.concatenate([[0], np.cumsum(lens)]), dev), i32(old, dev)
    pool = torch.randint(0, 256, tuple(kv.kv4_pool(L, n_pages, H, P, D).shape), device=dev, dtype=torch.uint8)
    want = pool.cpu().numpy()
    oracle_append(turned, bt, lens, old, want)
    kv.kv4_append(x, cu, i32(bt, dev), pool, start_pos=start, table=table, check=True)
    assert np.array_equal(pool.cpu().numpy(), want)
    # the FP8 append that rotates, against the one that takes rotated keys
    a, b = (torch.zeros((L, n_pages, 2, H, P, D), dtype=torch.uint8, device=dev) for _ in range(2))
    got = kv.kv_rope_append(x, table, cu, i32(bt, dev), a, start_pos=start, check=True)
    assert torch.equal(got, kv.kv_quant_append(turned[:, :T].contiguous(), cu, i32(bt, dev), b, start_pos=start, check=True))
    assert torch.equal(a, b)


def test_append_and_gather_in_a_graph(dev):
    """Captured appends and gathers, small and large ones (with a workspace each), replay to the eager bits."""
    H, D, P = 2, 128, 16
    for lens, old in (([3, 1], [5, 40]), ([6000, 11000], [0, 9])):
        total = [a + b for a, b in zip(lens, old)]
        bt, n_pages = tables(total, P, 0, 2)
        btd, cu, start, ld = i32(bt, dev), i32([0, lens[0], sum(lens)], dev), i32(old, dev), i32(total, dev)
        table = kv.rope_table(rotary_frequencies(D)[0].to(dev), max(total))
        x = torch.randn((1, sum(lens), 2, H, D), device=dev).to(torch.bfloat16)
        graphs, outs = [], []
        kv.kv4_append(x, cu, btd, kv.kv4_pool(1, n_pages, H, P, D), start_pos=start, table=table)
        for _ in range(2):
            pool, g = kv.kv4_pool(1, n_pages, H, P, D), torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                kv.kv4_append(x, cu, btd, pool, start_pos=start, table=table)
                outs.append((pool, *kv.kv4_gather_dequant(pool[0], btd, ld, max(total))))
            graphs.append(g)
        for _ in range(3):
            x.copy_(torch.randn(x.shape, device=dev))
            for g in graphs:
                g.replay()
            want = kv.kv4_pool(1, n_pages, H, P, D)
            kv.kv4_append(x, cu, btd, want, start_pos=start, table=table)
            k, v = kv.kv4_gather_dequant(want[0], btd, ld, max(total))
            torch.cuda.synchronize()
            for o in outs:
                assert all(torch.equal(a, b) for a, b in zip(o, (want, k, v)))
