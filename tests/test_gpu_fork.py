"""GPU sequences that share pages (PagedFP8KVCache.fork), and the attention that reads the shared pages
once: the rows of a cache whose sequences were appended whole."""
import pytest
import torch

from zenyx_amd import kv
from zenyx_amd.train.cross_attention import CrossAttention
from zenyx_amd.train.fp8_kv_quantization import PagedFP4KVCache, PagedFP8KVCache, QuantizedRingAttention
from zenyx_amd.train.rotary import RotaryPositions

pytestmark = pytest.mark.gpu


def tokens(n, L, H, D, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn((L, n, 2, H, D), generator=g, device=dev, dtype=torch.bfloat16)


def same(a, b):
    """To the bit (a token beyond its static FP8 scale is a NaN, which equals nothing)."""
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def cache_of(four, L, H, D, pages, P, rope=None):
    return PagedFP4KVCache(L, H, D, pages, P, rope=rope) if four else PagedFP8KVCache(L, H, D, pages, P, rope=rope)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("P, n, rotary", [(16, 100, False), (32, 96, False), (16, 83, True), (48, 200, False), (16, 7, False)])
def test_forks_hold_what_whole_sequences_hold(dev, four, P, n, rotary):
    L, H, D = 2, 2, 64
    rope = RotaryPositions(D, 512) if rotary else None
    c, w = cache_of(four, L, H, D, 200, P, rope), cache_of(four, L, H, D, 200, P, rope)
    prompt = tokens(n, L, H, D, 0, dev)
    c.append(prompt, ["p"], [n])
    w.append(prompt, ["p"], [n])
    ids = ["a", "b", "c"]
    used = 200 - len(c._free)
    c.fork("p", ids)
    assert 200 - len(c._free) - used == (3 if n % P else 0)  # a copy of a page that the prompt ends inside, no more
    for i, s in enumerate(ids):
        w.append(prompt, [s], [n])
    more = [5, 1, 40, 17]
    x = tokens(sum(more), L, H, D, 1, dev)
    for cache in (c, w):  # every sequence goes on, the one that was forked too
        cache.append(x, ids + ["p"], more)
    for layer in range(L):
        for got, want in zip(c.gather(layer, ["p", *ids]), w.gather(layer, ["p", *ids])):
            assert same(got, want)
    c.fork("b", ["d", "e"], length=n // 2)
    c.append(x[:, :3].contiguous(), ["d"], [3])
    k, _ = c.gather(0, ["d", "e"])
    base, _ = w.gather(0, ["b"])
    assert same(k[0, :, :n // 2], base[0, :, :n // 2]) and same(k[1, :, :n // 2], base[0, :, :n // 2])
    assert same(c.gather(1, ids)[1], w.gather(1, ids)[1])


def test_freeing_forks(dev):
    c = PagedFP8KVCache(1, 1, 64, 20, 16)
    c.append(tokens(40, 1, 1, 64, 0, dev), ["p"], [40])
    c.fork("p", ["a", "b"])
    assert len(c._free) == 20 - 5
    c.free("p")
    assert len(c._free) == 20 - 4  # its own half page; the two whole ones are a's and b's
    k = c.gather(0, ["a"])[0].clone()
    c.free("b")
    assert len(c._free) == 20 - 3
    c.append(tokens(16, 1, 1, 64, 1, dev), ["q"], [16])
    assert same(c.gather(0, ["a"])[0], k)
    c.free("a")
    c.free("q")
    assert sorted(c._free) == list(range(20)) and not c._users and not c._common
    c.append(tokens(5, 1, 1, 64, 0, dev), ["p"], [5])
    c.fork("p", ["a"], length=0)
    assert c.lengths["a"] == 0 and c.pages["a"] == []
    c.append(tokens(5, 1, 1, 64, 0, dev), ["a"], [5])
    assert same(c.gather(0, ["a"])[0], c.gather(0, ["p"])[0])


def test_what_fork_refuses(dev):
    c = PagedFP8KVCache(1, 1, 64, 4, 16)
    c.append(tokens(40, 1, 1, 64, 0, dev), ["p"], [40])
    with pytest.raises(KeyError):
        c.fork("x", ["a"])
    for bad in (["a", "a"], ["p"]):
        with pytest.raises(ValueError):
            c.fork("p", bad)
    for n in (-1, 41):
        with pytest.raises(ValueError):
            c.fork("p", ["a"], length=n)
    with pytest.raises(MemoryError):
        c.fork("p", ["a", "b"])  # two copies of the half page, one page free
    assert list(c.pages) == ["p"] and len(c._free) == 1 and not c._users
    c.fork("p", ["a", "b"], length=32)
    c.fork("p", [])
    assert c.pages["a"] == c.pages["p"][:2]


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("D, P, rotary", [(128, 16, False), (64, 16, True), (128, 32, True)])
def test_attention_of_forks(dev, four, D, P, rotary, monkeypatch):
    """The same rows as over the same cache without what it knows of shared pages, to the types' accuracy:
    both are within one bf16 ulp (2^-7 of the value) + 2^-10 max|V| of the exact ones."""
    L, H, Hq, n = 1, 2, 8, 3000
    rope = RotaryPositions(D, 4096) if rotary else None
    c = PagedFP4KVCache(L, H, D, 900, P, rope=rope) if four else PagedFP8KVCache(L, H, D, 900, P, rope=rope,
                                                                                   overflow="saturate")
    c.append(tokens(n, L, H, D, 0, dev), ["p"], [n])
    c.append(tokens(2000, L, H, D, 5, dev), ["r"], [2000])
    ids = [f"a{i}" for i in range(20)]
    c.fork("p", ids)
    c.fork("r", ["s", "t"])
    c.fork("a3", ["a3x", "a3y"], length=2048)
    batch = ids + ["a3x", "a3y", "s", "t", "r"]
    more = [1 + 7 * i % 60 + 3 for i in range(len(batch))]
    c.append(tokens(sum(more), L, H, D, 1, dev), batch, more)
    monkeypatch.setattr(PagedFP8KVCache, "_LEAST_SAVED", 1)
    calls = []
    for name in ("paged_attention_shared", "paged_attention4_shared"):
        f = getattr(kv, name)
        monkeypatch.setattr(kv, name, lambda *a, f=f, **k: calls.append(1) or f(*a, **k))
    att = QuantizedRingAttention(c, ring_degree=1)
    g = torch.Generator(device=dev).manual_seed(2)
    rows = [1 + i % 4 for i in range(len(batch))]
    q1 = torch.randn((len(batch), Hq, D), generator=g, device=dev, dtype=torch.bfloat16)
    qn = torch.randn((sum(rows), Hq, D), generator=g, device=dev, dtype=torch.bfloat16)
    run = [lambda: att.decode(q1, 0, batch)]
    if D == 128 or four:  # the 8-bit prefill is for heads of 128
        run.append(lambda: att(qn, 0, batch, rows))
    got = [f() for f in run]
    assert len(calls) == len(run)
    cu_group, shared = c._groups(batch)
    assert cu_group.tolist() == [0, 22, 25]
    assert shared.tolist() == [2048 // P * P, 2000 // P * P]
    c._common.clear()
    want = [f() for f in run]
    assert len(calls) == len(run)
    vmax = float(c.gather(0, batch)[1].abs().max())
    for a, b in zip(got, want):
        assert ((a.float() - b.float()).abs() <= 2 * (2.0 ** -7 * b.float().abs() + 2.0 ** -10 * vmax)).all()


def test_few_forks_take_the_usual_kernels(dev, monkeypatch):
    c = PagedFP8KVCache(1, 2, 64, 100, 16)
    c.append(tokens(200, 1, 2, 64, 0, dev), ["p"], [200])
    c.fork("p", ["a"])
    monkeypatch.setattr(kv, "paged_attention_shared", None)
    q = torch.randn((2, 4, 64), device=dev, dtype=torch.bfloat16)
    assert QuantizedRingAttention(c).decode(q, 0, ["p", "a"]).shape == q.shape
    odd = PagedFP8KVCache(1, 2, 64, 9000, 8)  # pages that no matrix kernel takes
    odd.append(tokens(30000, 1, 2, 64, 0, dev), ["p"], [30000])
    odd.fork("p", ["a", "b", "c"])
    q = torch.randn((4, 4, 64), device=dev, dtype=torch.bfloat16)
    assert odd._groups(["p", "a", "b", "c"]) is None
    assert QuantizedRingAttention(odd).decode(q, 0, ["p", "a", "b", "c"]).shape == q.shape


def test_cached_states_read_by_rows_of_several_sequences(dev):
    """An encoder's states as a cached sequence that the hypotheses of a search are forks of: each row sees
    all of them, not causal."""
    c = PagedFP8KVCache(1, 2, 128, 400, 16)
    n = 1500
    x = tokens(n, 1, 2, 128, 0, dev)
    c.append(x, ["doc"], [n])
    beams = [f"b{i}" for i in range(40)]
    c.fork("doc", beams)
    att = QuantizedRingAttention(c, causal=False)
    q = torch.randn((40, 8, 128), device=dev, dtype=torch.bfloat16)
    assert c._groups(beams) is not None
    out = att.decode(q, 0, beams)
    k, v = (t[0].double() for t in c.gather(0, ["doc"], n))
    s = torch.matmul(q.double().view(40, 2, 4, 128).permute(1, 0, 2, 3).reshape(2, 160, 128), k.transpose(1, 2)) * 128 ** -0.5
    want = torch.matmul(torch.softmax(s, -1), v).view(2, 40, 4, 128).transpose(0, 1).reshape(40, 8, 128)
    # (gathered values are rounded to bf16 once more than the pages': 2^-8 of them each for scores and values)
    size = torch.matmul(q.double().abs().view(40, 2, 4, 128).permute(1, 0, 2, 3).reshape(2, 160, 128),
                        k.abs().transpose(1, 2)).amax() * 128 ** -0.5 * 2.0 ** -8
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -10 + 2.0 ** -8 + 2 * float(size)) * float(v.abs().max())
    assert ((out.double() - want).abs() <= tol).all()


def test_precisions_of_forks(dev, monkeypatch):
    """What attention to shared pages has the bits for takes it; "exact" over FP8 pages, with more, does not."""
    monkeypatch.setattr(PagedFP8KVCache, "_LEAST_SAVED", 1)
    calls = []
    for name in ("paged_attention_shared", "paged_attention4_shared"):
        f = getattr(kv, name)
        monkeypatch.setattr(kv, name, lambda *a, f=f, **k: calls.append(1) or f(*a, **k))
    q = torch.randn((3, 4, 128), device=dev, dtype=torch.bfloat16)
    for C, takes in ((PagedFP8KVCache, {"f16": 2, "bf16": 2, "exact": 0}),
                     (PagedFP4KVCache, {"f16": 2, "bf16": 2, "exact": 2})):
        c = C(1, 2, 128, 60, 16)
        c.append(tokens(100, 1, 2, 128, 0, dev), ["p"], [100])
        c.fork("p", ["a", "b"])
        for precision, n in takes.items():
            del calls[:]
            att = QuantizedRingAttention(c, precision=precision)
            a, b = att.decode(q, 0, ["p", "a", "b"]), att(q, 0, ["p", "a", "b"], [1, 1, 1])
            assert len(calls) == n
            assert ((a.float() - b.float()).abs() <= 2 * (2.0 ** -7 * b.float().abs() + 2.0 ** -7 * float(
                c.gather(0, ["p"])[1].abs().max()))).all()


def test_ids_again_and_again(dev, monkeypatch):
    """One sequence twice in a batch, ids freed and taken again by others, forks of forks whose source is
    gone, and groups that shrink as the batch changes: always what each sequence's own table says."""
    monkeypatch.setattr(PagedFP8KVCache, "_LEAST_SAVED", 1)
    # (scales are those of the first tokens: others may saturate, in both alike)
    c, w = (PagedFP8KVCache(1, 2, 64, 200, 16, overflow="saturate") for _ in range(2))
    x, y = tokens(100, 1, 2, 64, 0, dev), tokens(50, 1, 2, 64, 1, dev)
    c.append(x, ["p"], [100])
    c.fork("p", ["a", "b"])
    c.fork("a", ["c", "d"], length=70)
    c.free("a"), c.free("p")
    c.append(y, ["p"], [50])       # another sequence of that name
    c.fork("c", ["a"])
    w.append(x, ["b"], [100])
    first = x[:, :70].contiguous()
    for s in ("c", "d", "a"):
        w.append(first, [s], [70])
    w.append(y, ["p"], [50])
    att, plain = (QuantizedRingAttention(k, check=True) for k in (c, w))
    for batch in (["b", "c", "d", "a", "p"], ["a", "a", "p", "c"], ["d", "b"], ["p", "d", "p", "d"], ["c"]):
        q = torch.randn((len(batch), 4, 64), device=dev, dtype=torch.bfloat16)
        a, b = att.decode(q, 0, batch), plain.decode(q, 0, batch)
        vmax = float(w.gather(0, batch)[1].abs().max())
        assert ((a.float() - b.float()).abs() <= 2 * (2.0 ** -7 * b.float().abs() + 2.0 ** -10 * vmax)).all()
    for s in ("b", "c", "d", "a", "p"):
        c.free(s)
    assert len(c._free) == 200 and not c._users and not c._common


def test_training_and_serving_see_the_same(dev, monkeypatch):
    """An encoder's states of two sources, projected; a step of training on them, and serving from 4-bit pages
    that the rows' sequences are forks of.  What the pages hold is exact in bf16: cross attention to it and
    attention to the shared pages are off by a bf16 step (2^-8 of the value) each, weights rounded to bf16
    by another 2 x 2^-8 max|V| (numerator and sum), those of the pages 2^-15, fp32 sums 2^-15."""
    monkeypatch.setattr(PagedFP8KVCache, "_LEAST_SAVED", 1)
    D, H, Hq, lens = 128, 2, 8, [700, 1031]
    g = torch.Generator(device=dev).manual_seed(0)
    states = torch.randn((sum(lens), 64), generator=g, device=dev, dtype=torch.bfloat16)
    w = (torch.randn((64, 2 * H * D), generator=g, device=dev, dtype=torch.bfloat16) / 8).requires_grad_()
    wq = (torch.randn((64, Hq * D), generator=g, device=dev, dtype=torch.bfloat16) / 8).requires_grad_()
    rows = [6, 9]  # decoder rows of each source
    x = torch.randn((sum(rows), 64), generator=g, device=dev, dtype=torch.bfloat16)
    cu_q, cu_k = (torch.tensor([0, n[0], sum(n)], dtype=torch.int32, device=dev) for n in (rows, lens))
    q, kvs = (x @ wq).view(-1, Hq, D), (states @ w).view(-1, 2, H, D)
    out = CrossAttention()(q, kvs[:, 0], kvs[:, 1], cu_q, cu_k, max_q_per_seq=9, max_k_per_seq=1031)
    out.float().square().mean().backward()
    assert all(torch.isfinite(p.grad).all() and p.grad.any() for p in (w, wq))
    c = PagedFP4KVCache(1, H, D, 300, 16)
    c.append(kvs.detach()[None].contiguous(), ["s0", "s1"], lens)
    ids = [f"s{b}-{i}" for b in range(2) for i in range(rows[b])]
    for b in range(2):
        c.fork(f"s{b}", [s for s in ids if s.startswith(f"s{b}")])
    q = q.detach()
    served = QuantizedRingAttention(c, causal=False).decode(q, 0, ids)
    k, v = c.gather(0, ["s0", "s1"])
    held = [torch.cat([t[b, :, :n].transpose(0, 1) for b, n in enumerate(lens)]) for t in (k, v)]
    want = kv.cross_attention(q, *held, cu_q, cu_k)
    vmax = float(held[1].abs().max())
    tol = 2 * 2.0 ** -8 * want.float().abs() * (1 + 2.0 ** -8) + (2 * 2.0 ** -8 + 2.0 ** -14) * vmax
    assert ((served.float() - want.float()).abs() <= tol).all()
