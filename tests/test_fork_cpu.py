"""What a cache knows of its pages and rows around forks, without a GPU: the cache lies in host memory and
nothing is launched."""
import copy

import pytest
import torch

from zenyx_amd import kv
from zenyx_amd.train.fp8_kv_quantization import PagedFP4KVCache, PagedFP8KVCache, QuantizedRingAttention

HOST = torch.device("cpu")


def held(c, ids, lengths):
    """The cache with sequences of so many tokens, as appends would leave it."""
    entries = []
    for s, n in zip(ids, lengths):
        c._reserve(s, n, [], entries)
        c.lengths[s] = n
        c._len[c._row_of(s)] = n
    c._write_entries(entries)
    return c


def state(c):
    """Free pages, pages, lengths, users of pages, what is known to be shared, and table rows by sequence."""
    return (*copy.deepcopy((c._free, c.pages, c.lengths, c._users)), {s: sorted(k.values()) for s, k in c._common.items() if k},
            [(s, c._bt[r].tolist(), int(c._len[r])) for s, r in c._row.items()])


class Stop(Exception):
    pass


@pytest.fixture
def streams(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: None)


def failing(name, calls):
    """`name` of the module of kernels or of the cache, which raises at its call number `calls`."""
    def make(monkeypatch, c):
        where = kv if hasattr(kv, name) else c
        real, left = getattr(where, name), [calls]

        def f(*a, **k):
            left[0] -= 1
            if left[0] == 0:
                raise Stop
            return real(*a, **k)
        monkeypatch.setattr(where, name, f)
    return make


@pytest.mark.parametrize("C", [PagedFP8KVCache, PagedFP4KVCache])
@pytest.mark.parametrize("fault", [("tier_move_pages", 1), ("_write_entries", 1), ("_row_of", 1), ("_row_of", 3), ("_grow", 1)])
def test_a_fork_that_fails_leaves_the_cache_as_it_was(monkeypatch, streams, C, fault):
    """Pages, rows, tables and what is known of shared pages; the same fork then succeeds."""
    c = held(C(2, 1, 64, 60, 16, device=HOST), ["p", "r"], [40, 100])
    monkeypatch.setattr(kv, "tier_move_pages", lambda *a, **k: None)
    c.fork("p", ["x", "y"], length=32)
    ids = [f"n{i}" for i in range(14)]  # (more rows than the tables have at first)
    c._tables(["n1"])  # a row that a question about a sequence left behind
    before = state(c)
    with monkeypatch.context() as m:
        failing(*fault)(m, c)
        with pytest.raises(Stop):
            c.fork("p", ids)
    # (an id that is not in the cache need not keep its row; a table that has grown stays wide)
    after = state(c)
    assert after[:5] == before[:5]
    assert [x for x in after[5] if x[0] != "n1"] == [x for x in before[5] if x[0] != "n1"]
    assert set(c._row) - {"n1"} == {"p", "r", "x", "y"}
    assert sorted([*c._row.values(), *c._free_rows]) == list(range(len(c._row) + len(c._free_rows)))
    for r in c._free_rows:
        assert (c._bt[r] == -1).all() and c._len[r] == 0
    c.fork("p", ids)
    assert all(c.lengths[s] == 40 and c.pages[s][:2] == c.pages["p"][:2] for s in ids)
    for s in ["p", "r", "x", "y", *ids]:
        c.free(s)
    assert sorted(c._free) == list(range(60)) and not c._users and not c._common


def test_forks_share_whole_pages(monkeypatch, streams):
    moved = []
    monkeypatch.setattr(kv, "tier_move_pages", lambda dst, src, d, s, size, stream: moved.append((d.tolist(), s.tolist(), size)))
    c = held(PagedFP8KVCache(2, 1, 64, 30, 16, device=HOST), ["p"], [40])
    c.fork("p", ["a", "b"])
    size = c.pool[0, 0].numel()
    (d, s, n), = moved
    assert n == size and s == [(layer * 30 + c.pages["p"][2]) * size for layer in range(2) for _ in "ab"]
    assert d == [(layer * 30 + c.pages[x][2]) * size for layer in range(2) for x in "ab"]
    assert c._tables(["p", "a", "b"])[:, :2].unique(dim=0).shape[0] == 1
    assert c._lengths(["a", "b"]).tolist() == [40, 40]


def test_batches_that_the_kernel_of_shared_pages_refuses_take_the_usual_one(monkeypatch, streams):
    """More than 65,535 sequences, or more units of 128 positions than 32 bits count: prefill takes both."""
    c = held(PagedFP8KVCache(1, 1, 64, 8, 16, device=HOST), ["p"], [32])
    ids = list(range(65536))
    c.fork("p", ids)
    assert c._groups(ids[:-1]) is not None and c._groups(ids) is None
    taken = []
    monkeypatch.setattr(kv, "ring_attention_fp8", lambda q, *a, **k: taken.append("usual") or q)
    monkeypatch.setattr(kv, "paged_attention_shared", lambda q, *a, **k: taken.append("shared") or q)
    att = QuantizedRingAttention(c, check=False)
    att(torch.zeros((len(ids), 1, 64), dtype=torch.bfloat16), 0, ids, [1] * len(ids))
    assert taken == ["usual"]
    c = held(PagedFP8KVCache(1, 1, 64, 40, 1024, device=HOST), ["p"], [1024])
    ids = list(range(2000))
    c.fork("p", ids)
    assert c._groups(ids) is not None
    c._grow(width=1 << 14)  # 16 M positions a table, 128 K units
    assert c._groups(ids) is None


def shared_positions(C, Hkv, D, n, pages, P=16):
    """n forks of a sequence of so many pages, and their ids."""
    c = held(C(1, Hkv, D, pages + 2, P, device=HOST), ["p"], [pages * P])
    ids = [f"f{i}" for i in range(n)]
    c.fork("p", ids)
    return c, ids


@pytest.mark.parametrize("C, Hkv, D, n, pages, q_heads, rows, pays", [
    # what reading once saves is counted in bytes: 96 MiB over FP8 pages of 8 x 128, ...
    (PagedFP8KVCache, 8, 128, 25, 128, 32, 1, True), (PagedFP8KVCache, 8, 128, 24, 128, 32, 1, False),
    # ... of fewer heads more positions, of more heads fewer
    (PagedFP8KVCache, 2, 128, 25, 128, 8, 1, False), (PagedFP8KVCache, 2, 128, 97, 128, 8, 1, True),
    (PagedFP8KVCache, 1, 64, 97, 256, 4, 1, False), (PagedFP8KVCache, 32, 128, 7, 128, 32, 1, True),
    # 4 bits: 17/32 of the bytes
    (PagedFP4KVCache, 8, 128, 25, 128, 32, 1, False), (PagedFP4KVCache, 8, 128, 47, 128, 32, 1, True),
    # several rows, FP8: as one; heads that no other kernel takes
    (PagedFP8KVCache, 8, 128, 25, 128, 32, 8, True), (PagedFP8KVCache, 8, 128, 24, 128, 32, 8, False),
    (PagedFP8KVCache, 1, 64, 2, 1, 4, 2, True),
    # 4 bits: in proportion to a sequence's columns, and not for very many of them
    (PagedFP4KVCache, 8, 128, 25, 512, 32, 2, True), (PagedFP4KVCache, 8, 128, 25, 512, 32, 8, False),
    (PagedFP4KVCache, 8, 128, 25, 2048, 32, 8, True), (PagedFP4KVCache, 8, 128, 97, 512, 32, 4, False),
    (PagedFP4KVCache, 8, 128, 47, 256, 8, 4, True)])
def test_sharing_is_taken_where_it_saves_bytes_enough(monkeypatch, streams, C, Hkv, D, n, pages, q_heads, rows, pays):
    c, ids = shared_positions(C, Hkv, D, n, pages)
    assert c._groups(ids) is not None  # (what is shared is known whether it pays or not)
    taken = []
    for name in ("ring_attention_fp8", "paged_attention4_prefill", "paged_attention_decode", "paged_attention4_decode"):
        monkeypatch.setattr(kv, name, lambda q, *a, **k: taken.append(False) or q)
    for name in ("paged_attention_shared", "paged_attention4_shared"):
        monkeypatch.setattr(kv, name, lambda q, *a, **k: taken.append(True) or q)
    att = QuantizedRingAttention(c, check=False)
    q = torch.zeros((n * rows, q_heads, D), dtype=torch.bfloat16)
    att.decode(q, 0, ids) if rows == 1 else att(q, 0, ids, [rows] * n)
    assert taken == [pays]


def test_what_is_known_of_a_batch_follows_it(monkeypatch, streams):
    c, ids = shared_positions(PagedFP8KVCache, 8, 128, 30, 128)
    assert c._sharing_pays(ids, 1, 32) and not c._sharing_pays(ids[:20], 1, 32) and c._sharing_pays(ids, 1, 32)
    first = c._groups(ids)
    assert c._groups(ids) is first and first[0].tolist() == [0, 30] and first[1].tolist() == [2048]
    for s in ids[20:]:
        c.free(s)
    assert c._groups(ids)[0].tolist() == [0, 20, *range(21, 31)] and not c._sharing_pays(ids, 1, 32)
    assert c._groups([ids[0]]) is None and not c._sharing_pays([], 1, 32)


def test_queries_of_any_shape_reach_the_kernels_wrapper(monkeypatch, streams):
    """Which checks them: their shape is nobody else's business, with forks or without."""
    c = held(PagedFP8KVCache(1, 1, 64, 8, 16, device=HOST), ["p"], [32])
    seen = []
    monkeypatch.setattr(kv, "paged_attention_decode", lambda q, *a, **k: seen.append(q.dim()) or q)
    att = QuantizedRingAttention(c, check=False)
    for ids in (["p"], ["p", "a"]):
        for q in (torch.zeros(64), torch.zeros(1, 64), torch.zeros(1, 1, 1, 64)):
            att.decode(q, 0, ids)
        c.fork("p", ["a"]) if "a" not in c.lengths else None
    assert seen == 2 * [1, 2, 4]


def test_a_batch_asked_for_before_its_fork_was_made(monkeypatch, streams):
    """An id that was not in the cache, and is a fork by the next call."""
    c, ids = shared_positions(PagedFP8KVCache, 8, 128, 30, 128)
    batch = [*ids, "later"]
    assert c._groups(batch)[0].tolist() == [0, 30, 31]
    c.fork("p", ["later"])
    assert c._groups(batch)[0].tolist() == [0, 31]
