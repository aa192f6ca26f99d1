"""Attention to keys that many rows share, as timed cases.

Four kinds of call (32 query heads, 8 KV heads, head_dim 128 and pages of 16 tokens unless a
case says otherwise):

* ``shared8``  new tokens of many sequences attend to their FP8 pages, the first of which (a system
               prompt, a document) are the same pages for all sequences of a group;
* ``shared4``  the same over 4-bit pages;
* ``cross``    a decoder's rows attend to an encoder's states, sequences of both lengths packed;
* ``train``    the same and its gradients, as a training step takes them.

FP8 pages hold e4m3 codes ``[n_pages, 2, H, P, D]`` with a scale per K/V and head.  A 4-bit page
holds, per K/V and head, tiles of 16 tokens: e2m1 codes ``[D / 32][16][16]`` bytes (32 channels of
a token in 16 bytes, the even channel in the low bits), then one power of two per 32 channels,
``[D / 32][16]`` bytes (2^(byte - 127)).
"""
from __future__ import annotations

import math
import random

import torch

own = False

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # Two samples of one chat: the next token of each, one layer's attention.
        {"name": "shared8_two", "kind": "shared8", "groups": 1, "seqs_lo": 2, "seqs_hi": 2, "shared_lo": 1024,
         "shared_hi": 1024, "own_lo": 1, "own_hi": 60, "rows": 1, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "lens": 1},
        # A serving batch behind one system prompt.
        {"name": "shared8_chat", "kind": "shared8", "groups": 1, "seqs_lo": 64, "seqs_hi": 64, "shared_lo": 2048,
         "shared_hi": 2048, "own_lo": 100, "own_hi": 2000, "rows": 1, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "lens": 2},
        # Many questions about one long document.
        {"name": "shared8_document", "kind": "shared8", "groups": 1, "seqs_lo": 128, "seqs_hi": 128,
         "shared_lo": 32768, "shared_hi": 32768, "own_lo": 20, "own_hi": 500, "rows": 1, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "lens": 3},
        # Prompts of several users, each sampled a few times by a small model of 12 heads of 64.
        {"name": "shared8_samples", "kind": "shared8", "groups": 8, "seqs_lo": 1, "seqs_hi": 16, "shared_lo": 500,
         "shared_hi": 8000, "own_lo": 1, "own_hi": 700, "rows": 1, "q_heads": 12, "kv_heads": 12, "dim": 64,
         "page": 16, "lens": 4},
        # A serving batch behind one long prompt, 4-bit pages.
        {"name": "shared4_chat", "kind": "shared4", "groups": 1, "seqs_lo": 16, "seqs_hi": 16, "shared_lo": 8192,
         "shared_hi": 8192, "own_lo": 100, "own_hi": 1000, "rows": 1, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "lens": 5},
        # Four documents and up to 8 proposed tokens of each of the sequences that ask about them, checked at once.
        {"name": "shared4_proposals", "kind": "shared4", "groups": 4, "seqs_lo": 4, "seqs_hi": 16, "shared_lo": 4000,
         "shared_hi": 16000, "own_lo": 30, "own_hi": 600, "rows": 8, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "lens": 6},
        # A decoding step of 32 transcriptions: one row each on 1,500 states.
        {"name": "cross_step", "kind": "cross", "seqs": 32, "q_lo": 1, "q_hi": 1, "k_lo": 1500, "k_hi": 1500,
         "q_heads": 12, "kv_heads": 12, "dim": 64, "fused": True, "type": "float16", "lens": 7},
        # The prompts of a batch against their documents' states.
        {"name": "cross_prompt", "kind": "cross", "seqs": 8, "q_lo": 200, "q_hi": 1000, "k_lo": 1000, "k_hi": 8000,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "fused": True, "type": "bfloat16", "lens": 8},
        # A translation batch's training step: short ragged sequences on both sides.
        {"name": "train_pairs", "kind": "train", "seqs": 64, "q_lo": 5, "q_hi": 120, "k_lo": 5, "k_hi": 150,
         "q_heads": 12, "kv_heads": 12, "dim": 64, "fused": True, "type": "bfloat16", "lens": 9},
        # A transcription model's training step: 448 rows at most on 1,500 states.
        {"name": "train_speech", "kind": "train", "seqs": 16, "q_lo": 50, "q_hi": 448, "k_lo": 1500, "k_hi": 1500,
         "q_heads": 12, "kv_heads": 12, "dim": 64, "fused": True, "type": "float16", "lens": 10},
        # An image's 4,096 positions on a caption of 77 tokens, 8 of them.
        {"name": "train_caption", "kind": "train", "seqs": 8, "q_lo": 4096, "q_hi": 4096, "k_lo": 77, "k_hi": 77,
         "q_heads": 8, "kv_heads": 8, "dim": 64, "fused": False, "type": "bfloat16", "lens": 11},
        # Long answers about long documents, grouped heads.
        {"name": "train_long", "kind": "train", "seqs": 4, "q_lo": 1000, "q_hi": 2048, "k_lo": 2000, "k_hi": 8192,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "fused": True, "type": "bfloat16", "lens": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["shared8", "shared4", "cross", "train"])
    lens = rng.randrange(1 << 30)  # seeds the case's lengths
    kv_heads, dim = rng.choice([(8, 128), (8, 128), (4, 128), (2, 128), (12, 64), (8, 64), (16, 64)])
    if kind in ("shared8", "shared4"):
        kv_heads, dim = rng.choice([(kv_heads, dim), (kv_heads, dim), (kv_heads, dim), (4, 256)])
        q_heads = kv_heads * rng.choice([1, 4, 4, 8])
        groups = rng.choice([1, 1, 2, 5, 12])
        seqs = max(1, _log(rng, 1, 128) // groups)
        rows = rng.choice([1, 1, 1, 2, 5, 8])
        # at most half of the scores and keys that the largest listed case has
        most = 128 * 32768 * 32 // 2
        shared = max(16, min(_log(rng, 50, 32768), most // (groups * seqs * rows * q_heads)))
        fresh = max(rows, min(_log(rng, 1, 4000), 100_000_000 // (groups * seqs * kv_heads * dim)))
        return {"kind": kind, "groups": groups, "seqs_lo": max(1, seqs // rng.choice([1, 1, 4])), "seqs_hi": seqs,
                "shared_lo": max(1, shared // rng.choice([1, 2, 5])), "shared_hi": shared, "own_lo": rows,
                "own_hi": fresh, "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([16, 16, 32, 64]), "lens": lens}
    q_heads = kv_heads * rng.choice([1, 1, 2, 4])
    seqs = _log(rng, 1, 64)
    k_hi = _log(rng, 5, 8192)
    most = 4 * 2048 * 8192 * 32 * 128 // (8 if kind == "train" else 2)
    q_hi = max(1, min(_log(rng, 1, 4096), most // (seqs * k_hi * q_heads * dim)))
    return {"kind": kind, "seqs": seqs, "q_lo": max(1, q_hi // rng.choice([1, 2, 10])), "q_hi": q_hi,
            "k_lo": max(1, k_hi // rng.choice([1, 2, 10])), "k_hi": k_hi, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "fused": rng.random() < 0.5, "type": rng.choice(["bfloat16", "bfloat16", "float16"]),
            "lens": lens}


# ------------------------------------------------------------------ inputs

def _shape(case):
    """A matter of the case: (sequences of every group, tokens that they share, tokens of every
    sequence of its own, its rows), or (rows, states) of every sequence."""
    r = random.Random(case["lens"])
    if case["kind"] in ("cross", "train"):
        return ([r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])],
                [r.randint(case["k_lo"], case["k_hi"]) for _ in range(case["seqs"])])
    seqs = [r.randint(case["seqs_lo"], case["seqs_hi"]) for _ in range(case["groups"])]
    # whole pages are shared: what is left of a prompt is among a sequence's own tokens
    shared = [r.randint(case["shared_lo"], case["shared_hi"]) // case["page"] * case["page"] for _ in seqs]
    fresh = [r.randint(case["own_lo"], case["own_hi"]) for _ in range(sum(seqs))]
    rows = [min(n, r.randint(1, case["rows"])) for n in fresh]
    return seqs, shared, fresh, rows


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _starts(counts, dev):
    return torch.tensor([0] + counts, device=dev).cumsum(0).to(torch.int32)


def _tiles(n_pages, heads, page, dim, g, dev):
    """A layer of 4-bit pages filled with the codes of normal values."""
    pool = torch.empty((n_pages, 2, heads, page // 16, 17 * dim // 2), dtype=torch.uint8, device=dev)
    # of 16 codes, how often each appears among normal values coded in blocks of 32
    p = torch.tensor([.10, .19, .17, .13, .17, .13, .08, .03], dtype=torch.float64)
    cut = (torch.cat([p, p]).cumsum(0) * 128).round().long()
    nibble = torch.searchsorted(cut, torch.arange(256), right=True).clamp(max=15).to(torch.uint8).to(dev)
    power = torch.tensor([124] * 16 + [125] * 160 + [126] * 72 + [127] * 8, dtype=torch.uint8, device=dev)
    n = 8 * dim
    shape = pool[..., :n].shape
    lo, hi = (nibble[torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.int32)] for _ in range(2))
    pool[..., :n] = lo | (hi << 4)
    pool[..., n:] = power[torch.randint(0, 256, pool[..., n:].shape, generator=g, device=dev, dtype=torch.int32)]
    return pool


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    dim, heads = case["dim"], case["kv_heads"]
    if case["kind"] in ("cross", "train"):
        rows, states = _shape(case)
        t = _TYPES[case["type"]]
        s["most_q"], s["most_k"] = max(rows), max(states)
        s["cu_q"], s["cu_k"] = _starts(rows, dev), _starts(states, dev)
        s["q"] = torch.randn((sum(rows), case["q_heads"], dim), generator=g, device=dev).mul_(1.5).to(t)
        kv = torch.randn((sum(states), 2, heads, dim), generator=g, device=dev).to(t)
        # the two halves of a fused projection, or of two
        s["k"], s["v"] = (kv[:, 0], kv[:, 1]) if case["fused"] else (kv[:, 0].contiguous(), kv[:, 1].contiguous())
        if case["kind"] == "train":
            s["grad"] = torch.randn(s["q"].shape, generator=g, device=dev).to(t)
            s["leaves"] = [s[n].requires_grad_() for n in ("q", "k", "v")]
        # sequence and number within it of each row and state, as the plain form indexes them
        for n, cu, count in (("q", s["cu_q"], rows), ("k", s["cu_k"], states)):
            b = torch.repeat_interleave(torch.arange(len(count), device=dev), torch.tensor(count, device=dev))
            s["at_" + n] = b, torch.arange(sum(count), device=dev) - cu[b]
        return s
    page = case["page"]
    seqs, shared, fresh, rows = _shape(case)
    s["most_rows"], s["most_seqs"] = max(rows), max(seqs)
    group = [i for i, n in enumerate(seqs) for _ in range(n)]
    head = [shared[i] // page for i in group]
    need = [a + -(-n // page) for a, n in zip(head, fresh)]
    total = [shared[i] + n for i, n in zip(group, fresh)]
    # pages in no order: those of the prefixes first in the list, then each sequence's own
    first, at = [], 0
    for n in shared:
        first.append(at)
        at += n // page
    n_pages = at + sum(a - b for a, b in zip(need, head)) + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    own_at = at + torch.tensor([0] + [a - b for a, b in zip(need, head)], device=dev).cumsum(0)[:-1]
    col = torch.arange(max(max(need), 1), device=dev)
    head_t, need_t = torch.tensor(head, device=dev)[:, None], torch.tensor(need, device=dev)[:, None]
    index = torch.where(col < head_t, torch.tensor([first[i] for i in group], device=dev)[:, None] + col,
                        own_at[:, None] + col - head_t)
    s["bt"] = torch.where(col < need_t, order[index.clamp(max=n_pages - 1)], -1)
    s["lens"], s["shared"], s["cu_group"] = _ints(total, dev), _ints(shared, dev), _starts(seqs, dev)
    s["cu_q"] = _starts(rows, dev) if case["rows"] > 1 else None
    if case["kind"] == "shared8":
        pool = torch.randn((n_pages, 2, heads, page, dim), generator=g, device=dev, dtype=torch.bfloat16).mul_(64)
        s["pool"] = pool.to(torch.float8_e4m3fn).view(torch.uint8)
        s["scales"] = (torch.rand((2, heads), generator=g, device=dev) + 0.5) / 64
    else:
        s["pool"] = _tiles(n_pages, heads, page, dim, g, dev)
    s["q"] = torch.randn((sum(rows), case["q_heads"], dim), generator=g, device=dev).mul_(2.0).to(torch.bfloat16)
    # what the plain form indexes with: each row's sequence and number within it, each sequence's group and
    # place in it, the first sequence of every group, and each sequence's own pages
    seq = torch.repeat_interleave(torch.arange(len(rows), device=dev), torch.tensor(rows, device=dev))
    s["row_seq"], s["row_at"] = seq, torch.arange(len(seq), device=dev) - _starts(rows, dev)[seq]
    s["row_pos"] = torch.tensor(total, device=dev)[seq] - torch.tensor(rows, device=dev)[seq] + s["row_at"]
    s["seq_group"] = torch.tensor(group, device=dev)
    s["seq_at"] = torch.arange(len(group), device=dev) - s["cu_group"][s["seq_group"]]
    s["most_shared"], s["most_own"] = max(shared) // page, max(a - b for a, b in zip(need, head))
    own_col = head_t + torch.arange(s["most_own"], device=dev)
    s["own_bt"] = torch.where(own_col < need_t, s["bt"].gather(1, own_col.clamp(max=len(col) - 1)), 0)
    s["own_from"] = torch.tensor([shared[i] for i in group], device=dev)
    return s


# ------------------------------------------------------------------ the plain forms

def _cached(pages, s):
    """(K, V) fp32 [n, H, positions, D] of page lists [n, pages] (-1: anything)."""
    t = s["pool"][pages.clamp(min=0).long()]  # [n, pages, 2, H, ...]
    if s["kind"] == "shared8":
        v = t.view(torch.float8_e4m3fn).float() * s["scales"][:, :, None, None]
    else:
        dim = s["dim"]
        c = t[..., :8 * dim].unflatten(-1, (dim // 32, 16, 16))
        both = torch.stack([c & 15, c >> 4], -1).flatten(-2)  # [..., page / 16, D / 32, 16, 32]
        power = torch.exp2(t[..., 8 * dim:].unflatten(-1, (dim // 32, 16)).float() - 127)
        v = torch.tensor(_E2M1, device=t.device)[both.int()] * power[..., None]
        v = v.transpose(-3, -2).flatten(-2).flatten(-3, -2)
    v = v.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)
    return v[0], v[1]


def _plain_shared(s):
    heads, dim, rows = s["kv_heads"], s["dim"], s["most_rows"]
    group = s["q_heads"] // heads
    dev = s["q"].device
    n_seqs, n_groups = len(s["seq_group"]), s["groups"]
    # rows padded per sequence, [B, H, rows x group, D]
    q = torch.zeros((n_seqs, rows, s["q_heads"], dim), device=dev)
    q[s["row_seq"], s["row_at"]] = s["q"].float() * dim ** -0.5
    pos = torch.full((n_seqs, rows), -1, device=dev)
    pos[s["row_seq"], s["row_at"]] = s["row_pos"]
    q = q.view(n_seqs, rows, heads, group, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)
    # the group's keys, once for all its rows
    lead = s["bt"][s["cu_group"][:-1].long(), :max(1, s["most_shared"])]
    kp, vp = _cached(lead, s)
    all_q = torch.zeros((n_groups, s["most_seqs"], heads, rows * group, dim), device=dev)
    all_q[s["seq_group"], s["seq_at"]] = q
    all_q = all_q.transpose(1, 2).flatten(2, 3)
    sp = torch.matmul(all_q, kp.transpose(-1, -2))
    hidden = torch.arange(kp.shape[2], device=dev) >= s["shared"][:, None]
    sp.masked_fill_(hidden[:, None, None], -math.inf)
    # each sequence's own keys
    ko, vo = _cached(s["own_bt"], s)
    so = torch.matmul(q, ko.transpose(-1, -2))
    at = s["own_from"][:, None] + torch.arange(ko.shape[2], device=dev)
    late = at[:, None] > pos.repeat_interleave(group, 1)[..., None]
    so.masked_fill_(late[:, None], -math.inf)
    # one softmax over both
    back = s["seq_group"], slice(None), s["seq_at"]

    def per_seq(t):  # [G, H, seqs x rows x group, *] -> [B, H, rows x group, *]
        return t.unflatten(2, (s["most_seqs"], rows * group))[back]
    top = torch.maximum(per_seq(sp.amax(-1, keepdim=True)), so.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    all_top = torch.zeros((n_groups, s["most_seqs"], heads, rows * group, 1), device=dev)
    all_top[s["seq_group"], s["seq_at"]] = top
    pp, po = sp.sub_(all_top.transpose(1, 2).flatten(2, 3)).exp_(), so.sub_(top).exp_()
    total = per_seq(pp.sum(-1, keepdim=True)) + po.sum(-1, keepdim=True)
    o = (per_seq(torch.matmul(pp, vp)) + torch.matmul(po, vo)) / torch.where(total == 0, 1.0, total)
    o = o.unflatten(2, (rows, group)).transpose(1, 2).flatten(2, 3)
    return o[s["row_seq"], s["row_at"]].to(torch.bfloat16)


def _padded(x, at, n_seqs, most):
    out = torch.zeros((n_seqs, most, *x.shape[1:]), device=x.device)
    out[at] = x.float()
    return out


def _plain_cross(s):
    n, heads, dim = s["seqs"], s["kv_heads"], s["dim"]
    group, scale, dev = s["q_heads"] // heads, s["dim"] ** -0.5, s["q"].device

    def split(x):  # [B, rows, Hq, D] -> [B, H, group x rows, D]
        return x.unflatten(2, (heads, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)

    def joined(x):
        x = x.unflatten(2, (group, s["most_q"])).permute(0, 3, 1, 2, 4).flatten(2, 3)
        return x[s["at_q"]].to(s["q"].dtype)

    q = split(_padded(s["q"].detach(), s["at_q"], n, s["most_q"]))
    k, v = (_padded(s[i].detach(), s["at_k"], n, s["most_k"]).transpose(1, 2) for i in ("k", "v"))
    hidden = torch.arange(s["most_k"], device=dev) >= (s["cu_k"][1:] - s["cu_k"][:-1])[:, None]
    score = torch.matmul(q * scale, k.transpose(-1, -2)).masked_fill_(hidden[:, None, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p, v)
    if s["kind"] == "cross":
        return joined(o)
    do = split(_padded(s["grad"], s["at_q"], n, s["most_q"]))
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q)
    dk, dv = (t.transpose(1, 2)[s["at_k"]].to(s["q"].dtype) for t in (dk, dv))
    return {"out": joined(o), "dq": joined(dq), "dk": dk, "dv": dv}


def _plain(s):
    with torch.no_grad():
        return _plain_cross(s) if s["kind"] in ("cross", "train") else _plain_shared(s)


def _own(s):
    from zenyx_amd import kv

    if s["kind"] == "shared8":
        return kv.paged_attention_shared(s["q"], s["pool"], s["scales"], s["bt"], s["lens"], s["cu_group"], s["shared"],
                                         cu_q=s["cu_q"], max_q_per_seq=s["most_rows"])
    if s["kind"] == "shared4":
        return kv.paged_attention4_shared(s["q"], s["pool"], s["bt"], s["lens"], s["cu_group"], s["shared"],
                                          cu_q=s["cu_q"], max_q_per_seq=s["most_rows"])
    if s["kind"] == "cross":
        return kv.cross_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_q_per_seq=s["most_q"],
                                  max_k_per_seq=s["most_k"])
    from zenyx_amd.train.cross_attention import CrossAttention

    out = CrossAttention()(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_q_per_seq=s["most_q"],
                           max_k_per_seq=s["most_k"])
    dq, dk, dv = torch.autograd.grad(out, s["leaves"], s["grad"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    dim, heads, q_heads = case["dim"], case["kv_heads"], case["q_heads"]
    if case["kind"] in ("cross", "train"):
        rows, states = _shape(case)
        pairs = sum(a * b for a, b in zip(rows, states)) * q_heads * dim
        q, k = 2 * sum(rows) * q_heads * dim, 2 * sum(states) * heads * dim
        if case["kind"] == "cross":
            return {"bytes": 2 * q + 2 * k, "flops": 4 * pairs}
        # two products forward and five for the gradients; q, grad, k, v in, out, dq, dk, dv out
        return {"bytes": 4 * q + 4 * k, "flops": 14 * pairs}
    seqs, shared, fresh, rows = _shape(case)
    token = 2 * heads * (dim if case["kind"] == "shared8" else dim // 2 + dim // 32)
    group = [i for i, n in enumerate(seqs) for _ in range(n)]
    pairs = sum(r * (shared[i] + n) - r * (r - 1) // 2 for i, n, r in zip(group, fresh, rows))
    return {"bytes": (sum(shared) + sum(fresh)) * token + 4 * sum(rows) * q_heads * dim,
            "flops": 4 * pairs * q_heads * dim}


# ------------------------------------------------------------------ the definitions in 64 bits

def _page64(s, pages, j, h):
    """K (0) or V (1) of one head of a list of pages in 64 bits: [positions, D]."""
    t = s["pool"][pages.long(), j, h]
    if s["kind"] == "shared8":
        return t.reshape(-1, s["dim"]).view(torch.float8_e4m3fn).double() * s["scales"][j, h].double()
    dim, (nb, n) = s["dim"], t.shape[:2]
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=t.device)
    code = t[..., :8 * dim].reshape(nb, n, dim // 32, 16, 16).long()
    v = torch.empty((nb, n, dim // 32, 16, 32), dtype=torch.float64, device=t.device)
    v[..., 0::2], v[..., 1::2] = grid[code % 16], grid[code // 16]
    v *= 2.0 ** (t[..., 8 * dim:].reshape(nb, n, dim // 32, 16, 1).double() - 127.0)
    return v.permute(0, 1, 3, 2, 4).reshape(-1, dim)


def _exact_shared(case, s):
    """Every sequence by itself, over all the pages that its block table names."""
    seqs, shared, fresh, rows = _shape(case)
    group = [i for i, n in enumerate(seqs) for _ in range(n)]
    heads, dim = case["kv_heads"], case["dim"]
    grp = case["q_heads"] // heads
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for h in range(heads):
        at, kept = 0, (-1, None)
        for b, (i, n, r) in enumerate(zip(group, fresh, rows)):
            if kept[0] != i:  # the shared pages of the group, decoded once for its sequences
                kept = i, [_page64(s, s["bt"][b, :shared[i] // case["page"]], j, h) for j in range(2)]
            mine = s["bt"][b, shared[i] // case["page"]:-(-(shared[i] + n) // case["page"])]
            k, v = (torch.cat([kept[1][j], _page64(s, mine, j, h)[:n]]) for j in range(2))
            q = s["q"][at:at + r, h * grp:(h + 1) * grp].double()
            score = torch.matmul(q, k.t()) / math.sqrt(dim)
            seen = shared[i] + n - r + torch.arange(r, device=k.device)
            score.masked_fill_((torch.arange(len(k), device=k.device) > seen[:, None])[:, None], -math.inf)
            out[at:at + r, h * grp:(h + 1) * grp] = torch.matmul(torch.softmax(score, -1), v)
            at += r
    return out


def _exact_cross(case, s):
    rows, states = _shape(case)
    grp, dim = case["q_heads"] // case["kv_heads"], case["dim"]
    q, k, v = (s[n].detach() for n in ("q", "k", "v"))
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(out), torch.zeros(k.shape, dtype=torch.float64, device=q.device), None
    dv = torch.zeros_like(dk)
    a = c = 0
    for n, m in zip(rows, states):
        for h in range(case["q_heads"]):
            qh, kh, vh = q[a:a + n, h].double(), k[c:c + m, h // grp].double(), v[c:c + m, h // grp].double()
            p = torch.softmax(qh @ kh.t() / math.sqrt(dim), -1)
            out[a:a + n, h] = p @ vh
            if case["kind"] == "train":
                do = s["grad"][a:a + n, h].double()
                dp = do @ vh.t()
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(dim)
                dq[a:a + n, h] = ds @ kh
                dk[c:c + m, h // grp] += ds.t() @ qh
                dv[c:c + m, h // grp] += p.t() @ do
        a, c = a + n, c + m
    return out if case["kind"] == "cross" else {"out": out, "dq": dq, "dk": dk, "dv": dv}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_cross(case, s) if case["kind"] in ("cross", "train") else _exact_shared(case, s)
