"""Rotary positions and the 4-bit KV cache, as timed cases.

Five kinds of call on a paged KV cache (8 KV heads, 32 query heads, head_dim 128 and pages of
16 tokens unless a case says otherwise):

* ``rope``     rotary positions of query or key rows, or the gradient's rotation back;
* ``append8``  new tokens' keys are rotated, and keys and values stored as FP8 in their pages;
* ``append4``  the same into pages of 4 bits, then read back as contiguous bf16 K and V;
* ``decode4``  one query token per sequence attends to its 4-bit pages;
* ``prefill4`` blocks of new tokens attend to the 4-bit pages, causal.

A 4-bit page holds, per K/V and head, tiles of 16 tokens: e2m1 codes ``[D / 32][16][16]``
bytes (32 channels of a token in 16 bytes, the even channel in the low bits), then one power
of two per 32 channels, ``[D / 32][16]`` bytes (2^(byte - 127), 255: NaN).
"""
from __future__ import annotations

import math
import random

import torch

own = False

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # A decode step of a serving batch: the new tokens' queries of one layer, far positions.
        {"name": "rope_step", "kind": "rope", "rows": 64, "heads": 32, "dim": 128, "rot": 128, "interleaved": False,
         "transpose": False, "type": "bfloat16", "far": 131072},
        # A training step's gradient of the rotated queries, 4 sequences of 4,096 tokens.
        {"name": "rope_train_grad", "kind": "rope", "rows": 16384, "heads": 32, "dim": 128, "rot": 128,
         "interleaved": True, "transpose": True, "type": "bfloat16", "far": 4096},
        # A decode step's new tokens of all 32 layers, with the prompt's scales.
        {"name": "append8_step", "kind": "append8", "layers": 32, "seqs": 64, "lo": 1, "hi": 1, "old": 500,
         "static": True, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 16, "lens": 1},
        # 16 prompts of 1k-8k tokens, four layers in one call, scales from the batch.
        {"name": "append8_prompt", "kind": "append8", "layers": 4, "seqs": 16, "lo": 1024, "hi": 8192, "old": 0,
         "static": False, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 16, "lens": 2},
        # A decode step's new tokens of one layer, read back with the few tokens before them.
        {"name": "append4_step", "kind": "append4", "seqs": 64, "lo": 1, "hi": 1, "old": 200, "kv_heads": 8,
         "dim": 128, "rot": 128, "interleaved": False, "page": 16, "lens": 3},
        # 16 prompts of 1k-8k tokens of one layer, half of each head rotated, stored and read back.
        {"name": "append4_prompt", "kind": "append4", "seqs": 16, "lo": 1024, "hi": 8192, "old": 0, "kv_heads": 8,
         "dim": 128, "rot": 64, "interleaved": False, "page": 16, "lens": 4},
        # One chat: the next token of a single sequence, one layer's attention.
        {"name": "decode4_one", "kind": "decode4", "seqs": 1, "lo": 2048, "hi": 2048, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "lens": 5},
        # A serving batch: 16 sequences of 1k-8k tokens.
        {"name": "decode4_batch", "kind": "decode4", "seqs": 16, "lo": 1024, "hi": 8192, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "lens": 6},
        # A full long-context batch: 64 sequences at 32k.
        {"name": "decode4_long", "kind": "decode4", "seqs": 64, "lo": 32768, "hi": 32768, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "lens": 7},
        # Many short chats of a small model: 12 heads of 64, a KV head each.
        {"name": "decode4_short", "kind": "decode4", "seqs": 128, "lo": 100, "hi": 600, "q_heads": 12, "kv_heads": 12,
         "dim": 64, "page": 16, "lens": 8},
        # A few proposed tokens each of 16 running sequences, checked at once.
        {"name": "prefill4_few", "kind": "prefill4", "seqs": 16, "q_lo": 1, "q_hi": 5, "old_lo": 1000, "old_hi": 8000,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "lens": 9},
        # Chunked prefill of a running server: two sequences' next chunks on top of what is cached.
        {"name": "prefill4_chunk", "kind": "prefill4", "seqs": 2, "q_lo": 2048, "q_hi": 2048, "old_lo": 4000,
         "old_hi": 14000, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "lens": 10},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append8", "append4", "decode4", "decode4", "prefill4"])
    page = rng.choice([16, 16, 32, 64])
    kv_heads, dim = rng.choice([(8, 128), (8, 128), (4, 128), (16, 128), (2, 128), (12, 64), (8, 64), (4, 256)])
    rot = rng.choice([dim, dim, dim // 2])
    inter = rng.random() < 0.4
    lens = rng.randrange(1 << 30)  # seeds the case's sequence lengths
    if kind == "rope":
        heads = rng.choice([8, 12, 32, 32, 71])
        return {"kind": kind, "rows": _log(rng, 1, 16384 * 32 * 128 // (heads * dim) // 2), "heads": heads,
                "dim": dim, "rot": rot, "interleaved": inter, "transpose": rng.random() < 0.4,
                "type": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), "far": _log(rng, 100, 131072)}
    if kind == "append8":
        static = rng.random() < 0.5
        seqs = _log(rng, 1, 64 if static else 16)
        layers = rng.choice([1, 1, 4, 12])
        hi = _log(rng, 1, 16) if static else min(_log(rng, 50, 32768), 256_000_000 // (seqs * layers * kv_heads * dim))
        return {"kind": kind, "layers": layers, "seqs": seqs, "lo": max(1, hi // rng.choice([1, 2, 4])), "hi": hi,
                "old": rng.randrange(500) if static else 0, "static": static, "kv_heads": kv_heads, "dim": dim,
                "rot": rot, "interleaved": inter, "page": page, "lens": lens}
    if kind == "append4":
        seqs = _log(rng, 1, 64)
        hi = min(_log(rng, 1, 16384), 100_000_000 // (seqs * kv_heads * dim))
        return {"kind": kind, "seqs": seqs, "lo": max(1, hi // rng.choice([1, 2, 4])), "hi": hi,
                "old": rng.randrange(1, 300) if hi < 500 else 0, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([0, rot, rot]), "interleaved": inter, "page": page, "lens": lens}
    if kind == "decode4":
        seqs = _log(rng, 1, 128)
        hi = min(_log(rng, 100, 32768), 500_000_000 // (seqs * kv_heads * dim))
        return {"kind": kind, "seqs": seqs, "lo": max(1, hi // rng.choice([1, 2, 8])), "hi": hi,
                "q_heads": kv_heads * rng.choice([1, 4, 4, 8]), "kv_heads": kv_heads, "dim": dim, "page": page,
                "lens": lens}
    kv_heads, dim = rng.choice([(8, 128), (8, 128), (4, 128), (2, 128), (8, 64)])
    seqs = _log(rng, 1, 16)
    q_hi = min(_log(rng, 1, 2048), 4096 // seqs)
    old = _log(rng, 1, 12000 // max(1, seqs // 4))
    return {"kind": kind, "seqs": seqs, "q_lo": max(1, q_hi // rng.choice([1, 2, 4])), "q_hi": q_hi,
            "old_lo": old // rng.choice([1, 2, 4]), "old_hi": old, "q_heads": kv_heads * rng.choice([1, 2, 4, 4]),
            "kv_heads": kv_heads, "dim": dim, "page": page, "lens": lens}


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """(tokens before, new tokens) of every sequence: plain lists, a matter of the case."""
    r = random.Random(case["lens"])
    n = case["seqs"]
    if case["kind"] == "decode4":
        return [0] * n, [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    if case["kind"] == "prefill4":
        return ([r.randint(case["old_lo"], case["old_hi"]) for _ in range(n)],
                [r.randint(case["q_lo"], case["q_hi"]) for _ in range(n)])
    return ([r.randint(0, case["old"]) for _ in range(n)], [r.randint(case["lo"], case["hi"]) for _ in range(n)])


def _table(n_pos, rot, dev):
    """cos | sin of every position's angles, made in 64 bits: what a model keeps."""
    half = torch.arange(rot // 2, dtype=torch.float64, device=dev)
    angle = torch.arange(n_pos, dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (-2.0 * half / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _pages(total, page, g, dev):
    """Block tables of sequences of ``total`` tokens over a shuffled pool: (tables, pages)."""
    need = [-(-t // page) for t in total]
    order = torch.randperm(sum(need) + 3, generator=g, device=dev).to(torch.int32)
    at = torch.tensor([0] + need, device=dev).cumsum(0)[:-1]
    col = torch.arange(max(max(need), 1), device=dev)
    live = col < torch.tensor(need, device=dev)[:, None]
    return torch.where(live, order[(at[:, None] + col).clamp(max=len(order) - 1)], -1), sum(need) + 3


def _tiles(n_pages, heads, page, dim, g, dev):
    """A layer of 4-bit pages filled with the codes of normal values."""
    pool = torch.empty((n_pages, 2, heads, page // 16, 17 * dim // 2), dtype=torch.uint8, device=dev)
    # of 16 codes, how often each appears among normal values coded in blocks of 32
    p = torch.tensor([.10, .19, .17, .13, .17, .13, .08, .03], dtype=torch.float64)
    cut = (torch.cat([p, p]).cumsum(0) * 128).round().long()
    nibble = torch.searchsorted(cut, torch.arange(256), right=True).clamp(max=15).to(torch.uint8).to(dev)
    power = torch.tensor([124] * 16 + [125] * 160 + [126] * 72 + [127] * 8, dtype=torch.uint8, device=dev)
    n = 8 * dim
    step = max(1, (1 << 28) // (pool[0].numel()))
    for i in range(0, n_pages, step):
        part = pool[i:i + step]
        shape = part[..., :n].shape
        lo, hi = (nibble[torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.int32)] for _ in range(2))
        part[..., :n] = lo | (hi << 4)
        part[..., n:] = power[torch.randint(0, 256, part[..., n:].shape, generator=g, device=dev, dtype=torch.int32)]
    return pool


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    if case["kind"] == "rope":
        x = torch.randn((case["rows"], case["heads"], case["dim"]), generator=g, device=dev)
        s["x"] = x.to(_TYPES[case["type"]])
        s["table"] = _table(case["far"], case["rot"], dev)
        s["positions"] = torch.randint(0, case["far"], (case["rows"],), generator=g, device=dev, dtype=torch.int32)
        return s
    old, new = _lengths(case)
    total = [a + b for a, b in zip(old, new)]
    page, dim, heads = case["page"], case["dim"], case["kv_heads"]
    s["bt"], n_pages = _pages(total, page, g, dev)
    s["lens"], s["old"], s["most"], s["most_new"] = _ints(total, dev), _ints(old, dev), max(total), max(new)
    s["cu"] = _ints([sum(new[:i]) for i in range(len(new) + 1)], dev)
    # sequence and position of each new token, as the plain form indexes them
    s["seq"] = torch.repeat_interleave(torch.arange(len(new), device=dev), torch.tensor(new, device=dev))
    s["pos"] = torch.arange(sum(new), device=dev) - s["cu"][s["seq"]] + s["old"][s["seq"]]
    if case["kind"] in ("append8", "append4"):
        layers = case.get("layers", 1)
        x = torch.randn((layers, sum(new), 2, heads, dim), generator=g, device=dev, dtype=torch.bfloat16)
        x[:, :, 0, heads // 2] *= 8  # a head that stands out, as keys' do
        s["x"] = x
        if case["rot"]:
            s["table"] = _table(max(total), case["rot"], dev)
        if case["kind"] == "append8":
            s["pool"] = torch.randint(0, 127, (layers, n_pages, 2, heads, page, dim), generator=g, device=dev,
                                      dtype=torch.uint8)
            s["scales"] = torch.rand((layers, 2, heads), generator=g, device=dev) * 0.02 + 0.1
        else:
            s["pool"] = _tiles(n_pages, heads, page, dim, g, dev)[None]
        return s
    s["pool"] = _tiles(n_pages, heads, page, dim, g, dev)
    rows = case["seqs"] if case["kind"] == "decode4" else sum(new)
    s["q"] = torch.randn((rows, case["q_heads"], dim), generator=g, device=dev).mul_(2.0).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------ the plain forms

def _rotate(x, cos, sin, interleaved, transpose=False):
    """x in 32 bits [..., D], cos and sin [..., rot / 2] broadcast over the heads."""
    r = 2 * cos.shape[-1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    if transpose:
        sin = -sin
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _rotated(s):
    """New keys and values [L, n_tok, 2, H, D] with the keys rotated, as bf16 holds them."""
    x = s["x"]
    if not s["rot"]:
        return x
    half = s["rot"] // 2
    row = s["table"][s["pos"]][:, None, :]
    k = _rotate(x[:, :, 0].float(), row[..., :half], row[..., half:], s["interleaved"]).to(x.dtype)
    return torch.stack([k, x[:, :, 1]], 2)


def _code4(x):
    """bf16 [..., D] -> what 4 bits hold of it: e2m1 times the power of two that brings the
    largest of 32 values to 6 or below."""
    v = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(v.abs().amax(-1, keepdim=True))
    power = torch.exp2((e - torch.where(m <= 0.75, 3, 2)).clamp(min=-125).float())
    y = (v / power).abs()
    code = (y > 0.25).int() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5)
    held = torch.tensor(_E2M1[:8], device=x.device)[code].copysign(v) * power
    return held.flatten(-2).to(torch.bfloat16)


def _decode_tiles(tiles, dim):
    """[..., page / 16, 17 D / 2] bytes -> fp32 [..., page, D]."""
    c = tiles[..., :8 * dim].unflatten(-1, (dim // 32, 16, 16))
    both = torch.stack([c & 15, c >> 4], -1).flatten(-2)  # [..., page / 16, D / 32, 16, 32]
    power = torch.exp2(tiles[..., 8 * dim:].unflatten(-1, (dim // 32, 16)).float() - 127)
    v = torch.tensor(_E2M1, device=tiles.device)[both.int()] * power[..., None]
    return v.transpose(-3, -2).flatten(-2).flatten(-3, -2)


def _cached(pool, s):
    """(K, V) fp32 [B, H, positions, D] of the block tables' pages; positions past a sequence hold something."""
    v = _decode_tiles(pool[s["bt"].clamp(min=0)], s["dim"])  # [B, nb, 2, H, P, D]
    v = v.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)
    return v[0], v[1]


def _attend(q, k, v, hidden):
    """q [B, Hkv, rows, D], k and v [B, Hkv, T, D], hidden [B, 1, rows or 1, T] -> fp32 like q."""
    score = torch.matmul(q * q.shape[-1] ** -0.5, k.transpose(-1, -2)).masked_fill_(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def _plain(s):
    kind = s["kind"]
    if kind == "rope":
        half = s["rot"] // 2
        row = s["table"][s["positions"].long()][:, None, :]
        return _rotate(s["x"].float(), row[..., :half], row[..., half:], s["interleaved"],
                       s["transpose"]).to(s["x"].dtype)
    if kind == "append8":
        x = _rotated(s).float()
        scales = s["scales"] if s["static"] else x.abs().amax((1, 4)).clamp(min=1e-8) / 448.0
        codes = (x / scales[:, None, :, :, None]).to(torch.float8_e4m3fn)
        page = s["bt"][s["seq"], s["pos"] // s["page"]].long()
        s["pool"].permute(1, 4, 0, 2, 3, 5)[page, s["pos"] % s["page"]] = codes.view(torch.uint8).transpose(0, 1)
        return {"codes": s["pool"].view(torch.float8_e4m3fn), "scales": scales}
    if kind == "append4":
        x = _code4(_rotated(s)[0])
        k, v = (t.to(torch.bfloat16) for t in _cached(s["pool"][0], s))
        live = torch.arange(k.shape[2], device=k.device) < s["lens"][:, None]
        out = []
        for j, t in enumerate((k, v)):
            t = torch.where(live[:, None, :, None], t, 0)
            t.transpose(1, 2)[s["seq"], s["pos"]] = x[:, j]
            out.append(t[:, :, :s["most"]].contiguous())
        return {"k": out[0], "v": out[1]}
    heads, dim = s["kv_heads"], s["dim"]
    group = s["q_heads"] // heads
    k, v = _cached(s["pool"], s)
    at = torch.arange(k.shape[2], device=k.device)
    if kind == "decode4":
        hidden = (at >= s["lens"][:, None])[:, None, None]
        o = _attend(s["q"].float().unflatten(1, (heads, group)), k, v, hidden)
        return o.flatten(1, 2).to(torch.bfloat16)
    rows, first = s["most_new"], s["pos"] - s["old"][s["seq"]]
    q = torch.zeros((s["seqs"], rows, s["q_heads"], dim), device=k.device)
    q[s["seq"], first] = s["q"].float()
    q = q.view(-1, rows, heads, group, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    own_pos = s["old"][:, None] + torch.arange(rows, device=k.device).repeat(group)
    hidden = (at > own_pos[..., None]) | (at >= s["lens"][:, None, None])
    o = _attend(q, k, v, hidden[:, None])
    o = o.unflatten(2, (group, rows)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[s["seq"], first].to(torch.bfloat16)


def _own(s):
    from zenyx_amd import kv

    kind = s["kind"]
    if kind == "rope":
        return kv.rope(s["x"], s["table"], s["positions"], interleaved=s["interleaved"], transpose=s["transpose"])
    if kind == "append8":
        scales = kv.kv_rope_append(s["x"], s["table"], s["cu"], s["bt"], s["pool"],
                                   scales=s["scales"] if s["static"] else None, start_pos=s["old"],
                                   interleaved=s["interleaved"], static_scales=s["static"])
        return {"codes": s["pool"].view(torch.float8_e4m3fn), "scales": scales}
    if kind == "append4":
        kv.kv4_append(s["x"], s["cu"], s["bt"], s["pool"], start_pos=s["old"], table=s.get("table"),
                      interleaved=s["interleaved"] and "table" in s)
        k, v = kv.kv4_gather_dequant(s["pool"][0], s["bt"], s["lens"], s["most"])
        return {"k": k, "v": v}
    if kind == "decode4":
        return kv.paged_attention4_decode(s["q"], s["pool"], s["bt"], s["lens"])
    return kv.paged_attention4_prefill(s["q"], s["cu"], s["old"], s["pool"], s["bt"], s["lens"],
                                       max_q_per_seq=s["most_new"])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    dim = case["dim"]
    if case["kind"] == "rope":
        n = case["rows"] * case["heads"]
        size = 4 if case["type"] == "float32" else 2
        return {"bytes": n * dim * 2 * size + case["rows"] * (4 + 4 * case["rot"]), "flops": 3 * n * case["rot"]}
    old, new = _lengths(case)
    heads, tokens, total = case["kv_heads"], sum(new), sum(old) + sum(new)
    packed = 2 * heads * (dim // 2 + dim // 32)  # bytes of a token's 4-bit K and V
    if case["kind"] == "append8":
        n = case["layers"] * tokens * 2 * heads * dim
        return {"bytes": 3 * n + 4 * tokens * case["rot"], "flops": 5 * n}
    if case["kind"] == "append4":
        n = tokens * 2 * heads * dim
        back = case["seqs"] * max(a + b for a, b in zip(old, new)) * 2 * heads * dim
        return {"bytes": 2 * n + tokens * packed + 4 * tokens * case["rot"] + total * packed + 2 * back,
                "flops": 5 * n + back}
    row = case["q_heads"] * dim
    if case["kind"] == "decode4":
        return {"bytes": total * packed + 4 * case["seqs"] * row + 4 * total // case["page"],
                "flops": 4 * total * row}
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(old, new))
    return {"bytes": total * packed + 4 * tokens * row + 4 * total // case["page"], "flops": 4 * pairs * row}


# ------------------------------------------------------------------ the definitions in 64 bits

def _turn64(x, table, positions, interleaved, sign):
    """Each pair of channels as one complex number, turned by its position's angle."""
    x = x.double().clone()
    n = table.shape[1] // 2
    t = table.double()[positions.long()]
    z = torch.complex(t[:, :n], sign * t[:, n:])[:, None]
    first = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    second = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    w = torch.complex(x[..., first], x[..., second]) * z
    x[..., first], x[..., second] = w.real, w.imag
    return x


def _near4(x):
    """64-bit [..., 32] -> the nearest e2m1 value (the even code of two as near) times the block's power."""
    grid = torch.tensor(_E2M1[:8], dtype=torch.float64, device=x.device)
    top = x.abs().amax(-1, keepdim=True)
    power = 2.0 ** torch.ceil(torch.log2(top.clamp(min=2.0 ** -130) / 6.0)).clamp(min=-125.0)
    power = torch.where(power * 6.0 < top, power * 2, power)
    y = x.abs() / power
    hi = torch.searchsorted(grid, y.contiguous()).clamp(1, 7)
    below, above = y - grid[hi - 1], grid[hi] - y
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return torch.where(up, grid[hi], grid[hi - 1]) * power * torch.where(torch.signbit(x), -1.0, 1.0)


def _page64(pool, pages, kv, dim):
    """K (0) or V (1) of a list of pages in 64 bits: [H, positions, D]."""
    t = pool[pages.long(), kv]  # [nb, H, P / 16, bytes]
    nb, heads, n = t.shape[:3]
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=t.device)
    code = t[..., :8 * dim].reshape(nb, heads, n, dim // 32, 16, 16).long()
    v = torch.empty((nb, heads, n, dim // 32, 16, 32), dtype=torch.float64, device=t.device)
    v[..., 0::2], v[..., 1::2] = grid[code % 16], grid[code // 16]
    v *= 2.0 ** (t[..., 8 * dim:].reshape(nb, heads, n, dim // 32, 16, 1).double() - 127.0)
    return v.permute(1, 0, 2, 4, 3, 5).reshape(heads, -1, dim)


def exact(case, seed):
    s = prepare(case, seed)
    kind, dim = case["kind"], case["dim"]
    if kind == "rope":
        return _turn64(s["x"], s["table"], s["positions"], s["interleaved"], -1.0 if s["transpose"] else 1.0)
    old, new = _lengths(case)
    if kind in ("append8", "append4"):
        x = s["x"].double()
        if s["rot"]:
            for layer in range(x.shape[0]):
                x[layer, :, 0] = _turn64(s["x"][layer, :, 0], s["table"], s["pos"], s["interleaved"],
                                         1.0).to(torch.bfloat16).double()
        page, row = s["bt"][s["seq"], s["pos"] // s["page"]].long(), s["pos"] % s["page"]
    if kind == "append8":
        scales = s["scales"].double() if s["static"] else x.abs().amax(1).amax(-1) / 448.0
        pool = s["pool"].view(torch.float8_e4m3fn).double()
        for layer in range(x.shape[0]):
            y = (x[layer] / scales[layer][None, :, :, None]).float().to(torch.float8_e4m3fn).double()
            pool[layer].transpose(1, 3)[page, row] = y.transpose(1, 2)
        return {"codes": pool, "scales": scales}
    if kind == "append4":
        held = _near4(x[0].unflatten(-1, (-1, 32))).flatten(-2)
        out = torch.zeros((2, case["seqs"], case["kv_heads"], s["most"], dim), dtype=torch.float64, device=x.device)
        at = 0
        for b, (a, n) in enumerate(zip(old, new)):
            pages = s["bt"][b, :-(-(a + n) // s["page"])]
            for j in range(2):
                out[j, b, :, :a] = _page64(s["pool"][0], pages, j, dim)[:, :a]
                out[j, b, :, a:a + n] = held[at:at + n, j].transpose(0, 1)
            at += n
        return {"k": out[0], "v": out[1]}
    heads, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    at = 0
    for b, (a, n) in enumerate(zip(old, new)):
        pages = s["bt"][b, :-(-(a + n) // s["page"])]
        k, v = (_page64(s["pool"], pages, j, dim)[:, :a + n] for j in range(2))
        rows = 1 if kind == "decode4" else n
        q = s["q"][at:at + rows].double().view(rows, heads, group, dim)
        for h in range(heads):
            score = torch.einsum("rgd,td->rgt", q[:, h], k[h]) / math.sqrt(dim)
            if kind == "prefill4":
                late = torch.arange(a + n, device=k.device) > a + torch.arange(n, device=k.device)[:, None]
                score.masked_fill_(late[:, None], -math.inf)
            out[at:at + rows, h * group:(h + 1) * group] = torch.einsum("rgt,td->rgd", torch.softmax(score, -1), v[h])
        at += rows
    return out
