"""CPU oracle of the rotary positions and the 4-bit KV pages -- TEST INFRASTRUCTURE ONLY (see
oracle.py).  Plain numpy from the definitions: the nearest code is searched for, not computed."""
from __future__ import annotations

import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
TILE = 16  # tokens
NAN_BYTE = 255
TOO_LARGE = 1.75 * 2.0 ** 127


def bf16(x) -> np.ndarray:
    """float64/32 -> the nearest bf16 value (ties to even), as float64; x exact in float32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32).astype(np.float64)
    return np.where(np.isnan(x), np.nan, r)


def rotate_f32(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, interleaved: bool) -> np.ndarray:
    """float32 rows [n, H, D] turned with cos / sin [n, rot / 2] (float32): every product and
    their sum rounded to float32."""
    x = np.ascontiguousarray(x, np.float32)
    half = cos.shape[1]
    y = x.copy()
    a = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    c, s = cos[:, None].astype(np.float32), sin[:, None].astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def encode_block(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """bf16 values [..., 32] -> (codes [..., 32] 0..15, power bytes [...])."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max(-1)
        bad = ~(top < TOO_LARGE)
    top = np.where(bad, 1.0, top)
    e = np.full(top.shape, -125)
    for k in range(-125, 128):  # the smallest power that brings the largest to 6 or below
        e = np.where(top > 6 * 2.0 ** (k - 1), np.maximum(k, -125), e)
    y = np.where(bad[..., None], 0.0, np.abs(x)) / 2.0 ** e[..., None]
    # of the two codes as near, the even one: a hair's preference decides exact ties only
    dist = np.abs(y[..., None] - E2M1) + np.where(np.arange(8) % 2, 1e-12, 0.0)
    code = dist.argmin(-1).astype(np.uint8)
    code |= np.where(np.signbit(x) & ~bad[..., None], 8, 0).astype(np.uint8)
    return code, np.where(bad, NAN_BYTE, e + 127).astype(np.uint8)


def decode_block(code: np.ndarray, byte: np.ndarray) -> np.ndarray:
    v = np.where(code & 8, -1.0, 1.0) * E2M1[code & 7] * 2.0 ** (byte.astype(np.float64) - 127)[..., None]
    return np.where((byte == NAN_BYTE)[..., None], np.nan, v)


def store(pool: np.ndarray, page: int, kv: int, h: int, row: int, x: np.ndarray) -> None:
    """One token's [D] values into a layer's pool [n_pages, 2, H, P / 16, 17 D / 2]."""
    D = x.shape[0]
    code, byte = encode_block(x.reshape(-1, 32))
    tile, n = pool[page, kv, h, row // TILE], row % TILE
    packed = code[:, 0::2] | (code[:, 1::2] << 4)  # [D / 32, 16]
    tile[:8 * D].reshape(D // 32, TILE, 16)[:, n] = packed
    tile[8 * D:].reshape(D // 32, TILE)[:, n] = byte


def load(pool: np.ndarray, bt_row: np.ndarray, n: int, kv: int) -> tuple[np.ndarray, np.ndarray]:
    """K or V of a sequence's first n positions: ([H, n, D] float64, [n] whether the page is good)."""
    n_pages, _, H, tiles, nb = pool.shape
    D, P = nb * 2 // 17, tiles * TILE
    t = np.arange(n)
    page = bt_row[t // P].astype(np.int64)
    ok = (page >= 0) & (page < n_pages)
    tile = pool[np.where(ok, page, 0), kv, :, (t % P) // TILE]  # [n, H, bytes]
    code = tile[..., :8 * D].reshape(n, H, D // 32, TILE, 16)[t, :, :, t % TILE]
    byte = tile[..., 8 * D:].reshape(n, H, D // 32, TILE)[t, :, :, t % TILE]
    full = np.stack([code & 15, code >> 4], -1).reshape(n, H, D // 32, 32)
    return decode_block(full, byte).reshape(n, H, D).transpose(1, 0, 2), ok


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, seen: np.ndarray, sm: float):
    """q [rows, D], k and v [n, D], seen [rows, n] -> (rows [rows, D] in float64, the largest
    sum |q k| a row meets, the largest |v| it meets)."""
    s = q @ k.T * sm
    s = np.where(seen, s, -np.inf)
    top = s.max(-1, initial=-np.inf, keepdims=True)
    with np.errstate(invalid="ignore"):
        p = np.where(seen, np.exp(s - np.where(np.isneginf(top), 0, top)), 0.0)
    total = p.sum(-1, keepdims=True)
    with np.errstate(invalid="ignore"):
        out = (p @ np.where(seen.any(0)[:, None], v, 0)) / np.where(total == 0, 1.0, total)
    qk = np.where(seen, np.abs(q) @ np.abs(k).T, 0.0).max(-1, initial=0.0)
    vm = np.where(seen.any(0)[:, None], np.abs(v), 0.0).max(0, initial=0.0)
    return out, qk, vm
