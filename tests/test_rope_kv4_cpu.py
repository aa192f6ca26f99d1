"""What rotary positions and 4-bit pages refuse, before any GPU is touched (the library checks its
arguments on the host and launches nothing), and the oracle of the 4-bit format by itself."""
import ctypes

import numpy as np
import pytest

from oracle import kv4 as R
from zenyx_amd import _native as N

P = 4096  # stands for a 16-byte aligned device pointer: a refused call does not follow it


@pytest.fixture(scope="module")
def lib():
    return N.load()


def rope_args(**kw):
    a = dict(x=P, dtype=0, n=4, H=2, D=64, xr=128, xh=64, table=P, n_pos=10, rot=64, pos=P, flags=0, out=2 * P,
             outr=128, outh=64, err=None, st=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, rc", [
    (dict(dtype=3), N.ZX_ERR_INVALID), (dict(flags=1), N.ZX_ERR_INVALID), (dict(D=68), N.ZX_ERR_UNSUPPORTED),
    (dict(rot=24), N.ZX_ERR_UNSUPPORTED), (dict(rot=0), N.ZX_ERR_INVALID), (dict(rot=80), N.ZX_ERR_INVALID),
    (dict(n_pos=0), N.ZX_ERR_INVALID), (dict(n_pos=(1 << 31) + 1), N.ZX_ERR_INVALID), (dict(n=-1), N.ZX_ERR_INVALID),
    (dict(x=None), N.ZX_ERR_INVALID), (dict(table=None), N.ZX_ERR_INVALID), (dict(pos=None), N.ZX_ERR_INVALID),
    (dict(table=P + 4), N.ZX_ERR_INVALID), (dict(x=P + 2), N.ZX_ERR_INVALID), (dict(xh=65), N.ZX_ERR_INVALID),
    (dict(xr=-128), N.ZX_ERR_INVALID), (dict(out=P, outr=256), N.ZX_ERR_INVALID),
    (dict(n=(1 << 31) - 1, H=64), N.ZX_ERR_UNSUPPORTED)])
def test_rope_refusals(lib, kw, rc):
    assert lib.zx_rope(*rope_args(**kw)) == rc
    assert b"rope" in lib.zx_last_error()


def test_rope_of_no_rows(lib):
    assert lib.zx_rope(*rope_args(n=0, x=None, out=None, pos=None)) == N.ZX_OK


def append_args(four, **kw):
    D = kw.get("D", 64)
    a = dict(x=P, xl=64 * 4 * D, L=1, T=64, H=2, D=D, table=P, n_pos=100, rot=64, cu=P, start=None, B=2, bt=P, mb=4,
             page=16, pool=P, pl=1 << 30, n_pages=9, scales=P, flags=0, err=None, ws=P, wsb=1 << 30, st=None)
    a.update(kw)
    if four:
        del a["scales"]
    return list(a.values())


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("kw, rc", [
    (dict(flags=64), N.ZX_ERR_INVALID), (dict(D=96, rot=64), N.ZX_ERR_UNSUPPORTED), (dict(x=None), N.ZX_ERR_INVALID),
    (dict(cu=None), N.ZX_ERR_INVALID), (dict(bt=None), N.ZX_ERR_INVALID), (dict(pool=None), N.ZX_ERR_INVALID),
    (dict(pool=P + 8), N.ZX_ERR_INVALID), (dict(x=P + 8), N.ZX_ERR_INVALID), (dict(T=1 << 31), N.ZX_ERR_INVALID),
    (dict(T=-1), N.ZX_ERR_INVALID), (dict(B=0), N.ZX_ERR_INVALID), (dict(mb=0), N.ZX_ERR_INVALID),
    (dict(page=0), N.ZX_ERR_INVALID), (dict(n_pages=0), N.ZX_ERR_INVALID), (dict(n_pages=1 << 31), N.ZX_ERR_INVALID),
    (dict(H=0), N.ZX_ERR_INVALID), (dict(L=0), N.ZX_ERR_INVALID), (dict(L=2, xl=8), N.ZX_ERR_INVALID),
    (dict(L=2, pl=16), N.ZX_ERR_INVALID), (dict(rot=40), N.ZX_ERR_UNSUPPORTED), (dict(rot=128), N.ZX_ERR_INVALID),
    (dict(n_pos=0), N.ZX_ERR_INVALID), (dict(ws=P + 8), N.ZX_ERR_INVALID),
    (dict(T=50000, xl=1 << 30, ws=None), N.ZX_ERR_WORKSPACE), (dict(T=50000, xl=1 << 30, wsb=8), N.ZX_ERR_WORKSPACE)])
def test_append_refusals(lib, four, kw, rc):
    f = lib.zx_kv4_append if four else lib.zx_kv_rope_append
    assert f(*append_args(four, **kw)) == rc
    assert (b"kv4_append" if four else b"kv_rope_append") in lib.zx_last_error()


def test_append_refusals_of_one_kind(lib):
    assert lib.zx_kv_rope_append(*append_args(False, flags=4)) == N.ZX_ERR_INVALID  # saturate, dynamic scales
    assert lib.zx_kv_rope_append(*append_args(False, flags=2 | 8)) == N.ZX_ERR_INVALID  # one pass and two
    assert lib.zx_kv_rope_append(*append_args(False, table=None)) == N.ZX_ERR_INVALID
    assert lib.zx_kv_rope_append(*append_args(False, H=40, D=128)) == N.ZX_ERR_UNSUPPORTED
    assert lib.zx_kv4_append(*append_args(True, flags=1)) == N.ZX_ERR_INVALID  # no scales to be static
    assert lib.zx_kv4_append(*append_args(True, page=24)) == N.ZX_ERR_UNSUPPORTED
    assert lib.zx_kv4_append(*append_args(True, table=None, flags=16)) == N.ZX_ERR_INVALID
    assert lib.zx_kv4_append(*append_args(True, T=0, x=None, ws=None)) == N.ZX_OK


def decode_args(**kw):
    a = dict(q=P, Hq=4, pool=P, n_pages=9, Hkv=2, D=128, page=16, bt=P, mb=4, sl=P, B=2, sm=0.1, out=P, err=None, ws=P,
             wsb=1 << 30, st=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, rc", [
    (dict(D=96), N.ZX_ERR_UNSUPPORTED), (dict(page=8), N.ZX_ERR_UNSUPPORTED), (dict(Hq=5), N.ZX_ERR_INVALID),
    (dict(Hq=0), N.ZX_ERR_INVALID), (dict(B=0), N.ZX_ERR_INVALID), (dict(mb=0), N.ZX_ERR_INVALID),
    (dict(n_pages=0), N.ZX_ERR_INVALID), (dict(q=None), N.ZX_ERR_INVALID), (dict(sl=None), N.ZX_ERR_INVALID),
    (dict(q=P + 8), N.ZX_ERR_INVALID), (dict(out=P + 2), N.ZX_ERR_INVALID), (dict(pool=P + 4), N.ZX_ERR_INVALID),
    (dict(B=65536), N.ZX_ERR_UNSUPPORTED), (dict(ws=None), N.ZX_ERR_WORKSPACE), (dict(wsb=64), N.ZX_ERR_WORKSPACE)])
def test_decode_refusals(lib, kw, rc):
    assert lib.zx_paged_attention4_decode(*decode_args(**kw)) == rc
    assert b"paged_attention4_decode" in lib.zx_last_error()


def prefill_args(**kw):
    a = dict(q=P, n_q=10, cu=P, qp=P, Hq=4, pool=P, n_pages=9, Hkv=2, D=128, page=16, bt=P, mb=4, kl=P, B=2, mq=5,
             causal=1, sm=0.1, flags=0, out=P, err=None, ws=None, wsb=0, st=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, rc", [
    (dict(D=96), N.ZX_ERR_UNSUPPORTED), (dict(page=40), N.ZX_ERR_UNSUPPORTED), (dict(Hq=3), N.ZX_ERR_INVALID),
    (dict(flags=8), N.ZX_ERR_INVALID), (dict(n_q=-1), N.ZX_ERR_INVALID), (dict(mq=-1), N.ZX_ERR_INVALID),
    (dict(B=0), N.ZX_ERR_INVALID), (dict(mb=1 << 27), N.ZX_ERR_INVALID), (dict(cu=None), N.ZX_ERR_INVALID),
    (dict(kl=None), N.ZX_ERR_INVALID), (dict(q=P + 8), N.ZX_ERR_INVALID), (dict(ws=P + 8), N.ZX_ERR_INVALID),
    (dict(n_q=1 << 30, mq=1 << 30, B=1 << 20), N.ZX_ERR_UNSUPPORTED)])
def test_prefill_refusals(lib, kw, rc):
    assert lib.zx_paged_attention4_prefill(*prefill_args(**kw)) == rc
    assert b"paged_attention4_prefill" in lib.zx_last_error()


def test_prefill_of_no_rows(lib):
    assert lib.zx_paged_attention4_prefill(*prefill_args(n_q=0, q=None, out=None)) == N.ZX_OK
    assert lib.zx_paged_attention4_prefill(*prefill_args(mq=0)) == N.ZX_OK


def test_gather_refusals(lib):
    a = [P, 9, 2, 128, 16, P, 4, P, 2, 64, P, P, None, None]

    def call(**kw):
        b = list(a)
        for i, v in kw.items():
            b[int(i[1:])] = v
        return lib.zx_kv4_gather_dequant(*b)
    assert call(_3=80) == N.ZX_ERR_UNSUPPORTED and call(_4=20) == N.ZX_ERR_UNSUPPORTED
    assert call(_0=None) == N.ZX_ERR_INVALID and call(_10=P + 2) == N.ZX_ERR_INVALID and call(_9=-1) == N.ZX_ERR_INVALID
    assert call(_9=0, _10=None) == N.ZX_OK


def test_workspace_queries(lib):
    assert lib.zx_kv4_append_workspace_bytes(1, 0, 8) == 0 and lib.zx_kv4_append_workspace_bytes(1, 33, 8) == 0
    assert lib.zx_kv4_append_workspace_bytes(4, 50000, 8) >= 50000 * 8
    assert lib.zx_kv_rope_append_workspace_bytes(1, -5, 8, 128, 0) == 0
    assert lib.zx_kv_rope_append_workspace_bytes(1, 64, 8, 128, 1) == 0  # static scales, few tokens: none
    assert lib.zx_kv_rope_append_workspace_bytes(1, 64, 8, 128, 0) >= 16 * 4
    assert lib.zx_kv_rope_append_workspace_bytes(1, 50000, 8, 128, 1) >= 50000 * 8
    assert lib.zx_paged_attention4_decode_workspace_bytes(4, 32, 8, 96, 10, 16) == 0
    assert lib.zx_paged_attention4_decode_workspace_bytes(4, 32, 8, 128, 10, 24) == 0
    assert lib.zx_paged_attention4_prefill_workspace_bytes(32, 8, 128, 16, 1024, 1, 4) > 0
    assert lib.zx_paged_attention4_prefill_workspace_bytes(32, 8, 128, 16, 1024, 64, 2048) == 0


def test_oracle_codes():
    x = np.zeros((4, 32))
    x[0, :9] = [6, -6, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25]  # ties go to the even code
    x[1, :2] = [6.0001, -0.1]   # just past 6: the next power
    x[2, 0] = np.nan
    x[3, 0] = R.TOO_LARGE
    code, byte = R.encode_block(x)
    assert byte.tolist() == [127, 128, 255, 255]
    assert R.decode_block(code, byte)[0, :9].tolist() == [6, -6, 4, 4, 2, 2, 1, 1, 0]
    assert np.isnan(R.decode_block(code, byte)[2:]).all()
    code, byte = R.encode_block(np.zeros((1, 32)))
    assert byte[0] == 2 and not code.any()
    # a half step of the largest binade (2 units of 6) is the largest error
    y = np.random.default_rng(0).standard_normal((200, 32))
    c, b = R.encode_block(R.bf16(y))
    assert np.all(np.abs(R.decode_block(c, b) - R.bf16(y)) <= 2.0 ** (b.astype(float) - 127)[:, None])


def test_oracle_tiles():
    rng = np.random.default_rng(1)
    pool = np.zeros((3, 2, 2, 2, 17 * 64 // 2), np.uint8)  # pages of 32
    x = R.bf16(rng.standard_normal((2, 2, 40, 64)))
    bt = np.array([2, 0], np.int32)
    for kv in range(2):
        for h in range(2):
            for t in range(40):
                R.store(pool, bt[t // 32], kv, h, t % 32, x[kv, h, t])
    for kv in range(2):
        got, ok = R.load(pool, bt, 40, kv)
        c, b = R.encode_block(x[kv].reshape(2, 40, 2, 32))
        assert ok.all() and np.array_equal(got, R.decode_block(c, b).reshape(2, 40, 64))
    assert not pool[1].any()


def test_ctypes_signatures_cover_the_new_entry_points():
    for name in ("zx_rope", "zx_rope_table", "zx_kv_rope_append", "zx_kv4_append", "zx_kv4_gather_dequant",
                 "zx_paged_attention4_decode", "zx_paged_attention4_prefill"):
        assert name in N.SIGNATURES and isinstance(getattr(N.load(), name), ctypes._CFuncPtr)


@pytest.mark.parametrize("n, H, D, row, head", [
    (4, 2, 64, 64, 64),    # row 1 of head 0 is row 0 of head 1
    (2, 2, 64, 72, 64),    # half-way into it
    (2, 2, 64, 64, 72), (3, 5, 64, 256, 64), (2, 3, 64, 144, 128), (2, 8, 64, 192 + 56, 64),
    (1000, 3, 64, 64, 64 * 999), (2, 2, 64, 0, 64), (2, 2, 64, 128, 0), (5, 4, 64, 72, 96)])
def test_rope_refuses_an_out_whose_rows_overlap(lib, n, H, D, row, head):
    cells = [(i * row + j * head) for i in range(n) for j in range(H)]
    cells.sort()
    assert min(b - a for a, b in zip(cells, cells[1:])) < D  # they do
    assert lib.zx_rope(*rope_args(n=n, H=H, D=D, xr=H * D, xh=D, outr=row, outh=head)) == N.ZX_ERR_INVALID
    assert b"overlap" in lib.zx_last_error()
    assert lib.zx_rope(*rope_args(n=n, H=H, D=D, xr=row, xh=head, outr=row, outh=head, out=P)) == N.ZX_ERR_INVALID


@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_refuses_a_workspace_off_16_bytes(lib, D):
    """Its parts and tables are read by 8 bytes, as prefill's, which refuses it too."""
    for off in (4, 8):
        assert lib.zx_paged_attention4_decode(*decode_args(ws=P + off, D=D)) == N.ZX_ERR_INVALID
        assert b"workspace" in lib.zx_last_error()
