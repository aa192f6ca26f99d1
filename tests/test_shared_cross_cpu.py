"""What attention to shared pages and cross attention refuse, before any GPU is touched (the library checks
its arguments on the host and launches nothing)."""
import pytest

from zenyx_amd import _native as N

P = 4096  # stands for a 16-byte aligned device pointer: a refused call does not follow it


@pytest.fixture(scope="module")
def lib():
    return N.load()


def shared_args(four, **kw):
    a = dict(q=P, n_q=4, cu_q=None, Hq=8, pool=P, n_pages=9, Hkv=2, D=128, page=16, scales=P, bt=P, mb=8, lens=P, B=4,
             cu_group=P, shared=P, G=1, most=1, causal=1, sm=0.1, out=P, err=None, ws=P, wsb=1 << 40, st=None)
    a.update(kw)
    if four:
        del a["scales"]
    return list(a.values())


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("kw, rc", [
    (dict(q=None), N.ZX_ERR_INVALID), (dict(pool=None), N.ZX_ERR_INVALID), (dict(bt=None), N.ZX_ERR_INVALID),
    (dict(lens=None), N.ZX_ERR_INVALID), (dict(out=None), N.ZX_ERR_INVALID), (dict(cu_group=None), N.ZX_ERR_INVALID),
    (dict(shared=None), N.ZX_ERR_INVALID), (dict(q=P + 8), N.ZX_ERR_INVALID), (dict(pool=P + 4), N.ZX_ERR_INVALID),
    (dict(out=P + 2), N.ZX_ERR_INVALID), (dict(ws=P + 8), N.ZX_ERR_INVALID), (dict(Hq=7), N.ZX_ERR_INVALID),
    (dict(Hq=0), N.ZX_ERR_INVALID), (dict(Hkv=0), N.ZX_ERR_INVALID), (dict(n_pages=0), N.ZX_ERR_INVALID),
    (dict(mb=0), N.ZX_ERR_INVALID), (dict(B=0, n_q=0), N.ZX_ERR_INVALID), (dict(G=-1), N.ZX_ERR_INVALID),
    (dict(G=5), N.ZX_ERR_INVALID), (dict(n_q=5), N.ZX_ERR_INVALID), (dict(n_q=-1), N.ZX_ERR_INVALID),
    (dict(most=-1), N.ZX_ERR_INVALID), (dict(D=96), N.ZX_ERR_UNSUPPORTED), (dict(D=32), N.ZX_ERR_UNSUPPORTED),
    (dict(page=24), N.ZX_ERR_UNSUPPORTED), (dict(page=8), N.ZX_ERR_UNSUPPORTED),
    (dict(mb=1 << 27), N.ZX_ERR_INVALID), (dict(B=65536, n_q=65536), N.ZX_ERR_UNSUPPORTED),
    (dict(cu_q=P, n_q=1 << 30), N.ZX_ERR_UNSUPPORTED),
    (dict(cu_q=P, n_q=1 << 26, most=1 << 26, B=60000, mb=1 << 20), N.ZX_ERR_UNSUPPORTED),
    (dict(ws=None), N.ZX_ERR_WORKSPACE), (dict(wsb=100), N.ZX_ERR_WORKSPACE)])
def test_shared_refusals(lib, four, kw, rc):
    f = lib.zx_paged_attention4_shared if four else lib.zx_paged_attention_shared
    assert f(*shared_args(four, **kw)) == rc
    assert (b"attention4_shared" if four else b"attention_shared") in lib.zx_last_error()


def test_shared_calls_without_rows(lib):
    for kw in (dict(cu_q=P, n_q=0), dict(cu_q=P, most=0)):
        assert lib.zx_paged_attention_shared(*shared_args(False, q=None, out=None, ws=None, **kw)) == N.ZX_OK
        assert lib.zx_paged_attention4_shared(*shared_args(True, q=None, out=None, ws=None, **kw)) == N.ZX_OK
    assert lib.zx_paged_attention_shared(*shared_args(False, scales=None)) == N.ZX_ERR_INVALID


def test_shared_workspace(lib):
    """Grows with what a call can need, 0 for what it refuses, and does not depend on how wide tables are once
    the chip is full."""
    def size(n_q=64, B=64, G=1, Hq=32, Hkv=8, D=128, page=16, mb=2048, most=1, four=False):
        f = lib.zx_paged_attention4_shared_workspace_bytes if four else lib.zx_paged_attention_shared_workspace_bytes
        return f(n_q, B, G, Hq, Hkv, D, page, mb, most)
    for bad in (dict(D=96), dict(Hq=30), dict(n_q=0), dict(most=0), dict(B=0), dict(mb=0), dict(page=0), dict(G=-1)):
        assert size(**bad) == 0
    for four in (False, True):
        assert 0 < size(four=four) == size(mb=1 << 16, four=four) < 1 << 27
        assert size(mb=1, four=four) <= size(four=four)
        assert size(n_q=256, most=4, four=four) > size(four=four)


def cross_args(**kw):
    a = dict(dtype=0, q=P, n_q=4, qr=128, qh=64, Hq=2, k=P, kr=128, kh=64, v=P, vr=128, vh=64, n_k=6, Hkv=2, D=64, cu_q=P,
             cu_k=P, k_lens=None, B=2, mq=4, mk=6, sm=0.1, flags=0, out=P, lse=None, err=None, ws=None, wsb=0, st=None)
    a.update(kw)
    return list(a.values())


def grad_args(**kw):
    a = dict(dtype=0, g=P, gr=128, gh=64, q=P, n_q=4, qr=128, qh=64, Hq=2, k=P, kr=128, kh=64, v=P, vr=128, vh=64, n_k=6,
             Hkv=2, D=64, out=P, lse=P, cu_q=P, cu_k=P, k_lens=None, B=2, mq=4, mk=6, sm=0.1, dq=P, dk=P, dv=P, err=None,
             ws=P, wsb=1 << 30, st=None)
    a.update(kw)
    return list(a.values())


BOTH = [(dict(dtype=2), N.ZX_ERR_INVALID), (dict(D=96), N.ZX_ERR_UNSUPPORTED), (dict(D=256), N.ZX_ERR_UNSUPPORTED),
        (dict(Hq=3), N.ZX_ERR_INVALID), (dict(Hq=0), N.ZX_ERR_INVALID), (dict(Hkv=0), N.ZX_ERR_INVALID),
        (dict(B=0), N.ZX_ERR_INVALID), (dict(n_q=-1), N.ZX_ERR_INVALID), (dict(n_k=-1), N.ZX_ERR_INVALID),
        (dict(mq=-1), N.ZX_ERR_INVALID), (dict(mk=-1), N.ZX_ERR_INVALID), (dict(q=None), N.ZX_ERR_INVALID),
        (dict(k=None), N.ZX_ERR_INVALID), (dict(v=None), N.ZX_ERR_INVALID), (dict(cu_q=None), N.ZX_ERR_INVALID),
        (dict(cu_k=None), N.ZX_ERR_INVALID), (dict(out=None), N.ZX_ERR_INVALID), (dict(q=P + 8), N.ZX_ERR_INVALID),
        (dict(k=P + 2), N.ZX_ERR_INVALID), (dict(v=P + 4), N.ZX_ERR_INVALID), (dict(out=P + 8), N.ZX_ERR_INVALID),
        (dict(qr=130), N.ZX_ERR_INVALID), (dict(kh=-64), N.ZX_ERR_INVALID), (dict(vr=-128), N.ZX_ERR_INVALID),
        (dict(kr=1 << 23), N.ZX_ERR_UNSUPPORTED), (dict(qh=1 << 29, Hq=4), N.ZX_ERR_UNSUPPORTED),
        (dict(n_q=1 << 30), N.ZX_ERR_UNSUPPORTED), (dict(n_k=1 << 31), N.ZX_ERR_UNSUPPORTED),
        (dict(B=1 << 30, mq=1 << 20, n_q=1 << 20), N.ZX_ERR_UNSUPPORTED)]


@pytest.mark.parametrize("kw, rc", BOTH + [(dict(flags=2), N.ZX_ERR_INVALID), (dict(ws=P + 8), N.ZX_ERR_INVALID),
                                           (dict(n_k=4000, mk=4000), N.ZX_ERR_WORKSPACE)])
def test_cross_refusals(lib, kw, rc):
    assert lib.zx_cross_attention(*cross_args(**kw)) == rc
    assert b"cross_attention" in lib.zx_last_error()


@pytest.mark.parametrize("kw, rc", BOTH + [
    (dict(g=None), N.ZX_ERR_INVALID), (dict(g=P + 8), N.ZX_ERR_INVALID), (dict(gr=4), N.ZX_ERR_INVALID),
    (dict(lse=None), N.ZX_ERR_INVALID), (dict(dq=None), N.ZX_ERR_INVALID), (dict(dk=None), N.ZX_ERR_INVALID),
    (dict(dv=None), N.ZX_ERR_INVALID), (dict(dq=P + 8), N.ZX_ERR_INVALID), (dict(dk=P + 8), N.ZX_ERR_INVALID),
    (dict(dv=P + 8), N.ZX_ERR_INVALID), (dict(ws=P + 8), N.ZX_ERR_INVALID), (dict(ws=None), N.ZX_ERR_WORKSPACE),
    (dict(wsb=16), N.ZX_ERR_WORKSPACE)])
def test_cross_gradient_refusals(lib, kw, rc):
    assert lib.zx_cross_attention_backward(*grad_args(**kw)) == rc
    assert b"cross_attention_backward" in lib.zx_last_error()


def test_cross_calls_without_rows(lib):
    assert lib.zx_cross_attention(*cross_args(n_q=0, q=None, out=None)) == N.ZX_OK
    assert lib.zx_cross_attention_backward(*grad_args(n_q=0, n_k=0, q=None, k=None, v=None, g=None, out=None, dq=None,
                                                      dk=None, dv=None, ws=None, wsb=0)) == N.ZX_OK
