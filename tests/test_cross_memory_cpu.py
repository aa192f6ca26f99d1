"""Where cross attention's outputs may lie, checked by the library on the host: calls that it takes are not
made here."""
import pytest

from test_shared_cross_cpu import cross_args, grad_args

from zenyx_amd import _native as N

P = 1 << 20  # stands for a device pointer
ROW = 128 * 2  # bytes of a row of 2 heads of 64


@pytest.fixture(scope="module")
def lib():
    return N.load()


def at(q=P, k=P + 0x10000, v=P + 0x20000, out=P + 0x30000):
    return dict(q=q, k=k, v=v, out=out)


@pytest.mark.parametrize("kw, what", [
    (dict(out=P + 16), "q"), (dict(out=P - 16), "q"), (dict(out=P + 3 * ROW), "q"), (dict(out=P - 4 * ROW + 16), "q"),
    (dict(out=P, qr=192), "q"), (dict(out=P, qr=64, qh=256), "q"),  # q's address, other strides
    (dict(out=P + 0x10000), "k"), (dict(out=P + 0x10000 + 6 * ROW - 16), "k"), (dict(out=P + 0x10000 - 16), "k"),
    (dict(out=P + 0x20000 + 16), "v"), (dict(out=P, k=P), "k"), (dict(out=P, v=P + ROW), "v"),
    (dict(out=P + 0x10000 + 4096, kr=1 << 22), "k")])
def test_out_in_the_inputs_memory_is_refused(lib, kw, what):
    given = at()
    given.update(kw)
    assert lib.zx_cross_attention(*cross_args(**given)) == N.ZX_ERR_INVALID
    text = lib.zx_last_error()
    assert b"memory" in text and (b"out must be q itself" if what == "q" else b"k's or v's") in text


@pytest.mark.parametrize("kw", [
    dict(dq=P), dict(dq=P + 3 * ROW), dict(dq=P + 0x40000), dict(dq=P + 0x10000), dict(dq=P + 0x20000 - 16),
    dict(dq=P + 0x30000), dict(dk=P), dict(dk=P + 0x10000), dict(dk=P + 0x40000), dict(dv=P + 0x20000), dict(dv=P + 0x30000),
    dict(dv=P + 0x60000 + 16), dict(dq=P + 0x60000), dict(dk=P + 0x50000 - 16, dq=P + 0x50000)])
def test_gradients_in_other_memory_are_refused(lib, kw):
    """q, k, v, out, grad, dq, dk, dv each 0x10000 apart."""
    given = dict(**at(), g=P + 0x40000, dq=P + 0x50000, dk=P + 0x60000, dv=P + 0x70000)
    given.update(kw)
    assert lib.zx_cross_attention_backward(*grad_args(**given)) == N.ZX_ERR_INVALID
    assert b"memory" in lib.zx_last_error()
