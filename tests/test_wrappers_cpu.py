"""What the wrappers of rotary positions and 4-bit pages do before the library is called, without a
GPU: the library is replaced by one that records its calls and launches nothing."""
import warnings

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from zenyx_amd import _native as N
from zenyx_amd import kv
from zenyx_amd.train.fp8_kv_quantization import PagedFP4KVCache, QuantizedRingAttention
from zenyx_amd.train.rotary import RotaryPositions


class Recorder:
    """Stands for the library: every entry point answers 0 and is written down."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def lib(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(N, "need_gpu", lambda: None)
    monkeypatch.setattr(N, "load", lambda: rec)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    kv._workspace_bytes.cache_clear()
    yield rec
    kv._workspace_bytes.cache_clear()


def aligned(*shape, dtype=torch.uint8):
    """A zeroed host tensor whose memory begins at a multiple of 16 bytes."""
    t = torch.zeros(shape, dtype=dtype)
    n = 16 // t.element_size()
    room = torch.zeros(t.numel() + n, dtype=dtype)
    skip = (-room.data_ptr() % 16) // t.element_size()
    return room[skip:skip + t.numel()].view(shape)


def host_calls():
    H, D, P, B = 2, 64, 16, 1
    x, q = aligned(1, 4, 2, H, D, dtype=torch.bfloat16), aligned(B, 4, D, dtype=torch.bfloat16)
    cu, bt, lens = (aligned(*s, dtype=torch.int32) for s in ((B + 1,), (B, 2), (B,)))
    table, pool8 = aligned(8, D, dtype=torch.float32), aligned(1, 3, 2, H, P, D)
    scales, pool4 = aligned(1, 2, H, dtype=torch.float32), aligned(1, 3, 2, H, 1, 17 * D // 2)
    return {
        "rope": lambda: kv.rope(x[0, :, 0], table, aligned(4, dtype=torch.int32)),
        "kv_rope_append": lambda: kv.kv_rope_append(x, table, cu, bt, pool8),
        "kv_rope_append, static": lambda: kv.kv_rope_append(x, table, cu, bt, pool8, scales=scales, static_scales=True),
        "kv4_append": lambda: kv.kv4_append(x, cu, bt, pool4),
        "kv4_append, rotated": lambda: kv.kv4_append(x, cu, bt, pool4, table=table, start_pos=lens),
        "kv4_gather_dequant": lambda: kv.kv4_gather_dequant(pool4[0], bt, lens),
        "kv4_gather_dequant, out": lambda: kv.kv4_gather_dequant(
            pool4[0], bt, lens, 32, out=tuple(aligned(B, H, 32, D, dtype=torch.bfloat16) for _ in range(2))),
        "paged_attention4_decode": lambda: kv.paged_attention4_decode(q, pool4[0], bt, lens),
        "paged_attention4_prefill": lambda: kv.paged_attention4_prefill(q, cu, lens, pool4[0], bt, lens),
        "paged_attention4_prefill, bounded": lambda: kv.paged_attention4_prefill(q, cu, lens, pool4[0], bt, lens,
                                                                                 max_q_per_seq=1)}


@pytest.mark.parametrize("name", list(host_calls()))
def test_calls_with_host_tensors_alone_are_refused(lib, name):
    """A kernel must not be handed addresses of host memory: with every tensor on the CPU the
    devices agree with each other, and the call is refused all the same."""
    with pytest.raises(ValueError, match="HIP device tensor"):
        host_calls()[name]()
    assert not [c for c, _ in lib.calls if not c.endswith("workspace_bytes")]


# ------------------------------------------------------------------ RotaryPositions as an operation

def plain_rope(x, table, positions, interleaved=False, transpose=False, out=None, check=False):
    """kv.rope by torch operations that autograd does not see (as it does not see the kernel), with
    its demand on alignment."""
    if x.data_ptr() % 16:
        raise ValueError("every head's row must be 16-byte aligned")
    y = torch.tensor(x.tolist(), dtype=x.dtype).view(x.shape)
    n = table.shape[1] // 2
    c, s = (t[:, None] for t in table[positions.long()].split(n, 1))
    s = -s if transpose else s
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


@pytest.fixture(params=[False, True])
def rotary(monkeypatch, request):
    monkeypatch.setattr(kv, "rope", plain_rope)
    f = torch.arange(8, dtype=torch.float64)
    angle = torch.arange(20, dtype=torch.float64)[:, None] * 100.0 ** (-f / 8)
    monkeypatch.setattr(kv, "rope_table", lambda *a: torch.cat([angle.cos(), angle.sin()], 1).float())
    return RotaryPositions(24, 20, rotary_dim=16, interleaved=request.param, device=torch.device("cpu"))


def test_gradients_at_any_alignment(rotary):
    """The gradient of a slice of a concatenation begins wherever the slice does."""
    p = torch.tensor([3, 0, 19], dtype=torch.int32)
    x = torch.randn((3, 2, 24), requires_grad=True)
    g = torch.randn(144 + 5)
    for lead in (0, 1, 2, 3, 5):
        y = torch.cat([torch.zeros(lead), rotary(x, p).flatten()])
        got, = torch.autograd.grad((y * g[:144 + lead]).sum(), x)
        want = plain_rope(g[lead:144 + lead].clone().view(3, 2, 24), rotary.table, p, rotary.interleaved, True)
        assert torch.equal(got, want), lead
    # an expanded gradient, and one that is not contiguous
    got, = torch.autograd.grad(rotary(x, p).sum(), x)
    assert torch.equal(got, plain_rope(torch.ones(3, 2, 24), rotary.table, p, rotary.interleaved, True))
    got, = torch.autograd.grad((rotary(x, p).transpose(0, 2).contiguous() * g[:144].view(24, 2, 3)).sum(), x)
    want = plain_rope(g[:144].view(24, 2, 3).transpose(0, 2).contiguous(), rotary.table, p, rotary.interleaved, True)
    assert torch.equal(got, want)


def test_forward_mode_derivatives(rotary):
    """The rotation is linear: a tangent turns as the values do, with or without a gradient asked for,
    at any alignment, and the two modes mix in either order."""
    p = torch.tensor([3, 0, 19], dtype=torch.int32)
    x, v = torch.randn((3, 2, 24)), torch.randn(145)[1:].view(3, 2, 24)
    turned = plain_rope(v.clone(), rotary.table, p, rotary.interleaved)
    for primal in (x, x.clone().requires_grad_()):
        with fwAD.dual_level():
            out = fwAD.unpack_dual(rotary(fwAD.make_dual(primal, v), p))
            assert torch.equal(out.primal, rotary(x, p)) and out.tangent is not None
            assert torch.equal(out.tangent, turned)
            with torch.no_grad():  # (ends reverse mode alone)
                assert torch.equal(fwAD.unpack_dual(rotary(fwAD.make_dual(primal, v), p)).tangent, turned)
            assert fwAD.unpack_dual(rotary(primal, p)).tangent is None
    # the tangent of a gradient: d/de of R^T sin(R (x + e v)) is R^T (cos(R x) * R v)
    leaf = x.clone().requires_grad_()
    rx, rv = (plain_rope(t.clone(), rotary.table, p, rotary.interleaved) for t in (x, v))
    want = plain_rope(rx.cos() * rv, rotary.table, p, rotary.interleaved, True)
    with fwAD.dual_level():
        y = rotary(fwAD.make_dual(leaf, v), p)
        grad, = torch.autograd.grad(-y.cos().sum(), leaf)
        torch.testing.assert_close(fwAD.unpack_dual(grad).tangent, want)
    # the gradient of a tangent, in x: <u, cos(R x) * R v> gives R^T (-sin(R x) * R v * u)
    u = torch.randn((3, 2, 24))
    with fwAD.dual_level():
        t = fwAD.unpack_dual(rotary(fwAD.make_dual(leaf, v), p).sin()).tangent
        grad, = torch.autograd.grad((t * u).sum(), leaf)
    torch.testing.assert_close(grad, plain_rope(-rx.sin() * rv * u, rotary.table, p, rotary.interleaved, True))
    # ... and in the tangent itself
    w = v.clone().requires_grad_()
    with fwAD.dual_level():
        t = fwAD.unpack_dual(rotary(fwAD.make_dual(x, w), p)).tangent
        grad, = torch.autograd.grad((t * u).sum(), w)
    assert torch.equal(grad, plain_rope(u, rotary.table, p, rotary.interleaved, True))


def test_a_trace_holds_the_rotation(rotary):
    """torch.jit.trace records the operation, not the allocation of its output alone."""
    p = torch.tensor([3, 0, 19], dtype=torch.int32)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")  # (the check of the heads' width is a Python branch)
        traced = torch.jit.trace(lambda t: rotary(t, p), (torch.randn((3, 2, 24)),))
    x = torch.randn((3, 2, 24))
    assert torch.equal(traced(x), rotary(x, p))


# ------------------------------------------------------------------ precision over 4-bit pages

@pytest.mark.parametrize("asked, given", [(None, "exact"), ("f16", "exact"), ("exact", "exact"), ("bf16", "bf16")])
def test_attention_over_4_bit_pages_keeps_the_bits_asked_for(monkeypatch, asked, given):
    """The 4-bit kernels have no fp16 weights: who asks for them (the default) gets more bits, not fewer."""
    seen = []

    def prefill(q, *args, precision="nothing passed", **kw):
        seen.append(precision)
        return q
    monkeypatch.setattr(kv, "paged_attention4_prefill", prefill)
    cache = PagedFP4KVCache(1, 2, 64, 4, device=torch.device("cpu"))
    cache.lengths, cache.pages = {0: 5}, {0: [1]}
    att = QuantizedRingAttention(cache, **({} if asked is None else {"precision": asked}), check=False)
    att(torch.zeros((5, 4, 64), dtype=torch.bfloat16), 0, [0], [5])
    assert seen == [given]


def test_4_bit_prefill_does_not_drop_bits_by_itself(lib, monkeypatch):
    """Weights rounded to bf16 are the caller's choice."""
    monkeypatch.setattr(kv, "_index", lambda t, name: -1)
    q, cu, lens = aligned(1, 4, 64, dtype=torch.bfloat16), aligned(2, dtype=torch.int32), aligned(1, dtype=torch.int32)
    bt, pool = aligned(1, 2, dtype=torch.int32), aligned(3, 2, 2, 1, 544)
    for kw, flag in (({}, N.ZX_PREFILL_EXACT_P), ({"precision": "exact"}, N.ZX_PREFILL_EXACT_P), ({"precision": "bf16"}, 0)):
        kv.paged_attention4_prefill(q, cu, lens, pool, bt, lens, max_q_per_seq=1, **kw)
        name, args = lib.calls[-1]
        assert name == "zx_paged_attention4_prefill" and args[17] == flag
