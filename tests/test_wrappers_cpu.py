"""What the wrappers of rotary positions and 4-bit pages do before the library is called, without a
GPU: the library is replaced by one that records its calls and launches nothing."""
import pytest
import torch

from zenyx_amd import _native as N
from zenyx_amd import kv


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
