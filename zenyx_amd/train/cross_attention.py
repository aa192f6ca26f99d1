"""Cross attention as a differentiable operation: a decoder's rows attend to an encoder's states,
sequences of other lengths on either side, packed or padded.  For serving, the states' keys and
values can be kept in the pages of a ``PagedFP8KVCache`` or ``PagedFP4KVCache`` instead, and every
sequence that reads them be a fork of theirs (``QuantizedRingAttention``)."""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as fwAD

from .. import kv


def _strided(t: torch.Tensor, group: int) -> torch.Tensor:
    """``t`` as the kernels take it (``group`` heads per KV head): the caller has no say in how autograd lays a
    gradient out."""
    vec = 16 // t.element_size()
    row, head, channel = t.stride()
    if channel == 1 and not (row % vec or head % vec or t.data_ptr() % 16) and row < 1 << 23 and \
            (group == 1 or head < (1 << 29) // group):
        return t
    return t.clone(memory_format=torch.contiguous_format)


class _Cross(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, k_lens, sm_scale, max_q, max_k, check, err):
        out, lse = kv.cross_attention(q, k, v, cu_q, cu_k, k_lens=k_lens, sm_scale=sm_scale, max_q_per_seq=max_q,
                                      max_k_per_seq=max_k, return_lse=True, zero_rest=True, check=check, err=err)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k, k_lens)
        ctx.sm_scale, ctx.max_q, ctx.max_k = sm_scale, max_q, max_k
        ctx.err = err  # (written again by the gradients' kernels: not among what must not change)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, cu_q, cu_k, k_lens = ctx.saved_tensors
        grad = _strided(grad, q.shape[1] // k.shape[1])
        dq, dk, dv = kv.cross_attention_backward(grad, q, k, v, out, lse, cu_q, cu_k, k_lens=k_lens, sm_scale=ctx.sm_scale,
                                                 max_q_per_seq=ctx.max_q, max_k_per_seq=ctx.max_k, err=ctx.err)
        return dq, dk, dv, *[None] * 8


class CrossAttention:
    """softmax(sm_scale q K^T) V over an encoder's states, all of which a row sees.  ``sm_scale``
    defaults to 1/sqrt(head_dim)."""

    def __init__(self, sm_scale: float | None = None):
        self.sm_scale = sm_scale

    def __call__(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor,
                 k_lens: torch.Tensor | None = None, max_q_per_seq: int | None = None,
                 max_k_per_seq: int | None = None, check: bool = False, err: torch.Tensor | None = None) -> torch.Tensor:
        """``kv.cross_attention``, differentiable (once, in reverse mode) in q, k and v.  Rows in no
        sequence, and rows and keys beyond the bounds, give zeros and take no gradient.  Without
        ``max_q_per_seq`` and ``max_k_per_seq`` the bounds are read back from ``cu_q`` and ``cu_k``,
        which waits for the device.  ``err`` (device int32 ``[1]``) collects the error bits of the call
        and of its gradients, ``check`` reads those of the call and raises."""
        if max_q_per_seq is None:
            max_q_per_seq = int((cu_q[1:] - cu_q[:-1]).max().item()) if cu_q.numel() > 1 else 0
        if max_k_per_seq is None:
            max_k_per_seq = int((cu_k[1:] - cu_k[:-1]).max().item()) if cu_k.numel() > 1 else 0
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad) or \
                any(fwAD.unpack_dual(t).tangent is not None for t in (q, k, v)):
            return _Cross.apply(q, k, v, cu_q, cu_k, k_lens, self.sm_scale, max_q_per_seq, max_k_per_seq, check, err)
        return kv.cross_attention(q, k, v, cu_q, cu_k, k_lens=k_lens, sm_scale=self.sm_scale,
                                  max_q_per_seq=max_q_per_seq, max_k_per_seq=max_k_per_seq, zero_rest=True, check=check,
                                  err=err)


__all__ = ["CrossAttention"]
