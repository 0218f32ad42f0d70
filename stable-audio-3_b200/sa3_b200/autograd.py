"""Differentiable forms of the operators that have a backward pass: rotary positions and cross-attention.

They take the arguments of sa3_b200.ops.rotary and ops.cross_attention without the output buffers, and give the same
values; gradients come from ops.rotary(inverse=True) and ops.cross_attention_backward. First derivatives only.

A training step captured into a CUDA graph calls the ops directly. These functions refuse to run under capture when a
gradient is wanted: autograd's accumulation nodes belong to the stream on which a leaf was first used, and a captured
backward pass that reaches the node of an eager one ends the process.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops


def _no_capture(what: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} cannot be captured with gradients: capture the forward and backward calls of "
                           "sa3_b200.ops instead")


def _rows(g: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernels read it: a row-major view with 16-byte rows (gradients of sums come expanded)."""
    if g.stride(1) == 1 and g.stride(0) >= g.shape[1] and (g.stride(0) * g.element_size()) % 16 == 0 and \
            g.data_ptr() % 16 == 0:
        return g
    return g.clone(memory_format=torch.contiguous_format)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, inv_freq, row_pos, how):
        ctx.how = how
        ctx.save_for_backward(inv_freq, row_pos)
        ctx.set_materialize_grads(False)
        return ops.rotary(q, inv_freq, k=k, row_pos=row_pos, **how)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        _no_capture("rotary")
        inv_freq, row_pos = ctx.saved_tensors
        how = dict(ctx.how, inverse=not ctx.how["inverse"])
        heads, kv_heads = how.pop("heads"), how.pop("kv_heads")
        how["row_pos"] = row_pos
        dq = None if dq is None or not ctx.needs_input_grad[0] else _rows(dq)
        dk = None if dk is None or not ctx.needs_input_grad[1] else _rows(dk)
        if dq is not None and dk is not None:
            dq, dk = ops.rotary(dq, inv_freq, heads=heads, k=dk, kv_heads=kv_heads, **how)
        elif dq is not None:
            dq = ops.rotary(dq, inv_freq, heads=heads, **how)
        elif dk is not None:
            dk = ops.rotary(dk, inv_freq, heads=kv_heads, **how)
        return dq, dk, None, None, None


def rotary(q: torch.Tensor, inv_freq: torch.Tensor, *, heads: int, head_dim: int = 64,
           k: Optional[torch.Tensor] = None, kv_heads: int = 0, row_pos: Optional[torch.Tensor] = None,
           rows_per_batch: int = 0, offset: int = 0, interleaved: bool = False, scale: float = 1.0,
           inverse: bool = False):
    """ops.rotary with gradients for q and k."""
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        _no_capture("rotary")
    how = dict(heads=heads, head_dim=head_dim, kv_heads=kv_heads, rows_per_batch=rows_per_batch, offset=offset,
               interleaved=interleaved, scale=scale, inverse=inverse)
    return _Rotary.apply(q, k, inv_freq, row_pos, how)


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens_q, cu_seqlens_k, k_lens, key_mask, how):
        where = dict(cu_seqlens_q=cu_seqlens_q, cu_seqlens_k=cu_seqlens_k, k_lens=k_lens, key_mask=key_mask)
        ctx.how = how
        # packed rows outside all sequences are not written by the kernel: zeros, not what was in memory
        out = None if cu_seqlens_q is None else torch.zeros(q.shape, device=q.device, dtype=q.dtype)
        out, lse = ops.cross_attention(q, k, v, out=out, return_lse=True, **where, **how)
        ctx.save_for_backward(q, k, v, out, lse, cu_seqlens_q, cu_seqlens_k, k_lens, key_mask)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        _no_capture("cross_attention")
        q, k, v, out, lse, cu_q, cu_k, k_lens, key_mask = ctx.saved_tensors
        # rows outside all sequences are not written by the kernels: their gradient is zero
        packed_q, packed_k = cu_q is not None, cu_k is not None
        grads = ops.cross_attention_backward(
            _rows(dout), q, k, v, out, lse, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, k_lens=k_lens, key_mask=key_mask,
            dq=torch.zeros(q.shape, device=q.device, dtype=q.dtype) if packed_q else None,
            dk=torch.zeros(k.shape, device=k.device, dtype=k.dtype) if packed_k else None,
            dv=torch.zeros(v.shape, device=v.device, dtype=v.dtype) if packed_k else None, **ctx.how)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None, None, None)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, heads: int, kv_heads: Optional[int] = None,
                    head_dim: int = 64, batch: int = 1, max_seqlen_q: int = 0, max_seqlen_k: int = 0,
                    cu_seqlens_q=None, cu_seqlens_k=None, k_lens=None, key_mask=None,
                    softmax_scale: Optional[float] = None) -> torch.Tensor:
    """ops.cross_attention with gradients for q, k and v."""
    how = dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim, batch=batch, max_seqlen_q=max_seqlen_q,
               max_seqlen_k=max_seqlen_k, softmax_scale=softmax_scale)
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return ops.cross_attention(q, k, v, cu_seqlens_q=cu_seqlens_q, cu_seqlens_k=cu_seqlens_k, k_lens=k_lens,
                                   key_mask=key_mask, **how)
    _no_capture("cross_attention")
    return _CrossAttention.apply(q, k, v, cu_seqlens_q, cu_seqlens_k, k_lens, key_mask, how)
