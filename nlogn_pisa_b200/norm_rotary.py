"""Norm of each query and key head with the position rotation, in one pass.

The layer before full attention normalises every head of q and k (RMS norm
with a learned weight of head_dim elements, shared by the heads of a tensor)
and rotates it by its position (split halves, as ``mixer.RotaryEmbedding``).
``qk_norm_rotary`` does both for q and k in one launch and has a gradient in
q, k and the two weights (pisa_qk_norm_rotary / pisa_qk_norm_rotary_bwd).
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .dense import aligned_rows, differentiated, flat, view
from .validation import require_cuda


def _operands(q, k, q_weight, k_weight, frequency, positions, position_offset):
    """The arguments that both entry points take after the gradients, from the weights on."""
    batch, tokens, q_heads, dim = q.shape
    at, at_sb = (None, 0) if positions is None else (positions.data_ptr(),
                                                     0 if positions.shape[0] == 1 else positions.stride(0))
    return (q_weight.data_ptr(), k_weight.data_ptr(), _lib.DTYPES[q_weight.dtype], frequency.data_ptr(), at, at_sb,
            position_offset, _lib.DTYPES[q.dtype], batch, tokens, q_heads, k.shape[2], dim)


def _forward(q, k, q_weight, k_weight, frequency, positions, position_offset, eps):
    q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
    _lib.launch(_lib.lib().pisa_qk_norm_rotary, q.get_device(), *view(q), *view(k),
                *_operands(q, k, q_weight, k_weight, frequency, positions, position_offset), eps, q_out.data_ptr(),
                k_out.data_ptr())
    return q_out, k_out


class QkNormRotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, frequency, positions, position_offset, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, frequency, positions)
        ctx.args = (position_offset, eps)
        return _forward(q, k, q_weight, k_weight, frequency, positions, position_offset, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, frequency, positions = ctx.saved_tensors
        position_offset, eps = ctx.args
        dq_out, dk_out = flat(dq_out), flat(dk_out)
        dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
        dq_weight, dk_weight = torch.empty_like(q_weight), torch.empty_like(k_weight)
        size = _lib.workspace_bytes("pisa_qk_norm_rotary_bwd_workspace_bytes", q.get_device(), q.shape[0], q.shape[1],
                                    q.shape[3])
        workspace = q.new_empty(size, dtype=torch.uint8)
        _lib.launch(_lib.lib().pisa_qk_norm_rotary_bwd, q.get_device(), *view(q), *view(k), dq_out.data_ptr(),
                    dk_out.data_ptr(), *_operands(q, k, q_weight, k_weight, frequency, positions, position_offset), eps,
                    dq.data_ptr(), dk.data_ptr(), dq_weight.data_ptr(), dk_weight.data_ptr(), workspace.data_ptr(), size)
        return dq, dk, dq_weight, dk_weight, None, None, None, None


def qk_norm_rotary(q, k, q_weight, k_weight, frequency, positions=None, position_offset=0, eps=1e-6):
    """(q_out, k_out) of q [B,T,Hq,D], k [B,T,H,D].

    Each head row x becomes x / sqrt(mean(x^2) + eps) * weight, then rotates:
    elements i and i + D/2 turn by position * frequency[i].  ``q_weight``,
    ``k_weight``: [D], both in fp32 or both in q's dtype; ``frequency``: [D/2] (as
    ``mixer.rotary_frequencies``; a zero leaves its pair unrotated);
    ``positions``: [1|B, T] integers, or None for ``position_offset`` + token.
    The gradient is reverse mode only: forward mode raises RuntimeError.
    """
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k must have shape [batch, tokens, heads, head_dim]")
    a, b = q.shape, k.shape
    if a[:2] != b[:2] or a[3] != b[3]:
        raise ValueError("q and k must share batch, tokens and head dimension")
    if 0 in a or 0 in b:
        raise ValueError("nonempty tensors are required")
    if q.dtype != k.dtype or q.get_device() != k.get_device() or not q.is_floating_point():
        raise ValueError("q and k must share a floating dtype and device")
    dim = a[3]
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.dim() != 1 or w.shape[0] != dim or w.dtype not in (torch.float32, q.dtype) or w.get_device() != q.get_device():
            raise ValueError(f"{name} must have head_dim elements in fp32 or q's dtype on q's device")
    if q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must share a dtype")
    if frequency.dim() != 1 or 2 * frequency.shape[0] != dim:
        raise ValueError("frequency must have head_dim / 2 elements")
    if positions is not None and (positions.dim() != 2 or positions.shape[0] not in (1, a[0])
                                  or positions.shape[1] != a[1] or positions.is_floating_point()):
        raise ValueError("positions must be integers of shape [1 or B, T]")
    require_cuda(q)
    _lib.dtype_code(q)
    if frequency.dtype != torch.float32 or frequency.get_device() != q.get_device():
        frequency = frequency.to(device=q.device, dtype=torch.float32)
    frequency = frequency.contiguous()
    if positions is not None:
        if positions.dtype != torch.int64 or positions.get_device() != q.get_device():
            positions = positions.to(device=q.device, dtype=torch.int64)
        positions = positions.contiguous()
    q, k = aligned_rows(q), aligned_rows(k)
    q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    args = (q, k, q_weight, k_weight, frequency, positions, int(position_offset), float(eps))
    if differentiated(q, k, q_weight, k_weight):
        return QkNormRotaryFunction.apply(*args)
    return _forward(*args)
