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
from .dense import aligned_rows, flat
from .validation import require_cuda


def _operands(q, k, q_weight, k_weight, frequency, positions, position_offset):
    """The leading arguments of both entry points after the tensors."""
    return (_lib.ptr(q_weight), _lib.ptr(k_weight), _lib.dtype_code(q_weight), _lib.ptr(frequency), _lib.ptr(positions),
            0 if positions is None or positions.shape[0] == 1 else positions.stride(0), position_offset,
            _lib.dtype_code(q), *q.shape[:3], k.shape[2], q.shape[3])


def _forward(q, k, q_weight, k_weight, frequency, positions, position_offset, eps):
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    with torch.cuda.device(q.device):
        _lib.check(_lib.lib().pisa_qk_norm_rotary(
            _lib.ptr(q), *q.stride()[:3], _lib.ptr(k), *k.stride()[:3],
            *_operands(q, k, q_weight, k_weight, frequency, positions, position_offset), eps, _lib.ptr(q_out),
            _lib.ptr(k_out), _lib.stream_of(q.device)))
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
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dq_weight, dk_weight = torch.empty_like(q_weight), torch.empty_like(k_weight)
        library = _lib.lib()
        with torch.cuda.device(q.device):
            size = library.pisa_qk_norm_rotary_bwd_workspace_bytes(q.shape[0], q.shape[1], q.shape[3])
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
            _lib.check(library.pisa_qk_norm_rotary_bwd(
                _lib.ptr(q), *q.stride()[:3], _lib.ptr(k), *k.stride()[:3], _lib.ptr(dq_out), _lib.ptr(dk_out),
                *_operands(q, k, q_weight, k_weight, frequency, positions, position_offset), eps, _lib.ptr(dq),
                _lib.ptr(dk), _lib.ptr(dq_weight), _lib.ptr(dk_weight), _lib.ptr(workspace), size,
                _lib.stream_of(q.device)))
        return dq, dk, dq_weight, dk_weight, None, None, None, None


def qk_norm_rotary(q, k, q_weight, k_weight, frequency, positions=None, position_offset=0, eps=1e-6):
    """(q_out, k_out) of q [B,T,Hq,D], k [B,T,H,D].

    Each head row x becomes x / sqrt(mean(x^2) + eps) * weight, then rotates:
    elements i and i + D/2 turn by position * frequency[i].  ``q_weight``,
    ``k_weight``: [D], both in fp32 or both in q's dtype; ``frequency``: [D/2] (as
    ``mixer.rotary_frequencies``; a zero leaves its pair unrotated);
    ``positions``: [1|B, T] integers, or None for ``position_offset`` + token.
    """
    if q.ndim != 4 or k.ndim != 4:
        raise ValueError("q and k must have shape [batch, tokens, heads, head_dim]")
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("q and k must share batch, tokens and head dimension")
    if min(*q.shape, *k.shape) <= 0:
        raise ValueError("nonempty tensors are required")
    if q.device != k.device or q.dtype != k.dtype or not q.is_floating_point():
        raise ValueError("q and k must share a floating dtype and device")
    dim = q.shape[3]
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.shape != (dim,) or w.dtype not in (torch.float32, q.dtype) or w.device != q.device:
            raise ValueError(f"{name} must have head_dim elements in fp32 or q's dtype on q's device")
    if q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must share a dtype")
    if frequency.shape != (dim // 2,) or dim % 2:
        raise ValueError("frequency must have head_dim / 2 elements")
    if positions is not None and (positions.ndim != 2 or positions.shape[0] not in (1, q.shape[0])
                                  or positions.shape[1] != q.shape[1] or positions.is_floating_point()):
        raise ValueError("positions must be integers of shape [1 or B, T]")
    require_cuda(q, k, q_weight, k_weight)
    _lib.dtype_code(q)
    frequency = frequency.to(device=q.device, dtype=torch.float32).contiguous()
    if positions is not None:
        positions = positions.to(device=q.device, dtype=torch.int64).contiguous()
    q, k = aligned_rows(q), aligned_rows(k)
    q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    args = (q, k, q_weight, k_weight, frequency, positions, int(position_offset), float(eps))
    if torch.is_grad_enabled() and any(t.requires_grad for t in args[:4]):
        return QkNormRotaryFunction.apply(*args)
    return _forward(*args)
