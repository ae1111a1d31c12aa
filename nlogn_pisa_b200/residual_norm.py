"""The norms around a branch of a decoder block, with its gate and the residual scale, in one pass.

Between two blocks a model adds a branch's output (attention's, the
feed-forward layer's) to the residual stream and normalises the sum for the
next branch; some norm the branch itself first, gate it per channel or token,
or scale either term.  ``residual_norm`` does all of it in one launch and has a
gradient (pisa_residual_norm / pisa_residual_norm_bwd).
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .dense import differentiated, flat
from .int8 import byte_rows, no_gradient, rows_of
from .validation import require_cuda


def _row_args(rows):
    return (None, 0) if rows is None else (rows.data_ptr(), rows.stride(0))


def _param_args(weight):
    return (None, 0) if weight is None else (weight.data_ptr(), _lib.DTYPES[weight.dtype])


def _forward(x, branch, gate, post_weight, weight, gate_rows, scales, eps, quantize, want_stats):
    """x, branch, gate as rows; h, n (or its bytes and scales) and the row statistics, as rows."""
    count, width = x.shape
    h = None if branch is None else x.new_empty(count, width)
    n = scale = stats = None
    if quantize:
        n, scale = byte_rows(x, (count, width)), x.new_empty(count, dtype=torch.float32)
    else:
        n = x.new_empty(count, width)
    if want_stats:
        stats = x.new_empty((count, 2), dtype=torch.float32)
    out = (None, n.data_ptr(), -(-width // 16) * 16, scale.data_ptr()) if quantize else (n.data_ptr(), None, 0, None)
    _lib.launch(_lib.lib().pisa_residual_norm, x.get_device(), *_row_args(x), *_row_args(branch), *_row_args(gate), gate_rows,
                0 if gate is None else _lib.DTYPES[gate.dtype], *_param_args(post_weight), *_param_args(weight),
                _lib.DTYPES[x.dtype], count, width, *scales, eps, None if h is None else h.data_ptr(), *out,
                None if stats is None else stats.data_ptr())
    return h, n, scale, stats


class ResidualNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, post_weight, weight, gate_rows, scales, eps):
        rows = [None if t is None else rows_of(t) for t in (x, branch, gate)]
        h, n, _, stats = _forward(*rows, post_weight, weight, gate_rows, scales, eps, False, True)
        n = n.view(x.shape)
        ctx.args = gate_rows, scales
        ctx.set_materialize_grads(False)
        if branch is None:
            ctx.save_for_backward(x, None, None, None, weight, stats)
            return n
        ctx.save_for_backward(x, branch, gate, post_weight, weight, stats)
        return h.view(x.shape), n

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, branch, gate, post_weight, weight, stats = ctx.saved_tensors
        gate_rows, scales = ctx.args
        dh, dn = grads if branch is not None else (None, *grads)
        if dh is None and dn is None:
            return (None,) * 8
        dn = torch.zeros_like(x, memory_format=torch.contiguous_format) if dn is None else flat(dn)
        dh = None if dh is None else flat(dh)
        rows, branch_rows, gate_view = (None if t is None else rows_of(t) for t in (x, branch, gate))
        count, width = rows.shape
        dx = x.new_empty(x.shape)
        dbranch = None if branch is None else x.new_empty(x.shape)
        dgate = None if gate is None else gate.new_empty(gate.shape)
        dpost, dweight = (None if w is None else w.new_empty(w.shape) for w in (post_weight, weight))
        size = _lib.workspace_bytes("pisa_residual_norm_bwd_workspace_bytes", x.get_device(), count, width,
                                    0 if gate is None else gate_rows)
        workspace = x.new_empty(size, dtype=torch.uint8)
        pointers = [None if t is None else t.data_ptr() for t in (dx, dbranch, dgate, dpost, dweight)]
        _lib.launch(_lib.lib().pisa_residual_norm_bwd, x.get_device(), None if dh is None else dh.data_ptr(), dn.data_ptr(),
                    *_row_args(rows), *_row_args(branch_rows), *_row_args(gate_view), gate_rows,
                    0 if gate is None else _lib.DTYPES[gate.dtype], *_param_args(post_weight), *_param_args(weight),
                    _lib.DTYPES[x.dtype], count, width, *scales, stats.data_ptr(), *pointers, workspace.data_ptr(), size)
        return dx, dbranch, dgate, dpost, dweight, None, None, None


def _gate_rows(gate, x):
    """How many rows share a row of the gate (0: a gate of x's own shape and dtype)."""
    if gate.shape == x.shape and gate.dtype == x.dtype:
        return 0
    if gate.numel() == x.shape[-1] and gate.shape[-1] == x.shape[-1]:
        return x.numel() // x.shape[-1]
    if gate.shape == (*x.shape[:-2], 1, x.shape[-1]):
        return x.shape[-2]
    raise ValueError("gate must have shape [D], [..., 1, D] or x's shape (then in x's dtype)")


def residual_norm(x, branch, weight, post_weight=None, gate=None, residual_scale=1.0, branch_scale=1.0, eps=1e-6,
                  quantize=False):
    """(h, n) of the residual stream x [..., T, D] and a branch's output of the same shape:

        y = branch / sqrt(mean(branch^2) + eps) * post_weight    (post_weight None: y = branch)
        h = residual_scale * x + branch_scale * gate * y         (gate None: 1)
        n = h / sqrt(mean(h^2) + eps) * weight

    ``branch`` None: h is x, and only the norm is computed.  ``weight``,
    ``post_weight``: [D] in fp32 or x's dtype.  ``gate``: [D] or [..., 1, D] (one
    per sequence) in fp32 or x's dtype, or a tensor like x.  n is computed from h
    before its rounding.  D at most 16384.  Gradients reach every tensor, in
    reverse mode only: forward mode raises RuntimeError.

    ``quantize``: (h, values, scale) with n in 8 bits, as ``quantize_int8`` of its
    fp32 values, for ``int8_linear``; for inference only.
    """
    if x.dim() < 2 or 0 in x.shape:
        raise ValueError("x must have shape [..., tokens, D] and be nonempty")
    width, device = x.shape[-1], x.get_device()
    if not x.is_floating_point():
        raise ValueError("x must be floating")
    if branch is None:
        if gate is not None or post_weight is not None or residual_scale != 1.0 or branch_scale != 1.0:
            raise ValueError("a gate, a post weight and scales belong to a branch")
    elif branch.shape != x.shape or branch.dtype != x.dtype:
        raise ValueError("branch must share x's shape and dtype")
    for name, w in (("weight", weight), ("post_weight", post_weight)):
        if w is not None and (w.shape != (width,) or w.dtype not in (torch.float32, x.dtype)):
            raise ValueError(f"{name} must have D elements in fp32 or x's dtype")
    gate_rows = 0
    if gate is not None:
        gate_rows = _gate_rows(gate, x)
        if gate.dtype not in (torch.float32, x.dtype):
            raise ValueError("gate must be in fp32 or x's dtype")
    tensors = [t for t in (x, branch, gate, post_weight, weight) if t is not None]
    require_cuda(*tensors)
    if any(t.get_device() != device for t in tensors):
        raise ValueError("all tensors must share a device")
    _lib.dtype_code(x)
    scales, eps = (float(residual_scale), float(branch_scale)), float(eps)
    if not all(math.isfinite(s) for s in scales):
        raise ValueError("scales must be finite")
    weight = weight.contiguous()
    post_weight = None if post_weight is None else post_weight.contiguous()
    if quantize:
        no_gradient("quantize=True", *tensors)
    elif differentiated(*tensors):
        if branch is None:
            return x, ResidualNormFunction.apply(x, None, None, None, weight, 0, scales, eps)
        return ResidualNormFunction.apply(x, branch, gate, post_weight, weight, gate_rows, scales, eps)
    rows = [None if t is None else rows_of(t) for t in (x, branch, gate)]
    h, n, scale, _ = _forward(*rows, post_weight, weight, gate_rows, scales, eps, quantize, False)
    h = x if h is None else h.view(x.shape)
    if quantize:
        return h, n.view(x.shape), scale.view(x.shape[:-1])
    return h, n.view(x.shape)
