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
from .int8 import byte_rows, empty, no_gradient, row_bytes, rows_of
from .validation import require_cuda


def _operands(x, branch, gate, gate_rows, post_weight, weight, scales):
    """The arguments that both entry points take for the forward's operands, and tensors to keep until the launch."""
    width = x.shape[-1]
    x, x_st = rows_of(x)
    args, kept = [x.data_ptr(), x_st, None, 0, None, 0, gate_rows, 0, None, 0], [x]
    if branch is not None:
        branch, stride = rows_of(branch)
        args[2:4] = branch.data_ptr(), stride
        kept.append(branch)
        if gate is not None:
            gate, stride = rows_of(gate)
            args[4:8] = gate.data_ptr(), stride, gate_rows, _lib.DTYPES[gate.dtype]
            kept.append(gate)
        if post_weight is not None:
            args[8:] = post_weight.data_ptr(), _lib.DTYPES[post_weight.dtype]
    return (*args, weight.data_ptr(), _lib.DTYPES[weight.dtype], _lib.DTYPES[x.dtype], x.numel() // width, width, *scales), kept


def _forward(x, branch, gate, post_weight, weight, gate_rows, scales, eps, quantize, want_stats):
    """h, n (or its bytes and scales) and the row statistics."""
    operands, _kept = _operands(x, branch, gate, gate_rows, post_weight, weight, scales)
    h = None if branch is None else empty(x)
    scale = stats = None
    if quantize:
        n, scale = byte_rows(x, x.shape), x.new_empty(x.shape[:-1], dtype=torch.float32)
        out = None, n.data_ptr(), row_bytes(x.shape[-1]), scale.data_ptr()
    else:
        n = empty(x)
        out = n.data_ptr(), None, 0, None
    if want_stats:
        stats = x.new_empty((*x.shape[:-1], 2), dtype=torch.float32)
    _lib.launch(_lib.lib().pisa_residual_norm, x.get_device(), *operands, eps, None if h is None else h.data_ptr(), *out,
                None if stats is None else stats.data_ptr())
    return h, n, scale, stats


class ResidualNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, post_weight, weight, gate_rows, scales, eps):
        h, n, _, stats = _forward(x, branch, gate, post_weight, weight, gate_rows, scales, eps, False, True)
        ctx.args = gate_rows, scales
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, branch, gate, post_weight, weight, stats)
        return n if branch is None else (h, n)

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
        operands, _kept = _operands(x, branch, gate, gate_rows, post_weight, weight, scales)
        dx, dweight = empty(x), torch.empty_like(weight)
        dbranch = dgate = dpost = None
        if branch is not None:
            dbranch = empty(x)
            dgate = None if gate is None else empty(gate)
            dpost = None if post_weight is None else torch.empty_like(post_weight)
        width = x.shape[-1]
        size = _lib.workspace_bytes("pisa_residual_norm_bwd_workspace_bytes", x.get_device(), x.numel() // width, width,
                                    0 if gate is None else gate_rows)
        workspace = x.new_empty(size, dtype=torch.uint8)
        _lib.launch(_lib.lib().pisa_residual_norm_bwd, x.get_device(), None if dh is None else dh.data_ptr(), dn.data_ptr(),
                    *operands, stats.data_ptr(), dx.data_ptr(), *(None if t is None else t.data_ptr() for t in (dbranch, dgate, dpost)),
                    dweight.data_ptr(), workspace.data_ptr(), size)
        return dx, dbranch, dgate, dpost, dweight, None, None, None


def _gate_rows(gate, x):
    """How many rows share a row of the gate (0: a gate of x's own shape and dtype)."""
    shape, of = x.shape, gate.shape
    if of == shape and gate.dtype == x.dtype:
        return 0
    if of and of[-1] == shape[-1]:
        if gate.numel() == shape[-1]:
            return x.numel() // shape[-1]
        if of[-2] == 1 and of[:-2] == shape[:-2]:
            return shape[-2]
    raise ValueError("gate must have shape [D], [..., 1, D] or x's shape (then in x's dtype)")


def residual_norm(x, branch, weight, post_weight=None, gate=None, residual_scale=1.0, branch_scale=1.0, eps=1e-6,
                  quantize=False):
    """(h, n) of the residual stream x [..., T, D] and a branch's output of the same shape:

        y = branch / sqrt(mean(branch^2) + eps) * post_weight    (post_weight None: y = branch)
        h = residual_scale * x + branch_scale * gate * y         (gate None: 1)
        n = h / sqrt(mean(h^2) + eps) * weight

    The scales are numbers.  ``branch`` None: h is x, and only the norm is computed.  ``weight``,
    ``post_weight``: [D] in fp32 or x's dtype.  ``gate``: [D] or [..., 1, D] (one
    per sequence) in fp32 or x's dtype, or a tensor like x.  n is computed from h
    before its rounding.  D at most 16384.  Gradients reach every tensor, in
    reverse mode only: forward mode raises RuntimeError.

    ``quantize``: (h, values, scale) with n in 8 bits, as ``quantize_int8`` of its
    fp32 values, for ``int8_linear``; for inference only.
    """
    shape, dtype, device = x.shape, x.dtype, x.get_device()
    if len(shape) < 2 or 0 in shape:
        raise ValueError("x must have shape [..., tokens, D] and be nonempty")
    if not dtype.is_floating_point:
        raise ValueError("x must be floating")
    tensors = [x, weight]
    if branch is None:
        if gate is not None or post_weight is not None or residual_scale != 1.0 or branch_scale != 1.0:
            raise ValueError("a gate, a post weight and scales belong to a branch")
    else:
        if branch.shape != shape or branch.dtype != dtype:
            raise ValueError("branch must share x's shape and dtype")
        tensors.append(branch)
    if weight.dim() != 1 or weight.shape[0] != shape[-1] or weight.dtype not in (torch.float32, dtype):
        raise ValueError("weight must have D elements in fp32 or x's dtype")
    weight = weight.contiguous()
    if post_weight is not None:
        if post_weight.dim() != 1 or post_weight.shape[0] != shape[-1] or post_weight.dtype not in (torch.float32, dtype):
            raise ValueError("post_weight must have D elements in fp32 or x's dtype")
        post_weight = post_weight.contiguous()
        tensors.append(post_weight)
    gate_rows = 0
    if gate is not None:
        gate_rows = _gate_rows(gate, x)
        if gate.dtype not in (torch.float32, dtype):
            raise ValueError("gate must be in fp32 or x's dtype")
        tensors.append(gate)
    for t in tensors:
        if t.get_device() != device:
            require_cuda(*tensors)
            raise ValueError("all tensors must share a device")
    require_cuda(x)
    _lib.dtype_code(x)
    if isinstance(residual_scale, torch.Tensor) or isinstance(branch_scale, torch.Tensor):
        raise ValueError("scales are numbers: a learned one is a gate")
    scales, eps = (float(residual_scale), float(branch_scale)), float(eps)
    if not (math.isfinite(scales[0]) and math.isfinite(scales[1])):
        raise ValueError("scales must be finite")
    if quantize:
        no_gradient("quantize=True", *tensors)
    elif differentiated(*tensors):
        if branch is None:
            return x, ResidualNormFunction.apply(x, None, None, None, weight, 0, scales, eps)
        return ResidualNormFunction.apply(x, branch, gate, post_weight, weight, gate_rows, scales, eps)
    h, n, scale, _ = _forward(x, branch, gate, post_weight, weight, gate_rows, scales, eps, quantize, False)
    h = x if branch is None else h
    return (h, n, scale) if quantize else (h, n)
