"""The gated product of a feed-forward layer, with its inputs kept in 8 bits for the backward.

``swiglu`` is silu(gate) * up; with ``checkpoint_bits=8`` what its backward needs
is held as bytes with a scale per 128 elements instead of the 16-bit tensors
(pisa_swiglu / pisa_swiglu_bwd).  ``swiglu_ffn`` is the whole layer, which keeps
its input and the two products in that form only and rebuilds the gated
product in its backward.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib
from .dense import carries_tangent, differentiated
from .int8 import GROUP, byte_rows, checkpoint_int8, empty, no_gradient, restore_int8, row_bytes, rows_of
from .validation import require_cuda


def _kept_args(kept, count, width):
    """Pointers into the buffer that holds gate and up in 8 bits: bytes of both, then scales of both."""
    step, groups = row_bytes(width), (width + GROUP - 1) // GROUP
    at = kept.data_ptr()
    scales = at + 2 * count * step
    return at, at + count * step, step, scales, scales + 4 * count * groups


def _forward(gate, up, keep):
    """The product, and the buffer that keeps gate and up in 8 bits, or None."""
    width = gate.shape[-1]
    (rows, g_st), (up_rows, u_st), count = rows_of(gate), rows_of(up), gate.numel() // width
    out, kept, pointers = empty(gate), None, (None, None, 0, None, None)
    if keep:
        size = 2 * count * (row_bytes(width) + 4 * ((width + GROUP - 1) // GROUP))
        kept = gate.new_empty(size, dtype=torch.int8)
        pointers = _kept_args(kept, count, width)
    _lib.launch(_lib.lib().pisa_swiglu, gate.get_device(), rows.data_ptr(), g_st, up_rows.data_ptr(), u_st,
                _lib.DTYPES[gate.dtype], count, width, out.data_ptr(), *pointers, None, 0, None)
    return out, kept


def _backward(dout, gate, up, kept, want_out=False):
    """(dgate, dup, and the product again or None) from gate and up, or from what was kept of them."""
    width = dout.shape[-1]
    (rows, stride), count = rows_of(dout), dout.numel() // width
    dgate, dup, out = empty(dout), empty(dout), empty(dout) if want_out else None
    if kept is None:
        (gate, g_st), (up, u_st) = rows_of(gate), rows_of(up)
        given = (gate.data_ptr(), g_st, up.data_ptr(), u_st, None, None, 0, None, None)
    else:
        given = (None, 0, None, 0, *_kept_args(kept, count, width))
    _lib.launch(_lib.lib().pisa_swiglu_bwd, dout.get_device(), rows.data_ptr(), stride, *given, _lib.DTYPES[dout.dtype], count,
                width, dgate.data_ptr(), dup.data_ptr(), None if out is None else out.data_ptr())
    return dgate, dup, out


class SwigluFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, keep):
        out, kept = _forward(gate, up, keep)
        if keep:
            ctx.save_for_backward(kept)
        else:
            ctx.save_for_backward(gate, up)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        saved = ctx.saved_tensors
        dgate, dup, _ = _backward(dout, None, None, *saved) if len(saved) == 1 else _backward(dout, *saved, None)
        return dgate, dup, None


def _check_bits(checkpoint_bits):
    if checkpoint_bits not in (None, 8):
        raise ValueError("checkpoint_bits must be None or 8")
    return checkpoint_bits == 8


def swiglu(gate, up, checkpoint_bits=None, quantize=False):
    """silu(gate) * up of two tensors [..., D] of one shape.

    Gradients reach both (reverse mode only).  ``checkpoint_bits=8``: the backward
    reads gate and up in 8 bits (``checkpoint_int8``), half of what 16-bit copies
    take; the product itself is exact.  ``quantize``: (values, scale), the product
    in 8 bits as ``quantize_int8`` of its fp32 values, for ``int8_linear`` (D at
    most 32768); for inference only.  gate and up may be halves of one tensor.
    """
    keep = _check_bits(checkpoint_bits)
    if gate.dim() < 1 or gate.shape != up.shape or gate.dtype != up.dtype or not gate.is_floating_point():
        raise ValueError("gate and up must share a shape and a floating dtype")
    if 0 in gate.shape:
        raise ValueError("nonempty tensors are required")
    require_cuda(gate, up)
    if gate.get_device() != up.get_device():
        raise ValueError("gate and up must share a device")
    code = _lib.dtype_code(gate)
    if quantize:
        no_gradient("quantize=True", gate, up)
        width = gate.shape[-1]
        (rows, g_st), (up_rows, u_st) = rows_of(gate), rows_of(up)
        values, scale = byte_rows(gate, gate.shape), gate.new_empty(gate.shape[:-1], dtype=torch.float32)
        _lib.launch(_lib.lib().pisa_swiglu, gate.get_device(), rows.data_ptr(), g_st, up_rows.data_ptr(), u_st, code,
                    gate.numel() // width, width, None, None, None, 0, None, None, values.data_ptr(), row_bytes(width),
                    scale.data_ptr())
        return values, scale
    if differentiated(gate, up):
        return SwigluFunction.apply(gate, up, keep)
    return _forward(gate, up, False)[0]


class SwigluFfnFunction(torch.autograd.Function):
    """The layer's products are torch's; its backward starts from bytes."""

    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda")
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down):
        gate, up = F.linear(x, w_gate, b_gate), F.linear(x, w_up, b_up)
        if gate.shape != up.shape:
            raise ValueError("the products of w_gate and w_up must share a shape")
        out, kept = _forward(gate, up, True)
        del gate, up
        ctx.dtype = x.dtype
        ctx.save_for_backward(*checkpoint_int8(x), kept, w_gate, w_up, w_down)
        return F.linear(out, w_down, b_down)

    @staticmethod
    @torch.amp.custom_bwd(device_type="cuda")
    @once_differentiable
    def backward(ctx, dy):
        x_values, x_scale, kept, w_gate, w_up, w_down = ctx.saved_tensors
        need = ctx.needs_input_grad
        dgate, dup, out = _backward(dy @ w_down, None, None, kept, need[3])
        dx = dgate @ w_gate + dup @ w_up if need[0] else None
        dgate, dup, dy = (t.reshape(-1, t.shape[-1]) for t in (dgate, dup, dy))
        weights = [None, None, dy.T @ out.view(-1, out.shape[-1]) if need[3] else None]
        if need[1] or need[2]:
            x = restore_int8(x_values, x_scale, ctx.dtype).view(-1, x_values.shape[-1])
            weights[:2] = (t.T @ x if needed else None for t, needed in ((dgate, need[1]), (dup, need[2])))
        biases = (t.sum(0) if needed else None for t, needed in zip((dgate, dup, dy), need[4:]))
        return dx, *weights, *biases


def swiglu_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None):
    """w_down(silu(w_gate(x)) * w_up(x)), its activations kept in 8 bits until the backward.

    x [..., K]; weights as nn.Linear holds them ([O, K]), all in x's dtype.  Between
    forward and backward x and the two inner products live as bytes with a scale
    per 128 elements and the gated product is rebuilt from them, about a third of
    what 16-bit copies take.  The forward's result does not depend on it.
    Under autocast the products run in its type.  Reverse mode only.
    """
    tensors = [t for t in (x, w_gate, w_up, w_down, b_gate, b_up, b_down) if t is not None]
    if any(t.dtype != x.dtype for t in tensors) or not x.is_floating_point():
        raise ValueError("x, weights and biases must share a floating dtype")
    if x.dim() < 1 or 0 in x.shape:
        raise ValueError("nonempty tensors are required")
    # the kernels read up's rows by gate's shape
    if w_gate.dim() != 2 or w_gate.shape[1] != x.shape[-1] or w_up.shape != w_gate.shape:
        raise ValueError("w_gate and w_up must share a shape [O, K], K that of x")
    if w_down.dim() != 2 or w_down.shape[1] != w_gate.shape[0]:
        raise ValueError("w_down must have shape [N, O], O that of w_gate")
    if 0 in w_gate.shape:
        raise ValueError("nonempty weights are required")
    require_cuda(*tensors)
    _lib.dtype_code(x)
    if carries_tangent(*tensors):
        raise RuntimeError("swiglu_ffn has no forward-mode derivative")
    if not differentiated(*tensors):
        return F.linear(swiglu(F.linear(x, w_gate, b_gate), F.linear(x, w_up, b_up)), w_down, b_down)
    return SwigluFfnFunction.apply(x, w_gate, w_up, w_down, b_gate, b_up, b_down)
