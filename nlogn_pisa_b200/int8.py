"""Tensors in 8 bits on the CUDA library, and products of them.

``quantize_int8`` rounds rows (tokens, or the output channels of a weight) to
signed bytes with one fp32 scale each, ``int8_linear`` multiplies such rows
with exact integer sums (pisa_quantize_int8, pisa_int8_linear), and
``Int8Linear`` is the layer on top.  ``checkpoint_int8`` / ``restore_int8`` keep
an activation for the backward with a scale per 128 elements.
"""

from __future__ import annotations

import torch
from torch import nn

from . import _lib
from .dense import carries_tangent, differentiated
from .validation import bare, require_cuda

GROUP = 128             # elements that share a scale of a kept activation
MAX_INNER = 1 << 17     # sums of fewer products of bytes fit 32 bits


def rows_of(t):
    """(tensor, stride): ``t``, or a copy where its strides need one, whose rows are contiguous and lie ``stride`` elements apart."""
    shape = t.shape
    width = shape[-1]
    if t.is_contiguous():
        return t, width
    if t.stride(-1) == 1 or width == 1:
        stride, count = 0, 1      # of the rows so far, from the last dimension on
        for n, step in zip(reversed(shape[:-1]), reversed(t.stride()[:-1])):
            if n == 1:
                continue
            if count == 1:
                stride = step
            elif step != stride * count:
                return t.contiguous(), width
            count *= n
        return t, stride if count > 1 else width
    return t.contiguous(), width


def empty(t):
    """A contiguous tensor like ``t`` (empty_like takes half the time of new_empty)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def row_bytes(width):
    """Bytes from one int8 row to the next, so that all start on 16."""
    return (width + 15) // 16 * 16


def byte_rows(like, shape):
    """An int8 tensor of ``shape`` whose rows start on 16 bytes."""
    width = shape[-1]
    step = row_bytes(width)
    if step == width:
        if shape == like.shape and like.is_contiguous():
            return torch.empty_like(like, dtype=torch.int8)
        return like.new_empty(shape, dtype=torch.int8)
    return like.new_empty((*shape[:-1], step), dtype=torch.int8)[..., :width]


def aligned_bytes(t):
    """rows_of for int8 rows that have to start on 16 bytes and not overlap."""
    t, stride = rows_of(t)
    if t.data_ptr() % 16 == 0 and (t.numel() == t.shape[-1] or (stride % 16 == 0 and stride >= t.shape[-1])):
        return t, stride
    return byte_rows(t, t.shape).copy_(t), row_bytes(t.shape[-1])


def no_gradient(name, *tensors):
    """Refuses a call whose result a gradient would have to pass."""
    if differentiated(*tensors):
        raise ValueError(f"{name} is for inference: it has no gradient")


def _floating(x, name):
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or not x.is_floating_point():
        raise ValueError(f"{name} must be a floating tensor with rows in its last dimension")
    if 0 in x.shape:
        raise ValueError("nonempty tensors are required")
    require_cuda(x)
    return _lib.dtype_code(x)


def _quantize(x, code, grouped):
    shape = x.shape
    width = shape[-1]
    rows, stride = rows_of(x)
    values = byte_rows(x, shape)
    scale = x.new_empty((*shape[:-1], -(-width // GROUP)) if grouped else shape[:-1], dtype=torch.float32)
    _lib.launch(_lib.lib().pisa_quantize_int8, x.get_device(), rows.data_ptr(), stride, code, x.numel() // width, width,
                int(grouped), values.data_ptr(), row_bytes(width), scale.data_ptr())
    return values, scale


def quantize_int8(x):
    """(values, scale) of x [..., K]: values int8 [..., K], scale fp32 [...], x ~ values * scale[..., None].

    Per row, each step one fp32 result: m = max(largest |x|, 2^-100), values =
    round(x * (127 / m)) to the nearest (ties to even), scale = m / 127.  Rows
    that hold an infinity or NaN become zeros under a scale of NaN.  The rows of
    ``values`` start on 16 bytes, as ``int8_linear`` takes them.  No gradient.
    """
    code = _floating(x, "x")
    no_gradient("quantize_int8", x)
    return _quantize(x, code, False)


def checkpoint_int8(x):
    """(values, scale) of an activation x [..., D] kept for a backward: as
    ``quantize_int8`` with a scale for every 128 elements of a row
    ([..., ceil(D / 128)]).  ``restore_int8`` gives it back.  No gradient is recorded."""
    code = _floating(x, "x")
    if carries_tangent(x):
        raise ValueError("checkpoint_int8 has no derivative")
    return _quantize(x, code, True)


def restore_int8(values, scale, dtype):
    """What ``checkpoint_int8`` kept, in ``dtype``: values * scale of each group."""
    if not isinstance(values, torch.Tensor) or values.dtype != torch.int8 or values.dim() < 1:
        raise ValueError("values must be int8 with rows in the last dimension")
    if 0 in values.shape:
        raise ValueError("nonempty tensors are required")
    if scale.dtype != torch.float32 or scale.shape != (*values.shape[:-1], -(-values.shape[-1] // GROUP)):
        raise ValueError("scale must be fp32 with one element per 128 of a row")
    require_cuda(values, scale)
    if scale.get_device() != values.get_device():
        raise ValueError("values and scale must share a device")
    out = values.new_empty(values.shape, dtype=dtype)
    code = _lib.dtype_code(out)
    (rows, stride), scale = aligned_bytes(values), scale.contiguous()
    _lib.launch(_lib.lib().pisa_restore_int8, values.get_device(), rows.data_ptr(), stride, scale.data_ptr(), code,
                values.numel() // values.shape[-1], values.shape[-1], out.data_ptr())
    return out


def int8_linear(x, weight, weight_scale, bias=None, x_scale=None, out_dtype=None):
    """x [..., K] times weight [O, K] transposed -> [..., O], both in 8 bits.

    out[t, o] = x_scale[t] * weight_scale[o] * sum_k x[t, k] * weight[o, k] +
    bias[o], the sums exact (K below 131072).  ``x``: int8 with ``x_scale`` [...]
    (as ``quantize_int8``, ``residual_norm`` and ``swiglu`` give them), or
    floating, which the call rounds as ``quantize_int8``.  ``weight``,
    ``weight_scale`` [O]: ``quantize_int8`` of a weight.  ``bias``: [O] in fp32 or
    ``out_dtype``, which defaults to x's floating dtype, or bf16 for int8.  int8
    rows that do not start on 16 bytes are copied.  For inference: no gradient.
    """
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.dtype != torch.int8:
        raise ValueError("weight must be int8 [O, K]")
    outer, inner = weight.shape
    if x.dim() < 1 or x.shape[-1] != inner:
        raise ValueError("x and weight must share their last dimension")
    if x.numel() == 0 or outer == 0:
        raise ValueError("nonempty tensors are required")
    if inner >= MAX_INNER:
        raise ValueError("sums of 131072 or more products may not fit 32 bits")
    shape, device, whole = x.shape[:-1], x.get_device(), x.dtype == torch.int8
    if weight_scale.dtype != torch.float32 or weight_scale.dim() != 1 or weight_scale.shape[0] != outer:
        raise ValueError("weight_scale must be fp32 with one element per output channel")
    if (x_scale is not None) != whole:
        raise ValueError("int8 x comes with x_scale, floating x without")
    if whole and (x_scale.dtype != torch.float32 or x_scale.shape != shape):
        raise ValueError("x_scale must be fp32 with one element per row of x")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if whole else x.dtype
    if out_dtype not in _lib.DTYPES:
        raise ValueError("the CUDA kernels support FP16, BF16 and FP32")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != outer or bias.dtype not in (torch.float32, out_dtype)):
        raise ValueError("bias must have one element per output channel in fp32 or the output's dtype")
    for t in (x, weight, weight_scale, x_scale, bias):
        if t is not None and t.get_device() != device:
            require_cuda(t, x)
            raise ValueError("x, weight, scales and bias must share a device")
    require_cuda(x)
    no_gradient("int8_linear", x, weight_scale, *([x_scale] if whole else []), *([] if bias is None else [bias]))
    count = x.numel() // inner
    weight, w_stride = aligned_bytes(weight)
    weight_scale = weight_scale.contiguous()
    bias_args = (None, 0)
    if bias is not None:
        bias = bias.contiguous()
        bias_args = bias.data_ptr(), _lib.DTYPES[bias.dtype]
    workspace, size = None, 0
    if whole:
        (rows, x_stride), x_scale, code = aligned_bytes(x), x_scale.contiguous(), _lib.S8
    else:
        (rows, x_stride), code = rows_of(x), _floating(x, "x")
    if not whole or _lib.status_checks():
        size = _lib.workspace_bytes("pisa_int8_linear_workspace_bytes", device, count, inner, outer, code)
        if size > 256 or _lib.status_checks():   # more than the status word: rows rounded on their way
            workspace = weight.new_empty(size)
    out = weight_scale.new_empty((*shape, outer), dtype=out_dtype)
    _lib.launch(_lib.lib().pisa_int8_linear, device, rows.data_ptr(), x_stride, code, x_scale.data_ptr() if whole else None,
                weight.data_ptr(), w_stride, weight_scale.data_ptr(), *bias_args, _lib.DTYPES[out_dtype], count, inner, outer,
                out.data_ptr(), None if workspace is None else workspace.data_ptr(), size)
    if _lib.status_checks():
        _lib.check_workspace(workspace, x.device)
    return out


class Int8Linear(nn.Module):
    """A linear layer with its weight in 8 bits, for inference.

    ``from_linear`` rounds the weight of an nn.Linear on the GPU.  The forward
    takes what ``int8_linear`` takes: floating tokens, or int8 ones and their
    scales.  Like it, it refuses tokens that require a gradient.
    """

    def __init__(self, in_features, out_features, bias=True):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        # rows of whole 16 bytes, as the products read them
        self.register_buffer("weight", torch.zeros(out_features, -(-in_features // 16) * 16, dtype=torch.int8))
        self.register_buffer("weight_scale", torch.zeros(out_features, dtype=torch.float32))
        self.register_buffer("bias", torch.zeros(out_features, dtype=torch.float32) if bias else None)

    def _apply(self, fn, recurse=True):
        """Scales and bias stay fp32 when the layer is cast to another type."""
        kept = {name: t for name, t in self._buffers.items() if t is not None and t.dtype == torch.float32}
        super()._apply(fn, recurse)
        for name, t in kept.items():
            device = self._buffers[name].device
            if self._buffers[name].dtype != torch.float32:
                self._buffers[name] = torch.empty_like(t, device=device) if t.is_meta else t.to(device)
        return self

    @classmethod
    @torch.no_grad()
    def from_linear(cls, *linears):
        """The layer of one nn.Linear, or of several with the same input, their outputs side by side.

        It takes over weights and biases alone: layers with hooks or a forward of their own (adapters) are refused."""
        if not all(bare(m, nn.Linear) for m in linears):
            raise ValueError("only linear layers without hooks or a forward of their own have an 8-bit form")
        first = linears[0]
        bias = first.bias is not None
        if any(m.in_features != first.in_features or (m.bias is not None) != bias for m in linears):
            raise ValueError("joined layers must share their input and all or none have a bias")
        layer = cls(first.in_features, sum(m.out_features for m in linears), bias).to(first.weight.device)
        values, scale = quantize_int8(torch.cat([m.weight for m in linears]).detach())
        layer.weight[:, :first.in_features] = values
        layer.weight_scale.copy_(scale)
        if bias:
            layer.bias = torch.cat([m.bias for m in linears]).detach().float()
        return layer

    def forward(self, x, x_scale=None, out_dtype=None):
        bias = self.bias
        if bias is not None and bias.dtype != torch.float32:
            bias = bias.float()
        return int8_linear(x, self.weight[:, :self.in_features], self.weight_scale, bias=bias, x_scale=x_scale,
                           out_dtype=out_dtype)
