"""Full attention on the CUDA library: whole prompts (with gradients) and decode.

``full_attention`` is the layer beside ``sparse_attention``: every query over
all keys of its sequence, for batches and for packed sequences, through
pisa_full_attn_fwd / pisa_full_attn_bwd.  ``prefix_attention`` is its serving
form for a step's newest tokens, over each sequence's own cache and a prefix
that all sequences share, through pisa_prefix_attn.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .validation import query_positions, require_cuda, validate_qkv


def aligned_rows(t):
    """``t`` itself when its rows are contiguous, start on 16 bytes and no
    dimension is broadcast (stride 0); otherwise a contiguous copy."""
    per = 16 // t.element_size()
    if (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and all(s % per == 0 and (s > 0 or n == 1) for s, n in zip(t.stride()[:-1], t.shape))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def flat(t):
    """A contiguous tensor that starts on 16 bytes."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strides(t):
    return t.stride()[:3]


def _cumulative(cu, rows, name, device):
    """Cumulative lengths on the queries' device.  Their values are checked
    where that costs nothing (host tensors) or was asked for (status checks):
    reading a device tensor would make the host wait."""
    if not isinstance(cu, torch.Tensor) or cu.ndim != 1 or cu.dtype not in (torch.int32, torch.int64) or cu.numel() < 2:
        raise ValueError(f"{name} must be a one-dimensional integer tensor of at least two entries")
    if not cu.is_cuda or _lib.status_checks():
        bounds = cu.tolist()
        if bounds[0] != 0 or bounds[-1] != rows or any(a > b for a, b in zip(bounds, bounds[1:])):
            raise ValueError(f"{name} must rise from zero to the packed length")
    if cu.is_cuda and cu.device != device:
        raise ValueError(f"{name} must be on the query device")
    return cu.to(device).contiguous()


def _packing(cu_q, cu_k):
    if cu_q is None:
        return None, None, 0, 0
    return _lib.ptr(cu_q), _lib.ptr(cu_k), cu_q.element_size(), cu_q.numel() - 1


def _forward(q, k, v, cu_q, cu_k, offset, scale, causal, want_lse, want_low=False):
    batch, tokens, q_heads, dim = q.shape
    heads, length, dim_v = k.shape[2], k.shape[1], v.shape[-1]
    out = torch.empty((batch, tokens, q_heads, dim_v), dtype=q.dtype, device=q.device)
    lse = torch.empty((batch, tokens, q_heads), dtype=torch.float32, device=q.device) if want_lse else None
    # what rounding the output to 16 bits dropped, for the backward's row products
    low = torch.empty_like(out) if want_low and q.dtype != torch.float32 else None
    library = _lib.lib()
    # the workspace holds only the status word: passed when it will be read
    workspace = None
    if _lib.status_checks():
        workspace = torch.empty(library.pisa_full_attn_fwd_workspace_bytes(
            batch, tokens, q_heads, heads, dim, dim_v, length, 0 if cu_q is None else cu_q.numel() - 1,
            _lib.dtype_code(q)), dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        _lib.check(library.pisa_full_attn_fwd(
            _lib.ptr(q), *_strides(q), _lib.ptr(k), *_strides(k), _lib.ptr(v), *_strides(v), *_packing(cu_q, cu_k),
            offset, _lib.dtype_code(q), batch, tokens, q_heads, heads, dim, dim_v, length, scale, int(causal),
            _lib.ptr(out), _lib.ptr(low), _lib.ptr(lse), _lib.ptr(workspace), 0 if workspace is None else workspace.numel(),
            _lib.stream_of(q.device)))
    _lib.check_workspace(workspace, q.device)
    return out, lse, low


def _backward(q, k, v, out, low, dout, lse, cu_q, cu_k, offset, scale, causal):
    batch, tokens, q_heads, dim = q.shape
    heads, length, dim_v = k.shape[2], k.shape[1], v.shape[-1]
    code = _lib.dtype_code(q)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dv = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    library = _lib.lib()
    sequences = 0 if cu_q is None else cu_q.numel() - 1
    size = library.pisa_full_attn_bwd_workspace_bytes(batch, tokens, q_heads, heads, dim, dim_v, length, sequences, code)
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        _lib.check(library.pisa_full_attn_bwd(
            _lib.ptr(q), *_strides(q), _lib.ptr(k), *_strides(k), _lib.ptr(v), *_strides(v), _lib.ptr(out),
            _lib.ptr(low), _lib.ptr(dout), _lib.ptr(lse), *_packing(cu_q, cu_k), offset, code, batch, tokens, q_heads, heads, dim,
            dim_v, length, scale, int(causal), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _lib.ptr(workspace), size,
            _lib.stream_of(q.device)))
    if _lib.status_checks():
        _lib.check_workspace(workspace, q.device)
    return dq, dk, dv


class FullAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, offset, scale, causal):
        out, lse, low = _forward(q, k, v, cu_q, cu_k, offset, scale, causal, True, True)
        ctx.save_for_backward(q, k, v, out, low, lse, cu_q, cu_k)
        ctx.args = (offset, scale, causal)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        q, k, v, out, low, lse, cu_q, cu_k = ctx.saved_tensors
        dout = flat(dout)
        dq, dk, dv = _backward(q, k, v, out, low, dout, lse, cu_q, cu_k, *ctx.args)
        return dq, dk, dv, None, None, None, None, None


def full_attention(q, k, v, cu_seqlens=None, cu_seqlens_k=None, scale=None, query_offset=None, causal=True,
                   return_lse=False):
    """Attention of q [B,Tq,Hq,D] over k [B,N,H,D], v [B,N,H,Dv] -> [B,Tq,Hq,Dv] (Hq a multiple of H).

    Without ``cu_seqlens`` query i sits at position ``query_offset + i``
    (default N - Tq: the last positions) and, with ``causal``, sees the keys up
    to it.  With ``cu_seqlens`` (batch 1) the rows are packed sequences;
    ``cu_seqlens_k`` gives their keys' lengths when those differ (earlier keys
    of a continued prompt), and each sequence's queries are its last positions.
    Sequences may be empty.  Cumulative lengths on the GPU are read there: the
    call never waits for the device.  Queries without a visible key give 0.
    ``return_lse`` adds the [B,Tq,Hq] log-sum-exp (not differentiable).
    """
    validate_qkv(q, k, v)
    require_cuda(q, k, v)
    _lib.dtype_code(q)
    scale = k.shape[-1] ** -0.5 if scale is None else float(scale)
    offset = 0
    if cu_seqlens is not None:
        if q.shape[0] != 1:
            raise ValueError("packed inputs require batch size one")
        if query_offset is not None:
            raise ValueError("packed sequences take no query_offset: their queries are their last positions")
        if cu_seqlens_k is None and q.shape[1] != k.shape[1]:
            raise ValueError("packed queries and keys of different lengths need cu_seqlens_k")
        same = cu_seqlens_k is None or cu_seqlens_k is cu_seqlens
        cu_seqlens = _cumulative(cu_seqlens, q.shape[1], "cu_seqlens", q.device)
        cu_seqlens_k = cu_seqlens if same else _cumulative(cu_seqlens_k, k.shape[1], "cu_seqlens_k", q.device)
        if cu_seqlens_k.shape != cu_seqlens.shape:
            raise ValueError("cu_seqlens and cu_seqlens_k must describe the same number of sequences")
        if cu_seqlens_k.dtype != cu_seqlens.dtype:
            cu_seqlens_k = cu_seqlens_k.to(cu_seqlens.dtype)
    elif cu_seqlens_k is not None:
        raise ValueError("cu_seqlens_k needs cu_seqlens")
    elif causal:
        if query_offset is not None and not isinstance(query_offset, int):
            raise ValueError("query_offset must be an integer; sequences at different positions are packed ones")
        _, offset = query_positions(q, k, query_offset)
    q, k, v = aligned_rows(q), aligned_rows(k), aligned_rows(v)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
        out, lse = FullAttentionFunction.apply(q, k, v, cu_seqlens, cu_seqlens_k, offset, scale, bool(causal))
    else:
        out, lse, _ = _forward(q, k, v, cu_seqlens, cu_seqlens_k, offset, scale, causal, return_lse)
    return (out, lse) if return_lse else out


@torch.no_grad()
def prefix_attention(q, k, v, lengths, prefix_k=None, prefix_v=None, scale=None, return_lse=False):
    """Decode attention of the Tq newest tokens of every sequence -> [B,Tq,Hq,Dv].

    q [B,Tq,Hq,D]; k, v: the sequences' own caches [B,capacity,H,D|Dv] with
    ``lengths`` [B] valid keys each (this step's included; integers on the
    GPU, clamped to the capacity); prefix_k, prefix_v: [P,H,D|Dv], shared by
    all sequences and read once for the whole batch.  Token t sees the prefix
    and its own keys up to lengths - Tq + t; without any, it gives 0.  For
    inference: no gradient is recorded.
    """
    validate_qkv(q, k, v)
    if not isinstance(lengths, torch.Tensor) or lengths.shape != q.shape[:1] or lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError("lengths must be one integer per sequence")
    if (prefix_k is None) != (prefix_v is None):
        raise ValueError("prefix_k and prefix_v come together")
    prefix = 0
    if prefix_k is not None:
        if (prefix_k.ndim != 3 or prefix_k.shape[1:] != k.shape[2:] or prefix_v.shape != (*prefix_k.shape[:2], v.shape[-1])
                or any(t.dtype != k.dtype or t.device != k.device for t in (prefix_k, prefix_v))):
            raise ValueError("prefix_k and prefix_v must have shape [P,H,D] with the caches' heads, dims, dtype and device")
        prefix = prefix_k.shape[0]
    require_cuda(q, k, v)
    if lengths.device != q.device:
        raise ValueError("lengths must be on the query device")
    code = _lib.dtype_code(q)
    scale = k.shape[-1] ** -0.5 if scale is None else float(scale)
    q, k, v, lengths = aligned_rows(q), aligned_rows(k), aligned_rows(v), lengths.contiguous()
    if q.shape[0] > 1 and q.shape[1] > 1 and q.stride(0) != q.shape[1] * q.stride(1):
        q = q.contiguous()
    if prefix:
        prefix_k, prefix_v = (aligned_rows(t[None])[0] for t in (prefix_k, prefix_v))
    batch, tokens, q_heads, dim = q.shape
    heads, capacity, dim_v = k.shape[2], k.shape[1], v.shape[-1]
    out = torch.empty((batch, tokens, q_heads, dim_v), dtype=q.dtype, device=q.device)
    lse = torch.empty((batch, tokens, q_heads), dtype=torch.float32, device=q.device) if return_lse else None
    library = _lib.lib()
    shared = (_lib.ptr(prefix_k), *prefix_k.stride()[:2], _lib.ptr(prefix_v), *prefix_v.stride()[:2]) if prefix else (
        None, 0, 0, None, 0, 0)
    with torch.cuda.device(q.device):
        size = library.pisa_prefix_attn_workspace_bytes(batch, tokens, q_heads, heads, dim, dim_v, capacity, prefix, code)
        workspace = torch.empty(max(size, 0), dtype=torch.uint8, device=q.device)
        _lib.check(library.pisa_prefix_attn(
            _lib.ptr(q), *_strides(q), _lib.ptr(k), *_strides(k), _lib.ptr(v), *_strides(v), _lib.ptr(lengths),
            lengths.element_size(), *shared, code, batch, tokens, q_heads, heads, dim, dim_v, capacity, prefix, scale,
            _lib.ptr(out), _lib.ptr(lse), _lib.ptr(workspace), size, _lib.stream_of(q.device)))
    return (out, lse) if return_lse else out
