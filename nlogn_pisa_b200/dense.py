"""Full attention on the CUDA library: whole prompts (with gradients) and decode.

``full_attention`` is the layer beside ``sparse_attention``: every query over
all keys of its sequence, for batches and for packed sequences, through
pisa_full_attn_fwd / pisa_full_attn_bwd.  ``prefix_attention`` is its serving
form for a step's newest tokens, over each sequence's own cache and a prefix
that all sequences share, through pisa_prefix_attn; ``continued_attention`` is
the form for many new tokens per sequence over such a prefix.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .validation import query_positions, require_cuda, validate_qkv


def aligned_rows(t):
    """``t`` itself when its rows are contiguous, start on 16 bytes and no
    dimension is broadcast (stride 0); otherwise a contiguous copy."""
    per = 16 // t.element_size()
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            if t.shape[-1] % per == 0:
                return t
        elif t.stride(-1) == 1 and all(n == 1 or (s > 0 and s % per == 0) for s, n in zip(t.stride()[:-1], t.shape)):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def differentiated(*tensors):
    """Whether autograd has to see a call on these tensors: one requires grad, or
    carries a tangent (forward mode, for which the operators' autograd functions raise)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                return True
    return carries_tangent(*tensors)


def carries_tangent(*tensors):
    # outside every dual level there are none: one attribute instead of a call per tensor
    if getattr(forward_ad, "_current_level", 0) < 0:
        return False
    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            return True
    return False


def flat(t):
    """A contiguous tensor that starts on 16 bytes."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _validate(q, k, v):
    """The operators' common contract; the usual call passes on a few comparisons."""
    if q.dim() == k.dim() == v.dim() == 4 and q.is_cuda and k.is_cuda and v.is_cuda and q.dtype in _lib.DTYPES:
        a, b, c = q.shape, k.shape, v.shape
        if (a[0] == b[0] and a[3] == b[3] and c[:3] == b[:3] and 0 not in a and 0 not in b and a[2] % b[2] == 0
                and q.dtype == k.dtype == v.dtype and q.get_device() == k.get_device() == v.get_device()):
            return
    validate_qkv(q, k, v)
    require_cuda(q, k, v)
    _lib.dtype_code(q)


def view(t):
    """Pointer and the three leading strides, as the entry points take them."""
    s = t.stride()
    return t.data_ptr(), s[0], s[1], s[2]


def _cumulative(cu, rows, name, q):
    """Cumulative lengths on the queries' device.  Their values are checked
    where that costs nothing (host tensors) or was asked for (status checks):
    reading a device tensor would make the host wait."""
    if not isinstance(cu, torch.Tensor) or cu.dim() != 1 or cu.dtype not in (torch.int32, torch.int64) or cu.shape[0] < 2:
        raise ValueError(f"{name} must be a one-dimensional integer tensor of at least two entries")
    if not cu.is_cuda or _lib.status_checks():
        bounds = cu.tolist()
        if bounds[0] != 0 or bounds[-1] != rows or any(a > b for a, b in zip(bounds, bounds[1:])):
            raise ValueError(f"{name} must rise from zero to the packed length")
    if not cu.is_cuda:
        cu = cu.to(q.device)
    elif cu.get_device() != q.get_device():
        raise ValueError(f"{name} must be on the query device")
    return cu.contiguous()


def _packing(cu_q, cu_k):
    if cu_q is None:
        return None, None, 0, 0
    return cu_q.data_ptr(), cu_k.data_ptr(), cu_q.element_size(), cu_q.shape[0] - 1


def _forward(q, k, v, cu_q, cu_k, offset, scale, causal, want_lse, want_low=False):
    batch, tokens, q_heads, dim = q.shape
    _, length, heads, dim_v = v.shape
    out = q.new_empty((batch, tokens, q_heads, dim_v))
    lse = q.new_empty((batch, tokens, q_heads), dtype=torch.float32) if want_lse else None
    # what rounding the output to 16 bits dropped, for the backward's row products
    low = torch.empty_like(out) if want_low and q.dtype != torch.float32 else None
    library, code, packing = _lib.lib(), _lib.DTYPES[q.dtype], _packing(cu_q, cu_k)
    # the workspace holds the status word, and over many keys the outputs on their way: passed when either is wanted
    workspace, size = None, 0
    if _lib.status_checks() or length > (65536 if low is None else 8192):
        size = _lib.workspace_bytes("pisa_full_attn_fwd_workspace_bytes", q.get_device(), batch, tokens, q_heads, heads, dim,
                                    dim_v, length, packing[3], code)
        workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    _lib.launch(library.pisa_full_attn_fwd, q.get_device(), *view(q), *view(k), *view(v), *packing, offset, code, batch,
                tokens, q_heads, heads, dim, dim_v, length, scale, int(causal), out.data_ptr(),
                None if low is None else low.data_ptr(), None if lse is None else lse.data_ptr(),
                None if workspace is None else workspace.data_ptr(), size)
    if _lib.status_checks():
        _lib.check_workspace(workspace, q.device)
    return out, lse, low


def _backward(q, k, v, out, low, dout, lse, cu_q, cu_k, offset, scale, causal):
    batch, tokens, q_heads, dim = q.shape
    _, length, heads, dim_v = v.shape
    library, code, packing = _lib.lib(), _lib.DTYPES[q.dtype], _packing(cu_q, cu_k)
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    size = _lib.workspace_bytes("pisa_full_attn_bwd_workspace_bytes", q.get_device(), batch, tokens, q_heads, heads, dim,
                                dim_v, length, packing[3], code)
    workspace = q.new_empty(size, dtype=torch.uint8)
    _lib.launch(library.pisa_full_attn_bwd, q.get_device(), *view(q), *view(k), *view(v), out.data_ptr(),
                None if low is None else low.data_ptr(), dout.data_ptr(), lse.data_ptr(), *packing, offset, code, batch,
                tokens, q_heads, heads, dim, dim_v, length, scale, int(causal), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                workspace.data_ptr(), size)
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
        ctx.set_materialize_grads(False)   # no zeros for lse
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        if dout is None:
            return (None,) * 8
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
    ``return_lse`` adds the [B,Tq,Hq] log-sum-exp (not differentiable).  The
    gradient is reverse mode only: forward mode raises RuntimeError.
    """
    _validate(q, k, v)
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
        cu_seqlens = _cumulative(cu_seqlens, q.shape[1], "cu_seqlens", q)
        cu_seqlens_k = cu_seqlens if same else _cumulative(cu_seqlens_k, k.shape[1], "cu_seqlens_k", q)
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
    if differentiated(q, k, v):
        out, lse = FullAttentionFunction.apply(q, k, v, cu_seqlens, cu_seqlens_k, offset, scale, bool(causal))
    else:
        out, lse, _ = _forward(q, k, v, cu_seqlens, cu_seqlens_k, offset, scale, causal, return_lse)
    return (out, lse) if return_lse else out


def prefix_attention(q, k, v, lengths, prefix_k=None, prefix_v=None, scale=None, return_lse=False):
    """Decode attention of the Tq newest tokens of every sequence -> [B,Tq,Hq,Dv].

    q [B,Tq,Hq,D]; k, v: the sequences' own caches [B,capacity,H,D|Dv] with
    ``lengths`` [B] valid keys each (this step's included; integers on the
    GPU, clamped to the capacity); prefix_k, prefix_v: [P,H,D|Dv], shared by
    all sequences and read once for the whole batch.  Token t sees the prefix
    and its own keys up to lengths - Tq + t; without any, it gives 0.  Made
    for a few tokens per sequence: own caches are read once per 16 query rows of
    a KV head, and B * Tq * Hq / H may not pass 1048560.  For
    inference: no gradient is recorded, and forward-mode tangents are refused.
    """
    _validate(q, k, v)
    if carries_tangent(q, k, v):
        raise ValueError("prefix_attention has no derivative")
    batch, tokens, q_heads, dim = q.shape
    _, capacity, heads, dim_v = v.shape
    device = q.get_device()
    if (not isinstance(lengths, torch.Tensor) or lengths.dim() != 1 or lengths.shape[0] != batch
            or lengths.dtype not in (torch.int32, torch.int64) or not lengths.is_cuda or lengths.get_device() != device):
        raise ValueError("lengths must be one integer per sequence on the query device")
    if (prefix_k is None) != (prefix_v is None):
        raise ValueError("prefix_k and prefix_v come together")
    scale = dim ** -0.5 if scale is None else float(scale)
    lengths = lengths.contiguous()
    q, k, v = aligned_rows(q), aligned_rows(k), aligned_rows(v)   # read through their pointers: no graph follows
    if batch > 1 and tokens > 1 and q.stride(0) != tokens * q.stride(1):
        q = q.contiguous()
    prefix, shared = 0, (None, 0, 0, None, 0, 0)
    if prefix_k is not None:
        if carries_tangent(prefix_k, prefix_v):
            raise ValueError("prefix_attention has no derivative")
        if (prefix_k.dim() != 3 or prefix_k.shape[1:] != k.shape[2:] or prefix_v.shape != (*prefix_k.shape[:2], dim_v)
                or any(t.dtype != q.dtype or t.device != q.device for t in (prefix_k, prefix_v))):
            raise ValueError("prefix_k and prefix_v must have shape [P,H,D] with the caches' heads, dims, dtype and device")
        prefix = prefix_k.shape[0]
        if prefix:
            prefix_k, prefix_v = aligned_rows(prefix_k), aligned_rows(prefix_v)
            shared = (prefix_k.data_ptr(), *prefix_k.stride()[:2], prefix_v.data_ptr(), *prefix_v.stride()[:2])
    out = q.new_empty((batch, tokens, q_heads, dim_v))
    lse = q.new_empty((batch, tokens, q_heads), dtype=torch.float32) if return_lse else None
    code = _lib.DTYPES[q.dtype]
    size = _lib.workspace_bytes("pisa_prefix_attn_workspace_bytes", device, batch, tokens, q_heads, heads, dim, dim_v,
                                capacity, prefix, code)
    if size < 0:
        raise ValueError("shapes outside the envelope of prefix_attention")
    workspace = q.new_empty(size, dtype=torch.uint8)
    _lib.launch(_lib.lib().pisa_prefix_attn, device, *view(q), *view(k), *view(v), lengths.data_ptr(),
                lengths.element_size(), *shared, code, batch, tokens, q_heads, heads, dim, dim_v, capacity, prefix, scale,
                out.data_ptr(), None if lse is None else lse.data_ptr(), workspace.data_ptr(), size)
    if _lib.status_checks():
        _lib.check_workspace(workspace, q.device)
    return (out, lse) if return_lse else out


# elements of an output that are joined at a time: half a gigabyte of fp32
JOIN_ELEMENTS = 1 << 27


def continued_attention(q, k, v, prefix_k, prefix_v):
    """Attention of many new tokens q [B,T,Hq,D] of every sequence, the last
    ones of its own k, v [B,N,H,D|Dv], over a prefix [P,H,D|Dv] that all share
    and their own keys -> [B,T,Hq,Dv].

    prefix_attention's result for prompts after a shared prefix, on
    full_attention's tiles: the queries of the whole batch against the prefix
    as one sequence, each sequence against its own keys, joined by their
    log-sum-exp in fp32 (with what rounding dropped from either part).  No
    gradient is recorded.
    """
    _validate(q, k, v)
    _, offset = query_positions(q, k)
    batch, tokens, heads, dim = q.shape
    scale, q = dim ** -0.5, aligned_rows(q)
    own = _forward(q, aligned_rows(k), aligned_rows(v), None, None, offset, scale, True, True, True)
    rows = aligned_rows(q.reshape(1, batch * tokens, heads, dim))
    shared = _forward(rows, aligned_rows(prefix_k[None]), aligned_rows(prefix_v[None]), None, None, 0, scale, False, True, True)
    shared = [None if t is None else t.view(batch, tokens, *t.shape[2:]) for t in shared]
    out, step = own[0], max(1, JOIN_ELEMENTS // own[0][0].numel())
    for b in range(0, batch, step):
        at = slice(b, b + step)
        top = torch.maximum(own[1][at], shared[1][at])
        weights = [(part[1][at] - top).exp_()[..., None] for part in (own, shared)]
        total = torch.zeros_like(out[at], dtype=torch.float32)
        for (value, _, low), weight in zip((own, shared), weights):
            exact = value[at].float()
            if low is not None:
                exact += low[at]
            total += exact.mul_(weight)
        out[at] = total.div_(weights[0] + weights[1])
    return out
