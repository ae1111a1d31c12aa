"""The PISA token mixer of the xmixers LLaMA models, on this library.

Mirror of PyramidSparseAttention
(xmixers/xmixers/modules/token_mixers/vanilla_attention/pyramid_sparse_attention.py:71-222):
q/k/v projections, split-half rotary encoding of q and k (pisa_rotary), block
selection and attention over the selected blocks (select_blocks /
sparse_attention), the output projection, and the decode cache (PyramidCache
for keys, TensorCache for values) with the same dictionary layout.  The
config is duck-typed: any object with the PisaConfig field names
(xmixers/xmixers/pisa_config.py:8-46) works.  PyramidSparseAttention serves the
PISA selection methods (pisa, pisa1, pisa2), FullAttention the layers between
them that see every key (attention_method "full"); NSA is another layer.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib, dense
from .attention import sparse_attention
from .cache import PyramidCache, TensorCache
from .dense import full_attention
from .norm_rotary import qk_norm_rotary
from .selection import select_blocks


def rotary_frequencies(head_dim, base, fraction):
    """Per-pair frequencies base^(-2i/D) for the first int(D/2 * fraction) pairs,
    0 for the rest (the xmixers RotaryEmbedding, lrpe.py:20-27 with type 3)."""
    theta = base ** (-2 / head_dim * torch.arange(head_dim // 2, dtype=torch.int64)).float()
    theta[int(head_dim // 2 * fraction):] = 0
    return theta


def token_positions(length, device, cu_seqlens=None, offset=0):
    """[1, length] positions; under cu_seqlens each document restarts at 0
    (pyramid_sparse_attention.py:6-11)."""
    positions = torch.arange(length, device=device)[None] + offset
    if cu_seqlens is not None:
        for begin, end in zip(cu_seqlens[:-1].tolist(), cu_seqlens[1:].tolist()):
            positions[:, begin:end] -= begin
    return positions


def _projections(mixer, x):
    """q [B,T,Hq,D], k and v [B,T,H,D] of a mixer: three products, or one whose
    outputs lie side by side where the mixer has been given a ``qkv_proj``
    (``model.int8_projections``)."""
    cfg = mixer.config
    heads = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.num_key_value_heads
    joined = getattr(mixer, "qkv_proj", None)
    if joined is None:
        parts = mixer.q_proj(x), mixer.k_proj(x), mixer.v_proj(x)
    else:
        parts = joined(x).split([n * cfg.head_dim for n in heads], -1)
    return [t.view(*x.shape[:2], n, cfg.head_dim) for t, n in zip(parts, heads)]


def _rotary(x, frequency, positions):
    out = torch.empty_like(x)
    pos = positions.to(device=x.device, dtype=torch.int64).contiguous()
    pos_sb = 0 if pos.shape[0] == 1 else pos.stride(0)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().pisa_rotary(
            _lib.ptr(x), *x.stride()[:3], _lib.ptr(out), *out.stride()[:3], _lib.ptr(pos), pos_sb, 0,
            _lib.ptr(frequency), _lib.dtype_code(x), *x.shape, _lib.stream_of(x.device)))
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, frequency, positions):
        ctx.save_for_backward(frequency, positions)
        return _rotary(x.contiguous() if x.stride(-1) != 1 else x, frequency, positions)

    @staticmethod
    def backward(ctx, dout):
        frequency, positions = ctx.saved_tensors
        # the transpose of a rotation by a is the rotation by -a
        return _rotary(dout.contiguous(), -frequency, positions), None, None


class RotaryEmbedding(nn.Module):
    def __init__(self, head_dim, base, fraction):
        super().__init__()
        if head_dim % 2:
            raise ValueError("RoPE needs an even head dimension")
        self.register_buffer("theta", rotary_frequencies(head_dim, base, fraction).reshape(1, -1), persistent=False)

    def forward(self, x, positions):
        if not x.is_cuda:
            raise ValueError("nlogn_pisa_b200 runs on CUDA tensors only; there is no CPU path")
        frequency = self.theta.flatten().to(device=x.device, dtype=torch.float32).contiguous()
        return _Rotary.apply(x, frequency, positions)


class PyramidSparseAttention(nn.Module):
    """Drop-in PISA token mixer (same parameter names, forward signature and cache layout)."""

    METHODS = ("pisa1", "pisa2", "pisa")

    def __init__(self, config, layer_idx=0):
        super().__init__()
        if config.attention_method not in self.METHODS:
            raise ValueError(f"attention_method {config.attention_method!r} is not served by nlogn_pisa_b200")
        self.config = config
        self.layer_idx = layer_idx
        # pyramid branching: the reference's is 2; a config may ask for 4 (this library's extension)
        self.branching = getattr(config, "branching", 2)
        q_width = config.num_attention_heads * config.head_dim
        kv_width = config.num_key_value_heads * config.head_dim
        self.q_proj = nn.Linear(config.hidden_size, q_width, bias=config.bias)
        self.k_proj = nn.Linear(config.hidden_size, kv_width, bias=config.bias)
        self.v_proj = nn.Linear(config.hidden_size, kv_width, bias=config.bias)
        self.o_proj = nn.Linear(q_width, config.hidden_size, bias=config.bias)
        self.rope = RotaryEmbedding(config.head_dim, config.rope_theta, config.rope_fraction)

    def forward(self, x, cu_seqlens=None, cache=None, use_cache=False, backend=None, attention_mask=None,
                past_key_values=None, **kwargs):
        if attention_mask is not None and not bool(attention_mask.all()):
            raise ValueError("Remove evaluation padding before native attention")
        if past_key_values is not None:
            cache = past_key_values[self.layer_idx] if len(past_key_values) > self.layer_idx else None
        cfg = self.config
        batch, length, _ = x.shape
        q, raw_k, v = _projections(self, x)
        offset = 0 if cache is None else cache["k"].shape[1]
        boundaries = cu_seqlens if cfg.rope_position_mode == "document" else None
        positions = token_positions(length, x.device, boundaries, offset)
        q = self.rope(q, positions)
        k = self.rope(raw_k, positions)
        pyramid = None
        next_cache = None
        if use_cache:
            next_cache = {} if cache is None else cache
            pyramid = (PyramidCache.from_keys(k.detach(), block_size=cfg.block_size, branching=self.branching)
                       if cache is None else cache["pyramid"].append(k.detach()))
            next_cache["pyramid"] = pyramid
            values = TensorCache.from_tensor(v.detach()) if cache is None else cache["value_storage"].append(v.detach())
            k, v = pyramid.keys, values.tensor
            next_cache.update(k=k, v=v, value_storage=values)
        elif cache is not None:
            k = torch.cat((cache["k"], k), dim=1)
            v = torch.cat((cache["v"], v), dim=1)
        schedule = "fused" if cache is not None and length == 1 else (cfg.prefill_routing or "auto")
        indices = select_blocks(q.detach(), k.detach(), method=cfg.attention_method, block_size=cfg.block_size,
                                topk=cfg.topk, cu_seqlens=cu_seqlens, query_offset=offset,
                                force_first=cfg.force_first, force_recent=cfg.force_recent, pyramid=pyramid,
                                leaf_tile=cfg.leaf_tile, routing_schedule=schedule, branching=self.branching)
        output = sparse_attention(q, k, v, indices, block_size=cfg.block_size, cu_seqlens=cu_seqlens,
                                  query_offset=offset)
        if past_key_values is not None and use_cache:
            while len(past_key_values) <= self.layer_idx:
                past_key_values.append(None)
            past_key_values[self.layer_idx] = next_cache
            next_cache = past_key_values
        return self.o_proj(output.reshape(batch, length, -1)), next_cache


def _attend_cache(q, stores, prefix, decode_tokens):
    """Attention of the newest tokens over the caches that end with them, and a shared prompt."""
    batch, tokens = q.shape[:2]
    if tokens <= decode_tokens:
        lengths = torch.full((batch,), stores[0].length, dtype=torch.int32, device=q.device)
        return dense.prefix_attention(q, stores[0].buffer, stores[1].buffer, lengths, prefix_k=prefix[0], prefix_v=prefix[1])
    keys, values = stores[0].tensor, stores[1].tensor
    if prefix[0] is not None:
        return dense.continued_attention(q, keys, values, *prefix)
    return full_attention(q, keys, values)


class _CachedAttention(torch.autograd.Function):
    """_attend_cache with the gradient in the newest tokens' q, k and v; what was
    cached before them is constant.  The backward recomputes over the cache:
    caches only grow at their end, so the rows it keeps hold what they held."""

    @staticmethod
    def forward(ctx, q, k, v, stores, prefix, decode_tokens):
        ctx.save_for_backward(q)
        ctx.cached = (stores[0].tensor, stores[1].tensor, *prefix)
        return _attend_cache(q, stores, prefix, decode_tokens)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, = ctx.saved_tensors
        keys, values, prefix_k, prefix_v = ctx.cached
        tokens = q.shape[1]
        if prefix_k is not None:
            keys, values = (torch.cat((p[None].expand(x.shape[0], -1, -1, -1), x), 1)
                            for p, x in ((prefix_k, keys), (prefix_v, values)))
        with torch.enable_grad():
            leaves = [x.detach().requires_grad_(True) for x in (q, keys, values)]
            out = full_attention(*leaves)
        dq, dk, dv = torch.autograd.grad(out, leaves, dout)
        return dq, dk[:, -tokens:], dv[:, -tokens:], None, None, None


class FullAttention(nn.Module):
    """Full-attention token mixer: projections, per-head norms of q and k with the
    rotation (qk_norm_rotary), attention over all keys, output projection.

    Training and prompts run full_attention (batches, or packed documents under
    ``cu_seqlens``).  With a cache, up to ``DECODE_TOKENS`` new tokens per
    sequence run prefix_attention over the cache, longer continuations
    full_attention again (continued_attention over a shared prefix).
    ``share_prefix`` turns the cache of one prompt into the start of a batch of
    answers to it, without copying its keys.
    With a cache, gradients reach this call's tokens; what earlier calls cached
    is constant.  A call with a cache and without ``use_cache`` (a look ahead)
    copies the cache and leaves it as it is.
    """

    DECODE_TOKENS = 16

    def __init__(self, config, layer_idx=0):
        super().__init__()
        if config.attention_method != "full":
            raise ValueError(f"attention_method {config.attention_method!r} is not full attention")
        self.config = config
        self.layer_idx = layer_idx
        q_width = config.num_attention_heads * config.head_dim
        kv_width = config.num_key_value_heads * config.head_dim
        self.q_proj = nn.Linear(config.hidden_size, q_width, bias=config.bias)
        self.k_proj = nn.Linear(config.hidden_size, kv_width, bias=config.bias)
        self.v_proj = nn.Linear(config.hidden_size, kv_width, bias=config.bias)
        self.o_proj = nn.Linear(q_width, config.hidden_size, bias=config.bias)
        self.q_norm = nn.Parameter(torch.ones(config.head_dim))
        self.k_norm = nn.Parameter(torch.ones(config.head_dim))
        self.eps = getattr(config, "rms_norm_eps", 1e-6)
        self.register_buffer("theta", rotary_frequencies(config.head_dim, config.rope_theta, config.rope_fraction),
                             persistent=False)

    def _apply(self, fn, recurse=True):
        """Frequencies stay fp32 when the layer is cast to another type."""
        super()._apply(fn, recurse)
        cfg = self.config
        self.theta = rotary_frequencies(cfg.head_dim, cfg.rope_theta, cfg.rope_fraction).to(self.theta.device)
        return self

    @staticmethod
    def _document_positions(length, cu_seqlens, device):
        """token_positions of packed documents, without reading their lengths on the host."""
        at = torch.arange(length, device=device)
        cu = cu_seqlens.to(device=device, dtype=torch.int64)
        document = torch.searchsorted(cu[1:], at, right=True).clamp_(max=cu.shape[0] - 1)
        return (at - cu[document])[None]

    @staticmethod
    def share_prefix(cache):
        """A cache whose prompt (batch 1) is shared by the sequences that follow."""
        if cache["k"].shape[0] != 1 or cache.get("prefix_k") is not None:
            raise ValueError("a shared prefix is the cache of a single prompt")
        return {"prefix_k": cache["k"][0], "prefix_v": cache["v"][0], "key_storage": None, "value_storage": None}

    def forward(self, x, cu_seqlens=None, cache=None, use_cache=False, attention_mask=None, past_key_values=None, **kwargs):
        if attention_mask is not None and not bool(attention_mask.all()):
            raise ValueError("Remove evaluation padding before native attention")
        if past_key_values is not None:
            cache = past_key_values[self.layer_idx] if len(past_key_values) > self.layer_idx else None
        if cache is not None and cu_seqlens is not None:
            raise ValueError("packed documents start without a cache")
        cfg = self.config
        batch, length, _ = x.shape
        q, k, v = _projections(self, x)
        prefix_k = prefix_v = None
        past = shared = 0
        if cache is not None:
            prefix_k, prefix_v = cache.get("prefix_k"), cache.get("prefix_v")
            shared = 0 if prefix_k is None else prefix_k.shape[0]
            past = 0 if cache["key_storage"] is None else cache["key_storage"].length
        positions = None
        if cu_seqlens is not None and cfg.rope_position_mode == "document":
            positions = self._document_positions(length, cu_seqlens, x.device)
        weights = self.q_norm, self.k_norm
        if any(w.dtype not in (torch.float32, q.dtype) for w in weights) or weights[0].dtype != weights[1].dtype:
            weights = [w.float() for w in weights]   # fp32 weights keep their bits beside 16-bit activations
        q, k = qk_norm_rotary(q, k, *weights, self.theta, positions=positions, position_offset=shared + past, eps=self.eps)
        next_cache = None
        if use_cache or cache is not None:
            if cache is None or cache["key_storage"] is None:
                stores = TensorCache.from_tensor(k.detach()), TensorCache.from_tensor(v.detach())
            elif use_cache:
                stores = cache["key_storage"].append(k.detach()), cache["value_storage"].append(v.detach())
            else:   # a look ahead: the cache stays as it is
                stores = (TensorCache.from_tensor(cache["key_storage"].tensor).append(k.detach()),
                          TensorCache.from_tensor(cache["value_storage"].tensor).append(v.detach()))
            if use_cache:
                next_cache = {"k": stores[0].tensor, "v": stores[1].tensor, "key_storage": stores[0],
                              "value_storage": stores[1], "prefix_k": prefix_k, "prefix_v": prefix_v}
        if cache is None:
            output = full_attention(q, k, v, cu_seqlens=cu_seqlens)
        elif dense.differentiated(q, k, v):
            output = _CachedAttention.apply(q, k, v, stores, (prefix_k, prefix_v), self.DECODE_TOKENS)
        else:
            output = _attend_cache(q, stores, (prefix_k, prefix_v), self.DECODE_TOKENS)
        if past_key_values is not None and use_cache:
            while len(past_key_values) <= self.layer_idx:
                past_key_values.append(None)
            past_key_values[self.layer_idx] = next_cache
            next_cache = past_key_values
        return self.o_proj(output.reshape(batch, length, -1)), next_cache
