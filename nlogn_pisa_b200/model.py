"""A LLaMA-style decoder block around the PISA or the full-attention token mixer, for training runs.

The block of the reference's xmixers LLaMA models
(xmixers/xmixers/models/transformer/llama/modeling_llama.py): pre-norm
RMSNorm -> PyramidSparseAttention (FullAttention with attention_method
"full") -> residual, RMSNorm -> SwiGLU FFN -> residual.  Norms, projections and
the FFN are ordinary torch operations (GEMMs on cuBLAS); the selection and the
attention forward/backward run in this library.  Used by the benchmark's training configuration (one block,
data-parallel over the GPUs of a node).

With ``fused_norms`` (or any of ``post_norm``, ``branch_gate``, ``residual_scale``,
``branch_scale``) the norms, gates and residual sums between the branches run in
``residual_norm``; with ``checkpoint_bits=8`` the FFN keeps its activations in 8
bits (``swiglu_ffn``).  ``Int8DecoderBlock`` serves a trained block with every
projection in 8 bits.
"""

from __future__ import annotations

import copy
from dataclasses import dataclass

import torch
from torch import nn
import torch.nn.functional as F

from .int8 import Int8Linear, quantize_int8
from .mixer import FullAttention, PyramidSparseAttention
from .residual_norm import residual_norm
from .swiglu import swiglu, swiglu_ffn
from .validation import bare


@dataclass
class BlockConfig:
    """The PisaConfig fields the block and its mixer read (xmixers/xmixers/pisa_config.py:8-46)."""

    vocab_size: int = 50257
    hidden_size: int = 1024
    intermediate_size: int = 2816
    num_attention_heads: int = 16
    num_key_value_heads: int = 16
    head_dim: int = 64
    attention_method: str = "pisa2"
    block_size: int = 64
    topk: int = 16
    branching: int = 4
    prefill_routing: str | None = "auto"
    leaf_tile: int = 4
    force_first: bool = True
    force_recent: int = 1
    rope_theta: float = 10000.0
    rope_fraction: float = 0.5
    rope_position_mode: str = "document"
    rms_norm_eps: float = 1e-5
    bias: bool = False
    init_std: float = 0.02
    fused_norms: bool = False           # norms and residual sums in residual_norm
    post_norm: bool = False             # a norm after each branch too
    branch_gate: bool = False           # a learned gate per channel of each branch
    residual_scale: float = 1.0
    branch_scale: float = 1.0
    checkpoint_bits: int | None = None  # 8: the FFN's activations in 8 bits until the backward


# hooks that torch runs around every module's call
_global_hooks = getattr(nn.modules.module, "_has_any_global_hook", None) or (lambda: False)


def replaceable(module, kind):
    """Whether an operator on the module's parameters may stand in for calling it: a bare ``kind``, and no hooks on all modules."""
    return bare(module, kind) and not _global_hooks()


class RMSNorm(nn.Module):
    def __init__(self, dim, eps):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.eps)
        return (y * self.weight.float()).to(x.dtype)


class SwiGLU(nn.Module):
    """down(silu(gate(x)) * up(x)); with ``checkpoint_bits=8`` in one operator where the three are plain layers.  Around
    layers with hooks or a forward of their own (adapters) they are called, and the gated product keeps its inputs in 8 bits."""

    def __init__(self, hidden, inner, bias, checkpoint_bits=None):
        super().__init__()
        if checkpoint_bits not in (None, 8):
            raise ValueError("checkpoint_bits must be None or 8")
        self.checkpoint_bits = checkpoint_bits
        self.gate = nn.Linear(hidden, inner, bias=bias)
        self.up = nn.Linear(hidden, inner, bias=bias)
        self.down = nn.Linear(inner, hidden, bias=bias)

    def forward(self, x):
        if self.checkpoint_bits == 8:
            if not all(replaceable(m, nn.Linear) for m in (self.gate, self.up, self.down)):
                return self.down(swiglu(self.gate(x), self.up(x), checkpoint_bits=8))
            return swiglu_ffn(x, self.gate.weight, self.up.weight, self.down.weight, self.gate.bias, self.up.bias,
                              self.down.bias)
        return self.down(F.silu(self.gate(x)) * self.up(x))


class BranchJoin(nn.Module):
    """What lies between a branch and the next norm: the branch's own norm and gate, and the scales.

    The next norm is part of the operator where it is a plain RMSNorm; one of another kind, or with hooks, is called on
    the residual stream."""

    def __init__(self, cfg: BlockConfig):
        super().__init__()
        self.post_norm = nn.Parameter(torch.ones(cfg.hidden_size)) if cfg.post_norm else None
        self.gate = nn.Parameter(torch.ones(cfg.hidden_size)) if cfg.branch_gate else None
        self.scales = cfg.residual_scale, cfg.branch_scale
        self.eps = cfg.rms_norm_eps

    def forward(self, x, branch, norm, quantize=False):
        """residual_norm of the residual stream and the branch, with the next norm's weight."""
        fused = replaceable(norm, RMSNorm)
        weights = [w if w is None or w.dtype in (torch.float32, x.dtype) else w.float()
                   for w in (norm.weight if fused else x.new_ones(x.shape[-1]), self.post_norm, self.gate)]
        if quantize:
            weights = [None if w is None else w.detach() for w in weights]
        results = residual_norm(x, branch.to(x.dtype), weights[0], post_weight=weights[1], gate=weights[2],
                                residual_scale=self.scales[0], branch_scale=self.scales[1],
                                eps=norm.eps if isinstance(norm, RMSNorm) else self.eps, quantize=quantize and fused)
        if fused:
            return results
        h = results[0]
        return (h, *quantize_int8(norm(h))) if quantize else (h, norm(h))

    @staticmethod
    def first(x, norm):
        """The norm before the first branch."""
        if not replaceable(norm, RMSNorm):
            return norm(x)
        weight = norm.weight if norm.weight.dtype in (torch.float32, x.dtype) else norm.weight.float()
        return residual_norm(x, None, weight, eps=norm.eps)[1]


class DecoderBlock(nn.Module):
    """Embedding -> one pre-norm block -> final norm; returns the hidden states."""

    def __init__(self, cfg: BlockConfig):
        super().__init__()
        self.embed = nn.Embedding(cfg.vocab_size, cfg.hidden_size)
        self.norm1 = RMSNorm(cfg.hidden_size, cfg.rms_norm_eps)
        self.attn = (FullAttention if cfg.attention_method == "full" else PyramidSparseAttention)(cfg)
        self.norm2 = RMSNorm(cfg.hidden_size, cfg.rms_norm_eps)
        self.ffn = SwiGLU(cfg.hidden_size, cfg.intermediate_size, cfg.bias, cfg.checkpoint_bits)
        self.norm_out = RMSNorm(cfg.hidden_size, cfg.rms_norm_eps)
        self.join1 = self.join2 = None
        if cfg.fused_norms or cfg.post_norm or cfg.branch_gate or (cfg.residual_scale, cfg.branch_scale) != (1.0, 1.0):
            self.join1, self.join2 = BranchJoin(cfg), BranchJoin(cfg)
        for m in self.modules():
            if isinstance(m, (nn.Linear, nn.Embedding)):
                nn.init.normal_(m.weight, std=cfg.init_std)

    def forward(self, tokens, cu_seqlens=None):
        x = self.embed(tokens)
        if self.join1 is not None:
            n = BranchJoin.first(x, self.norm1)
            a, _ = self.attn(n, **({} if cu_seqlens is None else {"cu_seqlens": cu_seqlens}))
            x, n = self.join1(x, a, self.norm2)
            return self.join2(x, self.ffn(n), self.norm_out)[1]
        # mixers that know no packed documents are called as before
        a, _ = self.attn(self.norm1(x), **({} if cu_seqlens is None else {"cu_seqlens": cu_seqlens}))
        x = x + a
        x = x + self.ffn(self.norm2(x))
        return self.norm_out(x)


class Int8SwiGLU(nn.Module):
    """A SwiGLU layer in 8 bits, for inference: both inner products as one, the gated product rounded on its way."""

    def __init__(self, ffn: SwiGLU):
        super().__init__()
        if not bare(ffn, SwiGLU):
            raise ValueError("only a SwiGLU without hooks or a forward of its own has an 8-bit form")
        self.gate_up = Int8Linear.from_linear(ffn.gate, ffn.up)
        self.down = Int8Linear.from_linear(ffn.down)

    def forward(self, x, x_scale=None, out_dtype=None):
        gate, up = self.gate_up(x, x_scale, out_dtype).chunk(2, -1)
        return self.down(*swiglu(gate, up, quantize=True), out_dtype=gate.dtype)


def int8_projections(module):
    """A copy of a token mixer for inference with its projections in 8 bits: q, k and v of this package's mixers as one
    product, which rounds the tokens once.  Its parameters take no gradients, and tokens that require one are refused."""
    module = copy.deepcopy(module).requires_grad_(False)
    own = type(module).forward in (FullAttention.forward, PyramidSparseAttention.forward) and "forward" not in module.__dict__
    if own and all(isinstance(getattr(module, n, None), nn.Linear) for n in ("q_proj", "k_proj", "v_proj")):
        module.qkv_proj = Int8Linear.from_linear(module.q_proj, module.k_proj, module.v_proj)
        del module.q_proj, module.k_proj, module.v_proj
    for name, child in list(module.named_children()):
        if isinstance(child, nn.Linear):
            setattr(module, name, Int8Linear.from_linear(child))
    return module


class Int8DecoderBlock(nn.Module):
    """A trained DecoderBlock on the GPU with its projections in 8 bits, for inference.

    Norms and residual sums run in residual_norm, which gives the FFN its tokens
    in 8 bits; the mixer's projections round theirs.  Returns the hidden states
    and the mixer's cache.  The block's parameters are copied: training or casting
    it afterwards leaves this one as it is, and the other way round.  Post norms, gates and scales are the block's own:
    ``cfg`` is not read.
    """

    def __init__(self, block: DecoderBlock, cfg: BlockConfig | None = None):
        super().__init__()
        # a block without joins adds its branches as they are
        join1, join2 = (j or BranchJoin(BlockConfig()) for j in (block.join1, block.join2))
        self.embed, self.norm1, self.norm2, self.norm_out, self.join1, self.join2 = (
            copy.deepcopy(m).requires_grad_(False) for m in (block.embed, block.norm1, block.norm2, block.norm_out, join1, join2))
        self.attn = int8_projections(block.attn)
        self.ffn = Int8SwiGLU(block.ffn)

    @torch.no_grad()
    def forward(self, tokens, cu_seqlens=None, cache=None, use_cache=False):
        x = self.embed(tokens)
        a, cache = self.attn(BranchJoin.first(x, self.norm1), cu_seqlens=cu_seqlens, cache=cache, use_cache=use_cache)
        h, n, scale = self.join1(x, a, self.norm2, quantize=True)
        return self.join2(h, self.ffn(n, scale, x.dtype), self.norm_out)[1], cache
