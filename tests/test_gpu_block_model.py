"""The decoder block on residual_norm, 8-bit checkpoints and 8-bit projections."""

import copy
from dataclasses import replace

import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def config(**kw):
    from nlogn_pisa_b200.model import BlockConfig

    return BlockConfig(**{**dict(vocab_size=500, hidden_size=128, intermediate_size=352, num_attention_heads=4,
                                 num_key_value_heads=2, head_dim=32, attention_method="full"), **kw})


def blocks(dtype=F32, **kw):
    """A block of plain torch operations and one with the same parameters and ``kw``."""
    from nlogn_pisa_b200.model import DecoderBlock

    torch.manual_seed(1)
    plain = DecoderBlock(config(init_std=0.1)).to("cuda", dtype)
    other = DecoderBlock(config(init_std=0.1, **kw)).to("cuda", dtype)
    other.load_state_dict(plain.state_dict(), strict=False)
    return plain, other


def off(x, y):
    return float((x.double() - y.double()).norm() / y.double().norm())


@pytest.mark.parametrize("packed", [False, True])
def test_fused_norms_are_the_blocks(cuda_device, packed):
    """The same function and gradients.  Each of about twelve operators in fp32 is off by some hundred units of
    2^-24 and passes errors on at most tenfold: 7e-4 of the norm, and as much again for gradients."""
    plain, fused = blocks(fused_norms=True)
    tokens = torch.randint(0, 500, (1, 60) if packed else (3, 20), device="cuda")
    cu = torch.tensor([0, 13, 60], dtype=torch.int32, device="cuda") if packed else None
    d = torch.randn(*tokens.shape, 128, device="cuda")
    outs = [m(tokens, cu_seqlens=cu) for m in (plain, fused)]
    assert off(outs[1], outs[0]) < 7e-4
    grads = [torch.autograd.grad(o, list(m.parameters()), d) for o, m in zip(outs, (plain, fused))]
    for x, y in zip(*grads):
        assert off(y, x) < 1.4e-3


def test_all_options_train(cuda_device):
    """Post norms, gates, scales and 8-bit checkpoints at once: every parameter has a finite gradient."""
    _, block = blocks(BF16, post_norm=True, branch_gate=True, residual_scale=0.9, branch_scale=0.5, checkpoint_bits=8, bias=True)
    out = block(torch.randint(0, 500, (2, 37), device="cuda"))
    out.float().square().mean().backward()
    assert {n for n, _ in block.named_parameters()} >= {"join1.post_norm", "join1.gate", "join2.post_norm", "join2.gate"}
    for name, p in block.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()) and bool(p.grad.any()), name


def test_checkpoints_leave_the_forward_alone(cuda_device):
    """The forward is the one without them but for the product's roundings (a plain silu rounds in between);
    gradients stay within what steps of 1/254 of a group's largest value can move."""
    plain, kept = blocks(F32, checkpoint_bits=8)
    tokens = torch.randint(0, 500, (2, 50), device="cuda")
    outs = [m(tokens) for m in (plain, kept)]
    assert off(outs[1], outs[0]) < 7e-4
    d = torch.randn_like(outs[0])
    grads = [torch.autograd.grad(o, list(m.parameters()), d) for o, m in zip(outs, (plain, kept))]
    # a group's values are off by up to 1/254 of its largest, which is at most 11.3 times its rms: 4.5% each for gate, up and x
    for x, y in zip(*grads):
        assert off(y, x) < 0.14


@pytest.mark.parametrize("method", ["full", "pisa2"])
@pytest.mark.parametrize("options", [{}, {"post_norm": True, "branch_gate": True, "branch_scale": 0.5, "bias": True}])
def test_int8_block_is_its_operators(cuda_device, method, options):
    """Each step against its own definition from the step before; the block is the steps, bit for bit."""
    import nlogn_pisa_b200 as P
    from nlogn_pisa_b200 import mixer
    from nlogn_pisa_b200.model import DecoderBlock, Int8DecoderBlock

    torch.manual_seed(2)
    cfg = config(attention_method=method, head_dim=64, topk=8, block_size=16, branching=2, init_std=0.1, **options)
    block = DecoderBlock(cfg).to("cuda", BF16)
    served = Int8DecoderBlock(block, cfg)
    tokens = torch.randint(0, 500, (2, 90), device="cuda")
    out, cache = served(tokens)
    assert cache is None
    with torch.no_grad():
        x = block.embed(tokens)
        n = P.residual_norm(x, None, block.norm1.weight, eps=cfg.rms_norm_eps)[1]
        qkv = served.attn.qkv_proj(n)
        projections = [getattr(block.attn, p) for p in ("q_proj", "k_proj", "v_proj")]
        w, ws = R.quantized(torch.cat([p.weight for p in projections]).detach().float())
        values, scale = R.quantized(n.float())
        bias = None if projections[0].bias is None else torch.cat([p.bias for p in projections]).float()
        R.check("qkv", qkv, *R.int8_linear(values, scale, w, ws, bias, BF16))
        for part, p in zip(mixer._projections(served.attn, n), projections):
            assert torch.equal(part.flatten(2), P.Int8Linear.from_linear(p)(n))
        a, _ = served.attn(n)
        join = block.join1
        kw = dict(post_weight=join.post_norm, gate=join.gate, branch_scale=cfg.branch_scale) if options else {}
        h, n8, s = P.residual_norm(x, a, block.norm2.weight, eps=cfg.rms_norm_eps, quantize=True, **kw)
        both = served.ffn.gate_up(n8, s, BF16)
        w, ws = R.quantized(torch.cat((block.ffn.gate.weight, block.ffn.up.weight)).detach().float())
        bias = None if block.ffn.gate.bias is None else torch.cat((block.ffn.gate.bias, block.ffn.up.bias)).float()
        R.check("gate_up", both, *R.int8_linear(n8, s, w, ws, bias, BF16))
        a8, s8 = P.swiglu(both[..., :352], both[..., 352:], quantize=True)
        f = served.ffn.down(a8, s8, BF16)
        w, ws = R.quantized(block.ffn.down.weight.detach().float())
        R.check("down", f, *R.int8_linear(a8, s8, w, ws, None if bias is None else block.ffn.down.bias.float(), BF16))
        kw = dict(post_weight=block.join2.post_norm, gate=block.join2.gate, branch_scale=cfg.branch_scale) if options else {}
        assert torch.equal(P.residual_norm(h, f, block.norm_out.weight, eps=cfg.rms_norm_eps, **kw)[1], out)


def test_int8_block_with_a_cache(cuda_device):
    """A prompt in pieces gives each token what the whole prompt gives it, but for the rounding of shared steps:
    every token's rows are its own, so the only difference is attention's (bf16 tolerance of its operators)."""
    from nlogn_pisa_b200.model import DecoderBlock, Int8DecoderBlock

    torch.manual_seed(3)
    cfg = config(head_dim=64)
    served = Int8DecoderBlock(DecoderBlock(cfg).to("cuda", BF16), cfg)
    tokens = torch.randint(0, 500, (2, 40), device="cuda")
    whole, _ = served(tokens)
    parts, cache = [], None
    for piece in tokens.split([24, 1, 1, 14], 1):
        out, cache = served(piece, cache=cache, use_cache=True)
        parts.append(out)
    # attention's outputs differ by 2^-8 of themselves; the 8-bit steps behind it move by one where they are near a border
    assert off(torch.cat(parts, 1), whole) < 4 * 2.0 ** -8
    assert cache["k"].shape[1] == 40


def test_plain_block_is_unchanged(cuda_device):
    """Without the options the block has the parameters and operations that it had."""
    from nlogn_pisa_b200.model import DecoderBlock

    plain, _ = blocks()
    assert plain.join1 is None and not any("join" in n for n, _ in plain.named_parameters())
    tokens = torch.randint(0, 500, (2, 12), device="cuda")
    x = plain.embed(tokens)
    x = x + plain.attn(plain.norm1(x))[0]
    want = plain.norm_out(x + plain.ffn.down(torch.nn.functional.silu(plain.ffn.gate(plain.norm2(x))) * plain.ffn.up(plain.norm2(x))))
    assert torch.equal(plain(tokens), want)
    again = copy.deepcopy(plain)
    assert torch.equal(again(tokens), want)
    with pytest.raises(ValueError, match="checkpoint_bits"):
        DecoderBlock(replace(config(), checkpoint_bits=4))
