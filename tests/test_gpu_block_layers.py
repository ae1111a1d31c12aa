"""Layers around the decoder block's operators on the GPU: what they refuse, keep and call."""

import pytest
import torch
from torch.autograd import forward_ad

import block_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("autocast", [False, True])
def test_ffn_refuses_weights_that_do_not_fit(cuda_device, autocast):
    """Refused on the host, before any kernel runs; the layer works on afterwards."""
    import nlogn_pisa_b200 as P

    x, gate, up, down = (torch.ones(*s, device="cuda", requires_grad=True) for s in ((3, 64), (16, 64), (8, 64), (64, 16)))
    with torch.autocast("cuda", dtype=BF16, enabled=autocast):
        for args in ((x, gate, up, down), (x, up, gate, down), (x, gate, gate[:, :32], down), (x, gate, gate, down[:, :8])):
            with pytest.raises(ValueError, match="must"):
                P.swiglu_ffn(*args)
        y = P.swiglu_ffn(x, gate, gate, down)
    # 16 products of silu(64) * 64 = 4096: exact in every type
    assert bool((y == 65536).all())


def config(**kw):
    from nlogn_pisa_b200.model import BlockConfig

    return BlockConfig(**{**dict(vocab_size=300, hidden_size=128, intermediate_size=352, num_attention_heads=4,
                                 num_key_value_heads=2, head_dim=64, topk=8, block_size=16, branching=2, init_std=0.1), **kw})


def test_int8_layers_refuse_tokens_with_gradients(cuda_device):
    """In grad mode a gradient would be lost; without it, and under no_grad, the layers run."""
    import nlogn_pisa_b200 as P
    from nlogn_pisa_b200 import mixer
    from nlogn_pisa_b200.model import Int8SwiGLU, SwiGLU, int8_projections

    torch.manual_seed(1)
    layers = [P.Int8Linear.from_linear(torch.nn.Linear(128, 48, device="cuda", dtype=BF16)),
              Int8SwiGLU(SwiGLU(128, 352, True).to("cuda", BF16))]
    for kind, method in ((mixer.FullAttention, "full"), (mixer.PyramidSparseAttention, "pisa2")):
        attention = int8_projections(kind(config(attention_method=method)).to("cuda", BF16))
        assert not any(p.requires_grad for p in attention.parameters())
        layers.append(lambda x, attention=attention: attention(x)[0])
    x = torch.randn(2, 40, 128, device="cuda", dtype=BF16)
    for layer in layers:
        leaf = x.clone().requires_grad_(True)
        for tokens in (leaf, leaf * 1):
            with pytest.raises(ValueError, match="inference"):
                layer(tokens)
        with torch.no_grad():
            quiet = layer(leaf)
        out = layer(x)
        assert torch.equal(out, quiet) and not out.requires_grad
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="inference"):
            layers[0](forward_ad.make_dual(x, torch.ones_like(x)))


def test_int8_mixers_leave_the_original_trainable(cuda_device):
    from nlogn_pisa_b200 import mixer
    from nlogn_pisa_b200.model import int8_projections

    attention = mixer.FullAttention(config(attention_method="full")).to("cuda", BF16)
    int8_projections(attention)
    assert all(p.requires_grad for p in attention.parameters()) and hasattr(attention, "q_proj")


@pytest.mark.parametrize("cast", [F16, BF16])
def test_int8_layer_cast_with_its_model(cuda_device, cast):
    """A cast changes the tokens' type, not what the layer holds: the same product of the same tokens."""
    import nlogn_pisa_b200 as P

    torch.manual_seed(2)
    linear = torch.nn.Linear(100, 30, device="cuda")
    layer, other = P.Int8Linear.from_linear(linear), P.Int8Linear.from_linear(linear).to(cast)
    x = torch.randn(5, 100, device="cuda").to(cast)
    assert torch.equal(other.bias, linear.bias)
    for out_dtype in (None, F32):
        assert torch.equal(layer(x, out_dtype=out_dtype), other(x, out_dtype=out_dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_checkpointed_ffn_around_other_layers(cuda_device, dtype):
    """With a hook or an adapter the layers are called: the same forward, and the gradients of the gated product's kept
    inputs, for the adapter too."""
    import nlogn_pisa_b200 as P
    from nlogn_pisa_b200.model import SwiGLU

    torch.manual_seed(3)
    ffn = SwiGLU(96, 200, True, 8).to("cuda", dtype)
    x = torch.randn(2, 9, 96, device="cuda", dtype=dtype, requires_grad=True)
    plain, calls = ffn(x), []
    hooks = [getattr(ffn, n).register_full_backward_hook(lambda *a: calls.append(1)) for n in ("gate", "up", "down")]
    out = ffn(x)
    assert torch.equal(out, plain)
    out.sum().backward()
    assert len(calls) == 3
    for hook in hooks:
        hook.remove()

    class Adapter(torch.nn.Module):
        def __init__(self, layer):
            super().__init__()
            self.layer, self.low = layer, torch.nn.Linear(layer.in_features, layer.out_features, False).to("cuda", dtype)

        def forward(self, x):
            return self.layer(x) + self.low(x)

    for name in ("gate", "up", "down"):
        setattr(ffn, name, Adapter(getattr(ffn, name)))
    d = torch.randn_like(plain)
    leaves = [x, *ffn.parameters()]
    got, want = ffn(x), ffn.down(P.swiglu(ffn.gate(x), ffn.up(x), checkpoint_bits=8))
    assert torch.equal(got, want)
    for g, w in zip(*(torch.autograd.grad(y, leaves, d) for y in (got, want))):
        assert torch.equal(g, w) and bool(g.any())


@pytest.mark.parametrize("options", [{"fused_norms": True}, {"post_norm": True, "branch_gate": True, "branch_scale": 0.5}])
def test_fused_block_with_watched_norms(cuda_device, options):
    """Hooks on the norms see their calls and change the outputs by a rounding of the residual stream at most."""
    from nlogn_pisa_b200.model import DecoderBlock, Int8DecoderBlock

    torch.manual_seed(4)
    cfg = config(attention_method="full", **options)
    block = DecoderBlock(cfg).cuda()
    tokens = torch.randint(0, 300, (2, 30), device="cuda")
    with torch.no_grad():
        plain = block(tokens)
    served = Int8DecoderBlock(block, cfg)
    served_plain, _ = served(tokens)
    seen = []
    hooks = [n.register_forward_hook(lambda m, args, out: seen.append((m, out)))
             for b in (block, served) for n in (b.norm1, b.norm2, b.norm_out)]
    out = block(tokens)
    # the bound of test_fused_norms_are_the_blocks: some hundred units of 2^-24 for each of about twelve operators
    assert len(seen) == 3 and float((out - plain).norm() / plain.norm()) < 7e-4
    grads = torch.autograd.grad(out.square().sum(), list(block.parameters()))
    assert all(bool(g.isfinite().all()) and bool(g.any()) for g in grads)
    seen.clear()
    hidden, _ = served(tokens)
    # here an 8-bit step may move: one of 127 to a value, in few of many
    assert len(seen) == 3 and float((hidden - served_plain).norm() / served_plain.norm()) < 1 / 127
    for hook in hooks:
        hook.remove()
    with torch.no_grad():
        assert torch.equal(block(tokens), plain) and torch.equal(served(tokens)[0], served_plain)


@pytest.mark.parametrize("method", ["full", "pisa2"])
@pytest.mark.parametrize("bias", [False, True])
def test_int8_output_projection(cuda_device, method, bias):
    """The mixer's last product against its definition, on the tokens that reach it."""
    from nlogn_pisa_b200.model import DecoderBlock, Int8DecoderBlock

    torch.manual_seed(5)
    block = DecoderBlock(config(attention_method=method, bias=bias)).to("cuda", BF16)
    served, seen = Int8DecoderBlock(block), []
    served.attn.o_proj.register_forward_hook(lambda m, args, out: seen.append((args[0], out)))
    served(torch.randint(0, 300, (2, 90), device="cuda"))
    (x, out), = seen
    projection = block.attn.o_proj
    w, ws = R.quantized(projection.weight.detach().float())
    values, scale = R.quantized(x.float())
    R.check("o_proj", out, *R.int8_linear(values, scale, w, ws, projection.bias.detach().float() if bias else None, BF16))


@pytest.mark.parametrize("method", ["full", "pisa2"])
@pytest.mark.parametrize("options", [{}, {"post_norm": True, "branch_gate": True, "branch_scale": 0.5, "bias": True}])
def test_int8_block_against_the_floating_block(cuda_device, method, options):
    """What eight roundings to 8 bits can move (tokens and weights of four products, all blocks attended).  A value is off
    by half a step, 1 / 254 of its row's largest, so a row by c / 254 of its norm, c the largest over the rms; products
    with random weights pass relative errors on as they are, and so does what follows them."""
    from nlogn_pisa_b200.model import DecoderBlock, Int8DecoderBlock

    torch.manual_seed(6)
    block = DecoderBlock(config(attention_method=method, **options)).cuda()
    rows = [p.detach() for m in block.modules() if isinstance(m, torch.nn.Linear) for p in (m.weight,)]
    hooks = [m.register_forward_pre_hook(lambda m, args: rows.append(args[0].detach()))
             for m in block.modules() if isinstance(m, torch.nn.Linear)]
    tokens = torch.randint(0, 300, (2, 90), device="cuda")
    with torch.no_grad():
        want = block(tokens)
    for hook in hooks:
        hook.remove()
    c = max(float((t.abs().amax(-1) / t.square().mean(-1).sqrt()).max()) for t in rows)
    assert len(rows) == 14 and c < 16
    got, _ = Int8DecoderBlock(block)(tokens)
    assert float((got - want).norm() / want.norm()) < 8 * c / 254
