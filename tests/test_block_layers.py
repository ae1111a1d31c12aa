"""Layers around the decoder block's operators: what they refuse, keep and call (no GPU)."""

import itertools

import pytest
import torch


@pytest.mark.parametrize("grad", [False, True])
def test_ffn_refuses_weights_that_do_not_fit(grad):
    """The gated product reads up's rows by gate's shape: a smaller up would be read past its end."""
    import nlogn_pisa_b200 as P

    def zeros(*shape):
        return torch.zeros(*shape, requires_grad=grad)

    x = zeros(3, 64)
    for shapes, word in ((((16, 64), (8, 64), (64, 16)), "w_gate and w_up must share"),
                         (((8, 64), (16, 64), (64, 8)), "w_gate and w_up must share"),
                         (((8, 32), (8, 32), (64, 8)), "w_gate and w_up must share"),
                         (((64,), (64,), (64, 8)), "w_gate and w_up must share"),
                         (((8, 64), (8, 64), (64, 16)), "w_down must"), (((8, 64), (8, 64), (8,)), "w_down must"),
                         (((0, 64), (0, 64), (64, 0)), "nonempty weights")):
        with pytest.raises(ValueError, match=word):
            P.swiglu_ffn(x, *(zeros(*s) for s in shapes))


def test_int8_layer_passes_its_tokens_on(monkeypatch):
    """Tokens reach int8_linear as they came: cut off from their graph, they would lose their gradient without a word."""
    from nlogn_pisa_b200 import int8

    seen = []
    monkeypatch.setattr(int8, "int8_linear", lambda x, *args, **kw: seen.append(x) or x)
    layer = int8.Int8Linear(32, 8)
    x = torch.zeros(2, 32, requires_grad=True)
    layer(x * 1)
    layer(x.detach())
    assert [t.requires_grad for t in seen] == [True, False]


def test_int8_layer_is_built_without_memory_first():
    """Under the meta device, then given memory, then loaded."""
    from nlogn_pisa_b200 import int8

    source = int8.Int8Linear(40, 6)
    for t in source.state_dict().values():
        t.copy_(torch.randint(-100, 100, t.shape))
    for cast in (False, True):
        with torch.device("meta"):
            model = torch.nn.Sequential(int8.Int8Linear(40, 6))
        model = (model.half() if cast else model).to_empty(device="cpu")
        assert model[0].weight_scale.dtype == torch.float32 and not model[0].weight_scale.is_meta
        model[0].load_state_dict(source.state_dict())
        for name, t in source.state_dict().items():
            assert torch.equal(model[0].state_dict()[name], t), name


def test_int8_layer_moves_with_its_model():
    from nlogn_pisa_b200 import int8

    layer = int8.Int8Linear(40, 6)
    layer.weight_scale.copy_(torch.rand(6))
    scale = layer.weight_scale.clone()
    for move in (lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.float16), lambda m: m.float()):
        move(layer)
        assert layer.weight_scale.dtype == torch.float32 and torch.equal(layer.weight_scale, scale)
        assert layer.weight.dtype == torch.int8
    assert layer.to("meta").weight_scale.is_meta


@pytest.mark.parametrize("cast", ["half", "bfloat16", "double"])
def test_int8_layer_keeps_its_bias_in_fp32(cast):
    """Values that 16 bits do not hold survive a cast, on their own and within a model."""
    from nlogn_pisa_b200 import int8

    layer = int8.Int8Linear(40, 6)
    bias = torch.tensor([1 + 2.0 ** -20, -3e-9, 70000.5, 0.1, 1e30, 0.0])
    layer.bias.copy_(bias)
    getattr(torch.nn.Sequential(layer), cast)()
    assert layer.bias.dtype == torch.float32 and torch.equal(layer.bias, bias)
    assert getattr(int8.Int8Linear(40, 6, bias=False), cast)().bias is None
    default = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        assert int8.Int8Linear(40, 6).bias.dtype == torch.float32
    finally:
        torch.set_default_dtype(default)


def without_kernels(monkeypatch):
    """Rounding and the products of 8-bit layers on the host."""
    from nlogn_pisa_b200 import int8

    def rounded(w):
        scale = w.abs().amax(-1) / 127
        return (w / scale[:, None]).round().to(torch.int8), scale

    monkeypatch.setattr(int8, "quantize_int8", rounded)
    monkeypatch.setattr(int8, "int8_linear", lambda x, w, s, bias=None, **kw: x @ (w * s[:, None]).T + (0 if bias is None else bias))


class Adapted(torch.nn.Linear):
    """A linear layer with a low-rank part beside its weight."""

    def __init__(self, inner, outer):
        super().__init__(inner, outer)
        self.low, self.high = torch.nn.Linear(inner, 4, bias=False), torch.nn.Linear(4, outer, bias=False)

    def forward(self, x):
        return super().forward(x) + self.high(self.low(x))


def watchers(module, seen):
    """Ways to watch calls of a module, each with its undoing."""
    own = module.forward
    yield module.register_forward_hook(lambda *a: seen.append(1)).remove
    yield module.register_forward_pre_hook(lambda *a: seen.append(1)).remove
    module.forward = lambda *a, **kw: (seen.append(1), own(*a, **kw))[1]
    yield lambda: module.__dict__.pop("forward")
    yield torch.nn.modules.module.register_module_forward_hook(lambda m, *a: m is module and seen.append(1) or None).remove


@pytest.mark.parametrize("name", ["gate", "up", "down"])
def test_checkpointed_ffn_calls_its_layers(monkeypatch, name):
    """Hooks and layers with a forward of their own are not passed by; plain layers run as one operator."""
    from torch.nn import functional as F

    from nlogn_pisa_b200 import model

    whole = []
    monkeypatch.setattr(model, "swiglu", lambda g, u, checkpoint_bits: F.silu(g) * u)
    monkeypatch.setattr(model, "swiglu_ffn", lambda x, wg, wu, wd, bg, bu, bd: whole.append(1) or F.linear(
        F.silu(F.linear(x, wg, bg)) * F.linear(x, wu, bu), wd, bd))
    ffn, x = model.SwiGLU(8, 12, True, 8), torch.randn(3, 8)
    plain = ffn(x)
    assert whole == [1]
    seen = []
    for count, undo in enumerate(watchers(getattr(ffn, name), seen), 1):
        assert torch.equal(ffn(x), plain) and len(seen) == count and len(whole) == count
        undo()
        assert torch.equal(ffn(x), plain) and len(seen) == count
    layer = getattr(ffn, name)
    setattr(ffn, name, Adapted(layer.in_features, layer.out_features))
    whole.clear()
    assert torch.equal(ffn(x), ffn.down(F.silu(ffn.gate(x)) * ffn.up(x))) and not whole
    # a weight computed from others is still the layer's weight
    setattr(ffn, name, torch.nn.utils.parametrizations.weight_norm(layer))
    ffn(x).sum().backward()
    assert whole and all(p.grad is not None for p in getattr(ffn, name).parameters())


@pytest.mark.parametrize("options", [{"fused_norms": True}, {"post_norm": True, "branch_gate": True, "branch_scale": 0.5}])
@pytest.mark.parametrize("name", ["norm1", "norm2", "norm_out"])
def test_fused_block_calls_its_norms(monkeypatch, name, options):
    """A norm with hooks, or of another kind, is called; a plain RMSNorm is part of the operator."""
    from nlogn_pisa_b200 import model

    def rms(t, eps):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)

    whole = []

    def joined(x, branch, weight, post_weight=None, gate=None, residual_scale=1.0, branch_scale=1.0, eps=1e-6, quantize=False):
        whole.append(weight)
        if branch is not None:
            branch = branch if post_weight is None else rms(branch, eps) * post_weight
            x = residual_scale * x + branch_scale * (branch if gate is None else gate * branch)
        return x, rms(x, eps) * weight

    class Mix(torch.nn.Module):
        def forward(self, x):
            return x.cumsum(1), None

    monkeypatch.setattr(model, "residual_norm", joined)
    block = model.DecoderBlock(model.BlockConfig(vocab_size=30, hidden_size=16, intermediate_size=24, num_attention_heads=2,
                                                 num_key_value_heads=2, head_dim=8, attention_method="full", **options))
    block.attn = Mix()
    tokens = torch.randint(0, 30, (2, 5))
    plain, norm = block(tokens), getattr(block, name)
    assert [w is n.weight for w, n in zip(whole, (block.norm1, block.norm2, block.norm_out))] == [True] * 3
    seen = []
    for count, undo in enumerate(watchers(norm, seen), 1):
        # the same function in another order: some units of 2^-24 on values of order 1
        assert torch.allclose(block(tokens), plain, rtol=0, atol=1e-4) and len(seen) == count
        undo()
        assert torch.equal(block(tokens), plain) and len(seen) == count
    other = torch.nn.LayerNorm(16)
    torch.nn.init.normal_(other.weight)
    inputs = []
    other.register_forward_hook(lambda m, args, out: inputs.append((args[0], out)))
    setattr(block, name, other)
    out = block(tokens)
    (h, n), = inputs
    assert not torch.equal(out, plain)
    if name == "norm_out":
        assert torch.equal(out, n)
    if name == "norm1":
        assert torch.equal(h, block.embed(tokens))
    out.sum().backward()
    assert other.weight.grad is not None and all(p.grad is not None for p in block.parameters())


def test_int8_forms_refuse_what_they_would_drop(monkeypatch):
    """An 8-bit layer takes over weights: adapters, hooks and other forwards would be lost without a word."""
    from nlogn_pisa_b200 import int8, model

    class Other(model.SwiGLU):
        def forward(self, x):
            return self.down(self.gate(x).relu() * self.up(x))

    without_kernels(monkeypatch)
    plain = torch.nn.Linear(32, 8)
    assert int8.Int8Linear.from_linear(plain, torch.nn.Linear(32, 4)).out_features == 12
    for undo in itertools.islice(watchers(plain, []), 3):
        with pytest.raises(ValueError, match="hooks or a forward"):
            int8.Int8Linear.from_linear(torch.nn.Linear(32, 4), plain)
        undo()
    # a weight computed from others is taken as it is
    int8.Int8Linear.from_linear(torch.nn.utils.parametrizations.weight_norm(plain))
    with pytest.raises(ValueError, match="hooks or a forward"):
        int8.Int8Linear.from_linear(Adapted(32, 8))
    model.Int8SwiGLU(model.SwiGLU(32, 48, True))
    with pytest.raises(ValueError, match="SwiGLU"):
        model.Int8SwiGLU(Other(32, 48, True))
    ffn = model.SwiGLU(32, 48, True)
    ffn.down = Adapted(48, 32)
    with pytest.raises(ValueError, match="hooks or a forward"):
        model.Int8SwiGLU(ffn)
    mixer = torch.nn.Module()
    mixer.o_proj = Adapted(32, 8)
    with pytest.raises(ValueError, match="hooks or a forward"):
        model.int8_projections(mixer)


def test_int8_copy_of_a_mixer_with_its_own_forward(monkeypatch):
    """Only this package's mixers know the joined projection; others find theirs where they left them."""
    from nlogn_pisa_b200 import int8, mixer, model

    class Mix(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.q_proj, self.k_proj, self.v_proj, self.o_proj = (torch.nn.Linear(16, 16) for _ in range(4))

        def forward(self, x):
            return self.o_proj(self.q_proj(x) * self.k_proj(x) + self.v_proj(x)), None

    class Masked(mixer.FullAttention):
        def forward(self, x):
            return self.o_proj(self.q_proj(x) * self.k_proj(x) + self.v_proj(x)), None

    without_kernels(monkeypatch)
    cfg = model.BlockConfig(hidden_size=16, num_attention_heads=2, num_key_value_heads=2, head_dim=8, attention_method="full", bias=True)
    x = torch.randn(2, 3, 16)
    for own in (Mix(), Masked(cfg)):
        copy = model.int8_projections(own)
        assert all(isinstance(getattr(copy, n), int8.Int8Linear) for n in ("q_proj", "k_proj", "v_proj", "o_proj"))
        assert torch.allclose(copy(x)[0], own(x)[0], atol=0.2)
    joined = model.int8_projections(mixer.FullAttention(cfg))
    assert joined.qkv_proj.out_features == 48 and not hasattr(joined, "q_proj")


@pytest.mark.parametrize("options", [{}, {"post_norm": True, "branch_gate": True, "branch_scale": 0.5}])
def test_int8_block_is_a_copy(monkeypatch, options):
    """Neither block follows the other's training or casts."""
    from nlogn_pisa_b200 import model

    without_kernels(monkeypatch)
    cfg = model.BlockConfig(vocab_size=30, hidden_size=16, intermediate_size=24, num_attention_heads=2, num_key_value_heads=2,
                            head_dim=8, attention_method="full", **options)
    block = model.DecoderBlock(cfg)
    served = model.Int8DecoderBlock(block, cfg)
    before = {n: t.clone() for n, t in served.state_dict().items()}
    with torch.no_grad():
        for p in block.parameters():
            p.add_(1)
    assert all(torch.equal(t, before[n]) for n, t in served.state_dict().items())
    assert not any(p.requires_grad for p in served.parameters()) and all(p.requires_grad for p in block.parameters())
    served.half()
    assert all(p.dtype == torch.float32 for p in block.parameters())
    held = {t.untyped_storage().data_ptr() for t in block.state_dict().values()}
    assert not held & {t.untyped_storage().data_ptr() for t in model.Int8DecoderBlock(block, cfg).state_dict().values()}


@pytest.mark.parametrize("given", [{"post_norm": True}, {"branch_gate": True}, {"branch_scale": 0.5}, {"residual_scale": 2.0}, {}])
def test_int8_block_joins_as_its_block_does(monkeypatch, given):
    """A configuration that differs from the block's adds no norm, gate or scale to the served form, and takes none away."""
    from dataclasses import replace

    from nlogn_pisa_b200 import model

    without_kernels(monkeypatch)
    calls = []

    def joined(x, branch, weight, **kw):
        calls.append(kw)
        return (x, x) if not kw.get("quantize") else (x, x, None)

    monkeypatch.setattr(model, "residual_norm", joined)
    base = model.BlockConfig(vocab_size=30, hidden_size=16, intermediate_size=24, num_attention_heads=2, num_key_value_heads=2,
                             head_dim=8, attention_method="full")
    for own, cfg in ((base, replace(base, **given)), (replace(base, **given), base), (replace(base, **given), None)):
        block = model.DecoderBlock(own)
        served = model.Int8DecoderBlock(block, cfg)
        x, a = torch.zeros(2, 3, 16), torch.zeros(2, 3, 16)
        for join in (served.join1, served.join2):
            calls.clear()
            join(x, a, served.norm2)
            assert (calls[0]["post_weight"] is not None, calls[0]["gate"] is not None) == (own.post_norm, own.branch_gate)
            assert (calls[0]["residual_scale"], calls[0]["branch_scale"]) == (own.residual_scale, own.branch_scale)
