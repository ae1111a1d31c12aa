"""Layers around the decoder block's operators: what they refuse, keep and call (no GPU)."""

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
