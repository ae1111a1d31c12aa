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
