"""Layers around the decoder block's operators on the GPU: what they refuse, keep and call."""

import pytest
import torch

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
