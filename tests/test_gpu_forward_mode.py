"""Forward-mode differentiation through the dense operators is refused, never dropped."""

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def tensors():
    gen = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(1, 8, h, 64, generator=gen, device="cuda").to(BF16) for h in (4, 2, 2)]


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [True, False])
def test_full_attention(cuda_device, which, grad):
    import nlogn_pisa_b200 as P

    x = tensors()
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        plain = P.full_attention(*x)         # no tangent: an ordinary call
        assert forward_ad.unpack_dual(plain).tangent is None
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="jvp"):
            P.full_attention(*x)


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_qk_norm_rotary(cuda_device, which):
    import nlogn_pisa_b200 as P

    q, k, _ = tensors()
    x = [q, k, torch.ones(64, device="cuda"), torch.ones(64, device="cuda")]
    frequency = torch.rand(32, device="cuda")
    with torch.no_grad(), forward_ad.dual_level():
        P.qk_norm_rotary(*x, frequency)
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="jvp"):
            P.qk_norm_rotary(*x, frequency)


@pytest.mark.parametrize("which", [0, 1, 2, 3, 4])
def test_prefix_attention(cuda_device, which):
    import nlogn_pisa_b200 as P

    q, k, v = tensors()
    x = [q[:, :1], k, v, k[0], v[0]]
    n = torch.tensor([8], dtype=torch.int32, device="cuda")
    with torch.no_grad(), forward_ad.dual_level():
        P.prefix_attention(*x[:3], n, *x[3:])
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(ValueError, match="derivative"):
            P.prefix_attention(*x[:3], n, *x[3:])


def test_functional_jvp(cuda_device):
    import nlogn_pisa_b200 as P

    q, k, v = tensors()
    n = torch.tensor([8], dtype=torch.int32, device="cuda")
    w, frequency = torch.ones(64, device="cuda"), torch.rand(32, device="cuda")
    for call in (lambda x: P.full_attention(x, k, v), lambda x: P.prefix_attention(x[:, :1], k, v, n),
                 lambda x: P.qk_norm_rotary(x, k, w, w, frequency)[0]):
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.jvp(call, (q,), (torch.ones_like(q),))
