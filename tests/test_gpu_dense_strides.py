"""Dense operators on views whose dimensions of one element have strides of their own."""

import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


def odd(t, stride):
    """The same elements with ``stride`` for every dimension of one element (the last one apart)."""
    strides = [stride if n == 1 and i + 1 < t.dim() else s for i, (n, s) in enumerate(zip(t.shape, t.stride()))]
    return t.as_strided(t.shape, strides)


def test_no_copy_for_single_elements():
    from nlogn_pisa_b200.dense import aligned_rows

    one = torch.zeros(2, 5, 64, 1, dtype=BF16).transpose(2, 3)     # [2, 5, 1, 64] with a head stride of 1
    assert one.stride(2) == 1 and aligned_rows(one) is one
    part = odd(torch.zeros(2, 9, 1, 64, dtype=BF16)[:, :5], 3)     # not contiguous
    assert not part.is_contiguous() and aligned_rows(part) is part
    assert aligned_rows(torch.zeros(2, 5, 1, 64, dtype=BF16).expand(2, 5, 2, 64)).is_contiguous()   # broadcast heads are copied


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("stride", [1, 3, 1 << 33])
@pytest.mark.parametrize("batch,tokens,keys,heads,kv_heads", [(1, 1, 1, 1, 1), (1, 70, 300, 2, 1), (3, 1, 130, 4, 1), (1, 1, 200, 4, 2),
                                                              (2, 33, 33, 1, 1)])
def test_same_bits(cuda_device, dtype, stride, batch, tokens, keys, heads, kv_heads):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(keys)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    q, k, v, dout = (normal(batch, n, h, 64) for n, h in ((tokens, heads), (keys, kv_heads), (keys, kv_heads), (tokens, heads)))
    kq = normal(batch, tokens, kv_heads, 64)
    pk, pv = normal(90, kv_heads, 64), normal(90, kv_heads, 64)
    n = torch.full((batch,), keys, dtype=torch.int32, device="cuda")
    w, frequency = torch.ones(64, device="cuda"), torch.rand(32, device="cuda")

    def results(view):
        leaves = [view(x.detach()).requires_grad_(True) for x in (q, k, v)]
        out = P.full_attention(*leaves)
        found = [out, *torch.autograd.grad(out, leaves, view(dout))]
        found.append(P.prefix_attention(view(q), view(k), view(v), n))
        found.append(P.prefix_attention(view(q), view(k), view(v), n, prefix_k=view(pk), prefix_v=view(pv)))
        leaves = [view(x.detach()).requires_grad_(True) for x in (q, kq)]
        out = P.qk_norm_rotary(*leaves, w, w, frequency)
        return [*found, *out, *torch.autograd.grad(out, leaves, (view(dout), view(kq)))]

    for x, y in zip(results(lambda t: t), results(lambda t: odd(t, stride))):
        assert torch.equal(x, y)
