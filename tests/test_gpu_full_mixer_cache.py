"""The full-attention token mixer with caches: long continuations over a shared prompt."""

import pytest
import torch

from test_gpu_full_mixer import make, near, plain

pytestmark = pytest.mark.gpu


def answers(mixer, prompt, x, steps):
    """Outputs of x's tokens after a shared prompt, in steps of the given lengths."""
    from nlogn_pisa_b200.mixer import FullAttention

    with torch.no_grad():
        _, cache = mixer(prompt, use_cache=True)
        cache = FullAttention.share_prefix(cache)
        out, begin = [], 0
        for n in steps:
            y, cache = mixer(x[:, begin:begin + n], cache=cache, use_cache=True)
            out.append(y)
            begin += n
    return torch.cat(out, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (4, 4, 128), (8, 1, 96), (2, 1, 160)])
@pytest.mark.parametrize("prompt,steps", [(200, [1, 500, 1, 300]), (1, [17, 16, 129]), (700, [256]), (333, [15, 400, 3])])
def test_long_answers_share_a_prompt(cuda_device, dtype, heads, kv_heads, head_dim, prompt, steps):
    mixer = make(dtype, num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=head_dim)
    first = torch.randn(1, prompt, 256, device="cuda").to(dtype)
    x = torch.randn(3, sum(steps), 256, device="cuda").to(dtype)
    want = plain(mixer, torch.cat((first.expand(3, -1, -1), x), 1))[:, prompt:]
    near(answers(mixer, first, x, steps), want, dtype)


def test_many_rows(cuda_device):
    """More query rows per KV head than the decode kernels take."""
    mixer = make(torch.bfloat16, num_attention_heads=16, num_key_value_heads=1, head_dim=64)
    first = torch.randn(1, 300, 256, device="cuda").to(torch.bfloat16)
    x = torch.randn(64, 1100, 256, device="cuda").to(torch.bfloat16)
    got = answers(mixer, first, x, [1, 1099])
    for b in (0, 31, 63):
        near(got[b:b + 1], plain(mixer, torch.cat((first, x[b:b + 1]), 1))[:, 300:], torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_continued_attention_is_prefix_attention(cuda_device, dtype):
    """The same operation as the decode kernels', within what either rounds (the output, and its weights)."""
    import nlogn_pisa_b200 as P
    from nlogn_pisa_b200 import dense

    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(2, n, h, 64, generator=gen, device="cuda").to(dtype) for n, h in ((90, 4), (200, 2), (200, 2)))
    pk, pv = (torch.randn(500, 2, 64, generator=gen, device="cuda").to(dtype) for _ in range(2))
    want = P.prefix_attention(q, k, v, torch.tensor([200, 200], device="cuda"), prefix_k=pk, prefix_v=pv)
    tight = dense.JOIN_ELEMENTS
    got = dense.continued_attention(q, k, v, pk, pv)
    try:
        dense.JOIN_ELEMENTS = 1      # a sequence at a time
        assert torch.equal(got, dense.continued_attention(q, k, v, pk, pv))
    finally:
        dense.JOIN_ELEMENTS = tight
    unit = {torch.float32: 64 * 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    assert float((got.double() - want.double()).norm()) <= 2 * unit * float(want.double().norm())
