"""full_attention over very many keys: sums that keep their bits, items that outlast half a second."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
UNIT = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
# a truncating accumulator of 24 bits loses at most half a unit per addition on
# average: 2^-24 / 16 of the sum per key and half of that over a run of 65536
TRUNCATION = 2.0 ** -13


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("keys,tokens,dim,dim_v", [(65536, 3, 64, 64), (65537, 130, 64, 64), (131072, 2, 128, 128), (140001, 300, 128, 72),
                                                   (300000, 70, 40, 40), (1 << 20, 2, 64, 128), (1 << 21, 1, 8, 8)])
@pytest.mark.parametrize("ramp", [0.0, 12.0, -12.0])
def test_like_weights_of_many_keys(cuda_device, dtype, keys, tokens, dim, dim_v, ramp):
    """Values with a mean; logits near equal, or rising or falling along the keys (the rows' maxima move)."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(keys + dim)
    q = torch.randn(1, tokens, 2, dim, generator=gen, device="cuda").mul_(0.1)
    k = torch.randn(1, keys, 1, dim, generator=gen, device="cuda")
    q[..., 0] = dim ** 0.5
    k[..., 0] = torch.linspace(0, abs(ramp), keys, device="cuda")[None, :, None] * (1 if ramp > 0 else -1)
    v = 0.5 + torch.randn(1, keys, 1, dim_v, generator=gen, device="cuda")
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    out, lse = P.full_attention(q, k, v, return_lse=True)
    for h in range(2):
        for t in range(0, tokens, max(1, tokens // 8)):
            seen = keys - tokens + t + 1
            logits = (k[0, :seen, 0].double() @ q[0, t, h].double()) * dim ** -0.5
            weights = torch.softmax(logits, 0)
            want = weights @ v[0, :seen, 0].double()
            # rounding of the output, truncation on the way, and at random the rounding of the weights
            room = (UNIT[dtype] + TRUNCATION) * float(want.norm())
            room += 4 * UNIT[dtype] * float((weights.square() @ v[0, :seen, 0].double().square()).sum().sqrt())
            assert float((out[0, t, h].double() - want).norm()) <= room
            assert abs(float(lse[0, t, h]) - float(torch.logsumexp(logits, 0))) <= 1e-4


def test_packed_and_repeated(cuda_device):
    """A long sequence beside short ones: the short ones' bits do not change, nor any from run to run."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(2)
    lengths = [100, 140000, 300, 70000]
    cu = torch.tensor([0, 100, 140100, 140400, 210400], dtype=torch.int32, device="cuda")
    q_len = torch.tensor([0, 100, 300, 600, 601], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 601, 4, 64, generator=gen, device="cuda").to(BF16)
    k, v = (torch.randn(1, sum(lengths), 2, 64, generator=gen, device="cuda").to(BF16) for _ in range(2))
    out = P.full_attention(q, k, v, cu_seqlens=q_len, cu_seqlens_k=cu)
    for _ in range(3):
        assert torch.equal(out, P.full_attention(q, k, v, cu_seqlens=q_len, cu_seqlens_k=cu))
    begin = 0
    for s, n in enumerate(lengths):
        at = slice(int(q_len[s]), int(q_len[s + 1]))
        assert torch.equal(out[:, at], P.full_attention(q[:, at], k[:, begin:begin + n], v[:, begin:begin + n]))
        begin += n


def test_an_item_may_take_long(cuda_device):
    """Waits for a whole item allow for its length: no wait expires, and the status word says so."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(1)
    keys, dim = 1 << 26, 8
    q = torch.randn(1, 1, 1, dim, generator=gen, device="cuda").to(torch.bfloat16)
    k = torch.empty(1, keys, 1, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    v = torch.empty(1, keys, 1, dim, dtype=torch.bfloat16, device="cuda").normal_(0.5, 1.0, generator=gen)
    P.set_status_checks(True)
    try:
        out = P.full_attention(q, k, v)
    finally:
        P.set_status_checks(False)
    logits = (k[0, :, 0].float() @ q[0, 0, 0].float()).double() * dim ** -0.5
    want = torch.softmax(logits, 0) @ v[0, :, 0].double()
    # the output's rounding and the weights', and as much again for sums of 2^26 weights in fp32
    assert float((out[0, 0, 0].double() - want).norm()) <= 3 * 2.0 ** -8 * float(want.norm())
