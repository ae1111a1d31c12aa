"""prefix_attention over very long prefixes and caches: sums that keep their bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TRUNCATION = 2.0 ** -13     # of a sum over 65536 keys in a truncating fp32 accumulator


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix,capacity,batch,heads,kv_heads,dim", [
    (1 << 20, 64, 2048, 4, 1, 64), (1 << 20, 64, 16, 4, 1, 64), (200001, 300, 600, 8, 2, 128), (70000, 4096, 64, 8, 8, 64),
    (1, 1 << 20, 2, 4, 1, 64), (262144, 262144, 3, 4, 2, 128), (300000, 64, 300, 64, 8, 128)])
def test_like_weights_of_many_keys(cuda_device, dtype, prefix, capacity, batch, heads, kv_heads, dim):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(prefix + batch)

    def normal(*shape, size=1.0, mean=0.0):
        return torch.empty(shape, device="cuda").normal_(mean, size, generator=gen).to(dtype)

    q, k, v = normal(batch, 1, heads, dim, size=0.1), normal(batch, capacity, kv_heads, dim), normal(batch, capacity, kv_heads, dim, mean=0.5)
    pk, pv = normal(prefix, kv_heads, dim), normal(prefix, kv_heads, dim, mean=0.5)
    lengths = (torch.arange(batch, device="cuda") * 7919) % capacity + 1
    out = P.prefix_attention(q, k, v, lengths, prefix_k=pk, prefix_v=pv)
    for b in (0, batch // 2, batch - 1):
        n = int(lengths[b])
        for h in (0, heads - 1):
            g = h * kv_heads // heads
            keys, values = torch.cat((pk[:, g], k[b, :n, g])).double(), torch.cat((pv[:, g], v[b, :n, g])).double()
            weights = torch.softmax(keys @ q[b, 0, h].double() * dim ** -0.5, 0)
            want = weights @ values
            # rounding of the output, truncation on the way, and at random the rounding of the weights
            room = (UNIT[dtype] + TRUNCATION) * float(want.norm())
            room += 4 * UNIT[dtype] * float((weights.square() @ values.square()).sum().sqrt())
            assert float((out[b, 0, h].double() - want).norm()) <= room
