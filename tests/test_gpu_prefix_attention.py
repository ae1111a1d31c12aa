"""prefix_attention against its 64-bit form."""

import pytest
import torch

import dense_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def normal(gen, *shape, dtype=BF16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def compare(q, k, v, lengths, pk=None, pv=None, scale=None, index=torch.int32):
    import nlogn_pisa_b200 as P

    out, lse = P.prefix_attention(q, k, v, torch.tensor(lengths, dtype=index, device="cuda"), prefix_k=pk, prefix_v=pv,
                                  scale=scale, return_lse=True)
    scale = k.shape[-1] ** -0.5 if scale is None else scale
    batch, new, heads, _ = q.shape
    group = heads // k.shape[2]
    for b, n in enumerate(lengths):
        n = max(0, min(n, k.shape[1]))
        keys, values = k[b, :n].double(), v[b, :n].double()
        shared = 0
        if pk is not None:
            shared = pk.shape[0]
            keys, values = torch.cat((pk.double(), keys)), torch.cat((pv.double(), values))
        cols = torch.arange(shared + n, device="cuda")
        hidden = cols[None] > shared + n - new + torch.arange(new, device="cuda")[:, None]
        hidden &= cols[None] >= shared
        for h in range(heads):
            found = R.one_head(q[b, :, h].double(), keys[:, h // group], values[:, h // group], hidden, scale, q.dtype)
            R.check("out", out[b, :, h], *found["out"])
            R.check("lse", lse[b, :, h], *found["lse"])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,dim_v", [(8, 2, 128, 128), (4, 4, 64, 64), (16, 1, 64, 64), (6, 2, 80, 80),
                                                      (5, 1, 40, 96), (24, 1, 128, 64), (4, 2, 256, 256)])
@pytest.mark.parametrize("new", [1, 3])
def test_own_caches(cuda_device, dtype, heads, kv_heads, dim, dim_v, new):
    gen = torch.Generator(device="cuda").manual_seed(dim + new)
    lengths = [new, 0, 64, 65, 127, 700, 1000, 2]
    q = normal(gen, 8, new, heads, dim, dtype=dtype)
    k, v = normal(gen, 8, 1000, kv_heads, dim, dtype=dtype), normal(gen, 8, 1000, kv_heads, dim_v, dtype=dtype)
    compare(q, k, v, lengths)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (16, 1, 96), (3, 1, 80)])
@pytest.mark.parametrize("batch,new,prefix", [(1, 1, 1), (2, 1, 63), (5, 1, 64), (7, 2, 129), (40, 1, 1000), (33, 5, 515),
                                              (3, 1, 5000)])
def test_shared_prefix(cuda_device, dtype, heads, kv_heads, dim, batch, new, prefix):
    gen = torch.Generator(device="cuda").manual_seed(batch * 3 + prefix)
    lengths = [(b * 53) % 300 for b in range(batch)]
    q, k, v = normal(gen, batch, new, heads, dim, dtype=dtype), *(normal(gen, batch, 300, kv_heads, dim, dtype=dtype) for _ in range(2))
    pk, pv = (normal(gen, prefix, kv_heads, dim, dtype=dtype) for _ in range(2))
    compare(q, k, v, lengths, pk, pv)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 64), (8, 1, 128), (160, 160, 64)])
@pytest.mark.parametrize("prefix,capacity,lengths", [(129, 3000, [3000] * 17), (6000, 300, [0] * 20), (6000, 300, [1] * 300),
                                                     (2500, 2500, [2500, 0, 1] * 8)])
def test_prefix_and_caches_share_the_device(cuda_device, heads, kv_heads, dim, prefix, capacity, lengths):
    """From all the work in the caches to all of it in the prefix, whose key ranges follow from the lengths."""
    gen = torch.Generator(device="cuda").manual_seed(prefix + heads)
    if heads * len(lengths) > 3000:
        lengths = lengths[:18]
    batch = len(lengths)
    q, k, v = normal(gen, batch, 1, heads, dim), *(normal(gen, batch, capacity, kv_heads, dim) for _ in range(2))
    compare(q, k, v, lengths, *(normal(gen, prefix, kv_heads, dim) for _ in range(2)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lengths_are_clamped_and_empty_rows_are_zero(cuda_device, dtype):
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = normal(gen, 4, 2, 4, 64, dtype=dtype), *(normal(gen, 4, 90, 2, 64, dtype=dtype) for _ in range(2))
    compare(q, k, v, [-5, 1, 1 << 20, 0], index=torch.int64)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_keys_past_the_length_reach_nothing(cuda_device, dtype, poison):
    """Unwritten cache rows may hold anything, as may a later token of the same step."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(4)
    lengths = [1, 63, 64, 130, 299]
    q, k, v = normal(gen, 5, 1, 4, 128, dtype=dtype), *(normal(gen, 5, 300, 2, 128, dtype=dtype) for _ in range(2))
    pk, pv = (normal(gen, 77, 2, 128, dtype=dtype) for _ in range(2))
    n = torch.tensor(lengths, device="cuda")
    clean = P.prefix_attention(q, k, v, n, prefix_k=pk, prefix_v=pv)
    for b, m in enumerate(lengths):
        k[b, m:], v[b, m:] = poison, poison
    assert torch.equal(clean, P.prefix_attention(q, k, v, n, prefix_k=pk, prefix_v=pv))
    compare(q, k, v, lengths, pk, pv)
    two = normal(gen, 5, 2, 4, 128, dtype=dtype)
    for b, m in enumerate(lengths):
        v[b, m - 1] = poison            # the newest key: only the last token sees it
    out = P.prefix_attention(two, k, v, n, prefix_k=pk, prefix_v=pv)
    assert torch.isfinite(out[:, 0]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(cuda_device, dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)
    cache = normal(gen, 3, 400, 4, 64, dtype=dtype)
    q = normal(gen, 3, 2, 8, 64, dtype=dtype)
    compare(q.transpose(1, 2).contiguous().transpose(1, 2), cache[:, 10:300, :2], cache[:, 10:300, 2:], [5, 290, 100])
    head_major = normal(gen, 2, 500, 64, dtype=dtype).transpose(0, 1)
    compare(q, cache[:, :100, :2], cache[:, :100, 2:], [5, 100, 64], head_major, head_major[:, :, :])
    one = normal(gen, 3, 100, 1, 64, dtype=dtype)
    compare(q, one.expand(-1, -1, 2, -1), one.expand(-1, -1, 2, -1), [7, 100, 1])
    odd = normal(gen, 3 * 2 * 8 * 64 + 1, dtype=dtype)[1:].view(3, 2, 8, 64)
    compare(odd, cache[:, :, :2], cache[:, :, 2:], [400, 3, 60])


def test_wide_offsets(cuda_device):
    """Element offsets past 2^31 in a cache's rows."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    big = torch.empty(1, 300000, 64, 128, dtype=BF16, device="cuda")   # 2.5e9 elements
    k, v = big[:, :, 3:4], big[:, :, 60:61]
    k.copy_(normal(gen, 1, 300000, 1, 128))
    v.copy_(normal(gen, 1, 300000, 1, 128))
    q = normal(gen, 1, 1, 4, 128)
    compare(q, k, v, [300000])
    compare(q, k[:, :50], v[:, :50], [50], k[0], v[0])


def test_repeats_bit_for_bit_on_another_stream(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = normal(gen, 9, 1, 8, 128), *(normal(gen, 9, 900, 2, 128) for _ in range(2))
    pk, pv = (normal(gen, 3000, 2, 128) for _ in range(2))
    n = torch.arange(9, device="cuda") * 100 + 1
    first = P.prefix_attention(q, k, v, n, prefix_k=pk, prefix_v=pv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = P.prefix_attention(q, k, v, n, prefix_k=pk, prefix_v=pv)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)


def test_refusals(cuda_device):
    import nlogn_pisa_b200 as P

    q, k = torch.zeros(2, 1, 4, 64, dtype=BF16, device="cuda"), torch.zeros(2, 8, 2, 64, dtype=BF16, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="lengths"):
        P.prefix_attention(q, k, k, n[:1])
    with pytest.raises(ValueError, match="lengths"):
        P.prefix_attention(q, k, k, n.float())
    with pytest.raises(ValueError, match="lengths"):
        P.prefix_attention(q, k, k, n.cpu())
    with pytest.raises(ValueError, match="together"):
        P.prefix_attention(q, k, k, n, prefix_k=k[0])
    with pytest.raises(ValueError, match="prefix_k"):
        P.prefix_attention(q, k, k, n, prefix_k=k[0].float(), prefix_v=k[0].float())
    with pytest.raises(ValueError, match="prefix_k"):
        P.prefix_attention(q, k, k, n, prefix_k=k, prefix_v=k)
    with pytest.raises(ValueError, match="scale"):
        P.prefix_attention(q, k, k, n, scale=-1.0)
    with pytest.raises(ValueError, match="multiple of 8"):
        P.prefix_attention(q[..., :12], k[..., :12], k, n)
