"""full_attention with values that are not finite, visible and hidden: right elements and a bounded time."""

import math

import pytest
import torch

import dense_reference as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def normal(gen, *shape, dtype=BF16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def cumulative(lengths):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def device_ms(call, repeats=3):
    call()
    times = []
    for _ in range(repeats):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        call()
        end.record()
        end.synchronize()
        times.append(begin.elapsed_time(end))
    return min(times)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("queries,keys,causal", [
    ([700], None, True), ([700], None, False), ([130, 1, 300, 77], None, True), ([130, 1, 300, 77], None, False),
    ([5, 200, 129], [300, 333, 129], True), ([300, 100], [200, 90], True), ([256, 256], [129, 640], True)])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_single_elements(cuda_device, dtype, dim, queries, keys, causal, poison):
    """Single wild elements of V: their columns of the rows that see them, and nothing else."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(sum(queries) + dim)
    lengths = keys if keys is not None else queries
    tokens, total = sum(queries), sum(lengths)
    q, k, v = normal(gen, 1, tokens, 4, dim, dtype=dtype), *(normal(gen, 1, total, 2, dim, dtype=dtype) for _ in range(2))
    places = [(j, h, (j * 7 + h) % dim) for h in range(2) for j in range(h, total, 23)]
    clean = v.clone()
    for j, h, d in places:
        v[0, j, h, d], clean[0, j, h, d] = poison, 0
    out = P.full_attention(q, k, v, cu_seqlens=cumulative(queries), causal=causal,
                           **({} if keys is None else {"cu_seqlens_k": cumulative(keys)}))
    value, bound = R.attention(q, k, clean, causal=causal, queries=queries, keys=keys)
    wild = torch.zeros(tokens, 4, dim, dtype=torch.bool, device="cuda")
    q0 = k0 = 0
    for n, m in zip(queries, lengths):
        for j, h, d in places:
            if k0 <= j < k0 + m:
                first = max(0, (j - k0) - (m - n)) if causal else 0
                wild[q0 + first:q0 + n, 2 * h:2 * h + 2, d] = True
        q0, k0 = q0 + n, k0 + m
    assert torch.isfinite(out[0][~wild]).all()
    assert not torch.isfinite(out[0][wild]).any()
    if math.isinf(poison) and dtype == BF16:    # weights keep fp32's exponents: none is zero
        assert bool((out[0][wild] == poison).all())
    calm = out.masked_fill(wild[None], 0.0)
    R.check("out", calm, value["out"].masked_fill(wild[None], 0.0), bound["out"].masked_fill(wild[None], 0.0))


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_long_sequences(cuda_device, dtype, dim):
    """One NaN among the values of a long prompt: other columns and earlier rows keep their bits."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(3)
    length = 65536
    q, k, v = normal(gen, 1, length, 2, dim, dtype=dtype), *(normal(gen, 1, length, 1, dim, dtype=dtype) for _ in range(2))
    clean = P.full_attention(q, k, v)
    for at in (0, 1000, 40001, length - 1):
        bad = v.clone()
        bad[0, at, 0, 5] = math.nan
        out = P.full_attention(q, k, bad)
        assert torch.equal(out[:, :at], clean[:, :at])
        assert out[:, at:, :, 5].isnan().all()
        # rows past the tiles that hide the key: the other columns' sums are the same
        rest = [d for d in range(dim) if d != 5]
        later = at + 512
        assert torch.equal(out[:, later:, :, rest], clean[:, later:, :, rest])
        near = slice(at, min(later, length))
        assert torch.isfinite(out[:, near][..., rest]).all()
        rows = torch.arange(length, device="cuda")[near]
        hidden = torch.arange(length, device="cuda")[None] > rows[:, None]
        calm = bad.clone()
        calm[0, at, 0, 5] = 0
        for h in range(2):
            found = R.one_head(q[0, near, h].double(), k[0, :, 0].double(), calm[0, :, 0].double(), hidden, dim ** -0.5, dtype)
            R.check("out", out[0, near, h][:, rest], *(x[:, rest] for x in found["out"]))


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_time_and_status_do_not_follow_the_values(cuda_device, dtype, dim):
    """Wild values cost a bounded time per row: no wait of the kernel expires, at any length."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(4)
    length = 32768
    q, k, v = normal(gen, 1, length, 8, dim, dtype=dtype), *(normal(gen, 1, length, 2, dim, dtype=dtype) for _ in range(2))
    usual = device_ms(lambda: P.full_attention(q, k, v))
    first, every, last = v.clone(), torch.full_like(v, math.nan), v.clone()
    first[:, 0, :, 3] = math.nan
    last[:, 100::128] = math.inf
    P.set_status_checks(True)
    try:
        for bad in (first, every, last):
            assert device_ms(lambda: P.full_attention(q, k, bad)) < 40 * usual + 5
    finally:
        P.set_status_checks(False)


def test_queries_without_keys_stay_zero(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k = normal(gen, 1, 300, 4, 128), normal(gen, 1, 90, 2, 128)
    v = torch.full_like(k, math.nan)
    out, lse = P.full_attention(q, k, v, cu_seqlens=cumulative([200, 100]), cu_seqlens_k=cumulative([0, 90]), return_lse=True)
    assert not out[:, :210].any() and torch.isneginf(lse[:, :210]).all()
    assert out[:, 210:].isnan().all() and torch.isfinite(lse[:, 210:]).all()
