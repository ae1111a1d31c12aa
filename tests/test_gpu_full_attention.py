"""full_attention against its 64-bit form, forward and backward."""

import math

import pytest
import torch

import dense_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def normal(gen, *shape, dtype=BF16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def cumulative(lengths, dtype=torch.int32):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=dtype, device="cuda")


def compare(q, k, v, dout, queries=None, keys=None, grad=True, **kw):
    import nlogn_pisa_b200 as P

    call = dict(kw)
    if queries is not None:
        call["cu_seqlens"] = cumulative(queries)
        if keys is not None:
            call["cu_seqlens_k"] = cumulative(keys, torch.int64)
    leaves = [x.detach().requires_grad_(grad) for x in (q, k, v)]
    out, lse = P.full_attention(*leaves, return_lse=True, **call)
    value, bound = R.attention(q, k, v, scale=kw.get("scale"), causal=kw.get("causal", True), queries=queries, keys=keys,
                               offset=kw.get("query_offset"), dout=dout if grad else None)
    R.check("out", out, value["out"], bound["out"])
    R.check("lse", lse, value["lse"], bound["lse"])
    if grad:
        grads = torch.autograd.grad(out, leaves, dout)
        for name, x in zip(("dq", "dk", "dv"), grads):
            R.check(name, x, value[name], bound[name])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,dim_v", [(4, 2, 128, 128), (3, 3, 64, 64), (8, 1, 96, 96), (2, 1, 40, 72),
                                                      (4, 1, 8, 16), (2, 2, 200, 256)])
@pytest.mark.parametrize("tokens,keys", [(1, 1), (1, 130), (64, 64), (127, 127), (129, 300), (257, 257), (520, 520)])
def test_batches(cuda_device, dtype, heads, kv_heads, dim, dim_v, tokens, keys):
    gen = torch.Generator(device="cuda").manual_seed(tokens * 7 + keys + dim)
    q, k, v = (normal(gen, 2, n, h, d, dtype=dtype) for n, h, d in ((tokens, heads, dim), (keys, kv_heads, dim),
                                                                    (keys, kv_heads, dim_v)))
    compare(q, k, v, normal(gen, 2, tokens, heads, dim_v, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("queries,keys", [
    ([1], None), ([1, 1, 1], None), ([128, 128], None), ([127, 1, 129, 0, 256, 3], None), ([0, 5, 0, 0, 300], None),
    ([255, 257, 511], None), ([1, 64, 2], [700, 64, 130]), ([100, 5, 0, 40], [1000, 0, 7, 41]),
    ([300, 10], [200, 3]),           # more queries than keys: the first ones see nothing
    ([400], [129])])
@pytest.mark.parametrize("causal", [True, False])
def test_packed(cuda_device, dtype, dim, queries, keys, causal):
    gen = torch.Generator(device="cuda").manual_seed(sum(queries) + dim)
    tokens, total = sum(queries), sum(keys if keys is not None else queries)
    q, k, v = normal(gen, 1, tokens, 4, dim, dtype=dtype), *(normal(gen, 1, total, 2, dim, dtype=dtype) for _ in range(2))
    compare(q, k, v, normal(gen, 1, tokens, 4, dim, dtype=dtype), queries, keys, causal=causal)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_offset_scale_and_not_causal(cuda_device, dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = normal(gen, 2, 70, 4, 64, dtype=dtype), *(normal(gen, 2, 333, 2, 64, dtype=dtype) for _ in range(2))
    dout = normal(gen, 2, 70, 4, 64, dtype=dtype)
    compare(q, k, v, dout, query_offset=0)
    compare(q, k, v, dout, query_offset=131, scale=0.31)
    compare(q, k, v, dout, causal=False)
    compare(k.repeat(1, 1, 2, 1), q[:, :, :2].contiguous(), q[:, :, 2:].contiguous(), k.repeat(1, 1, 2, 1), causal=False)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", [30.0, 1e-3])
def test_large_and_small_logits(cuda_device, dtype, sizes):
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = normal(gen, 1, 400, 4, 64, dtype=dtype), *(normal(gen, 1, 400, 2, 64, dtype=dtype) for _ in range(2))
    compare((q.float() * sizes).to(dtype), k, v, normal(gen, 1, 400, 4, 64, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale", [1e-4, 1e-33])
def test_small_scales(cuda_device, dtype, scale):
    """Weights near equal; the kernels may divide statistics by the scale."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = normal(gen, 1, 300, 4, 64, dtype=dtype), *(normal(gen, 1, 300, 2, 64, dtype=dtype) for _ in range(2))
    compare(q, k, v, normal(gen, 1, 300, 4, 64, dtype=dtype), [200, 0, 100], [300, 0, 0], scale=scale)


def test_rising_logits(cuda_device):
    """The running maximum grows with every tile of keys."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, v = normal(gen, 1, 900, 2, 128), normal(gen, 1, 900, 2, 128)
    q[..., 0] = 8.0
    k = normal(gen, 1, 900, 2, 128) * 0.1
    k[..., 0] = (torch.arange(900, device="cuda") * 0.25).to(BF16)[None, :, None]
    compare(q, k, v, normal(gen, 1, 900, 2, 128))
    compare(q, k.flip(1).contiguous(), v, normal(gen, 1, 900, 2, 128))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(cuda_device, dtype):
    """Slices of a fused projection, cache views, broadcast heads and unaligned rows."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    fused = normal(gen, 2, 200, 8, 64, dtype=dtype)
    q, k, v = fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:]
    dout = normal(gen, 2, 200, 4, 64, dtype=dtype)
    compare(q, k, v, dout)
    cache = normal(gen, 2, 512, 2, 64, dtype=dtype)
    compare(q, cache[:, :300], cache[:, 100:400], dout)
    by_head = normal(gen, 2, 4, 200, 64, dtype=dtype).transpose(1, 2)
    compare(by_head, k, v, dout.transpose(1, 2).contiguous().transpose(1, 2))
    one = normal(gen, 2, 200, 1, 64, dtype=dtype)
    compare(q, one.expand(-1, -1, 2, -1), one.expand(-1, -1, 2, -1), dout)
    odd = normal(gen, 2 * 200 * 4 * 64 + 1, dtype=dtype)[1:].view(2, 200, 4, 64)
    compare(odd, k, v, odd.clone())
    compare(odd, k, v, odd)


def test_broadcast_keys_get_summed_gradients(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(9)
    q, one = normal(gen, 2, 150, 4, 64, dtype=F32), normal(gen, 1, 150, 1, 64, dtype=F32)
    dout = normal(gen, 2, 150, 4, 64, dtype=F32)
    k, v = (one.clone().requires_grad_(True) for _ in range(2))
    out = P.full_attention(q, k.expand(2, -1, 2, -1), v.expand(2, -1, 2, -1))
    dk, dv = torch.autograd.grad(out, (k, v), dout)
    value, bound = R.attention(q, one.expand(2, -1, 2, -1), one.expand(2, -1, 2, -1), dout=dout)
    for name, x in (("dk", dk), ("dv", dv)):
        R.check(name, x, value[name].sum((0, 2), keepdim=True), 2 * bound[name].sum((0, 2), keepdim=True))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim", [64, 128])
def test_hidden_places_reach_nothing(cuda_device, dtype, poison, dim):
    """Rows outside a query's sequence, and later keys, may hold anything."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(10)
    lengths = [70, 130, 300]
    q, k, v, dout = normal(gen, 1, 500, 4, dim, dtype=dtype), *(normal(gen, 1, 500, 2, dim, dtype=dtype) for _ in range(2)), \
        normal(gen, 1, 500, 4, dim, dtype=dtype)
    value, bound = R.attention(q, k, v, queries=lengths, dout=dout)
    for first, last in ((70, 200), (200, 500), (0, 70)):
        bad = [x.clone() for x in (q, k, v, dout)]
        for x in bad:
            x[:, first:last] = poison
        leaves = [x.requires_grad_(True) for x in bad[:3]]
        out = P.full_attention(*leaves, cu_seqlens=cumulative(lengths))
        grads = torch.autograd.grad(out, leaves, bad[3])
        keep = torch.ones(500, dtype=torch.bool, device="cuda")
        keep[first:last] = False
        for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            R.check(name, x[:, keep], value[name][:, keep], bound[name][:, keep])
    # later keys and values of the same sequence
    for at in (1, 77, 128, 250, 299):
        x, y = k.clone(), v.clone()
        x[:, at:], y[:, at:] = poison, poison
        out = P.full_attention(q[:, :300], x[:, :300], y[:, :300])
        clean, room = R.attention(q[:, :300], k[:, :300], v[:, :300])
        R.check("out", out[:, :at], clean["out"][:, :at], room["out"][:, :at])
        y = v.clone()
        y[:, at:] = poison          # values alone: the weights of the rows before are clean
        out = P.full_attention(q[:, :300], k[:, :300], y[:, :300])
        R.check("out", out[:, :at], clean["out"][:, :at], room["out"][:, :at])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_past_the_last_sequence(cuda_device, dtype):
    """cu_seqlens that end early: the rows after them give zeros everywhere."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(11)
    q, k, v, dout = (normal(gen, 1, 640, 2, 64, dtype=dtype) for _ in range(4))
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out, lse = P.full_attention(*leaves, cu_seqlens=cumulative([100, 133]), return_lse=True)
    grads = torch.autograd.grad(out, leaves, dout)
    value, bound = R.attention(q[:, :233], k[:, :233], v[:, :233], queries=[100, 133], dout=dout[:, :233])
    assert torch.isneginf(lse[:, 233:]).all()
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        R.check(name, x[:, :233], value[name], bound[name])
        assert not x[:, 233:].any(), name


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (BF16, 128), (F16, 64)])
def test_repeats_bit_for_bit_and_follows_streams(cuda_device, dtype, dim):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(12)
    q, k, v, dout = normal(gen, 1, 1500, 4, dim, dtype=dtype), *(normal(gen, 1, 1500, 2, dim, dtype=dtype) for _ in range(2)), \
        normal(gen, 1, 1500, 4, dim, dtype=dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]

    def step():
        out = P.full_attention(*leaves, cu_seqlens=cumulative([700, 800]))
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(first, again):
        assert torch.equal(x, y)


def test_gradient_against_differences(cuda_device):
    """Directional differences of the fp32 forward against its gradient."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(13)
    lengths = [37, 70]
    x = [normal(gen, 1, 107, h, 64, dtype=F32) for h in (4, 2, 2)]
    way = [normal(gen, *t.shape, dtype=F32) * 0.1 for t in x]
    w = normal(gen, 1, 107, 4, 64, dtype=F32)
    step = 2.0 ** -5

    def loss(sign):
        moved = [(a.double() + sign * step * d.double()).float() for a, d in zip(x, way)]
        return float((P.full_attention(*moved, cu_seqlens=cumulative(lengths)).double() * w.double()).sum()), moved

    (up, xu), (down, xd) = loss(1), loss(-1)
    leaves = [t.clone().requires_grad_(True) for t in x]
    out = P.full_attention(*leaves, cu_seqlens=cumulative(lengths))
    grads = torch.autograd.grad(out, leaves, w)
    along = sum(float((g.double() * d.double()).sum()) for g, d in zip(grads, way))
    exact = {s: R.attention(*m, queries=lengths) for s, m in (("up", xu), ("down", xd))}
    noise = sum(float((b["out"] * w.double().abs()).sum()) for _, b in exact.values())
    value, _ = R.attention(*x, queries=lengths, dout=w)
    true = sum(float((value[n] * d.double()).sum()) for n, d in zip(("dq", "dk", "dv"), way))
    truth = (float((exact["up"][0]["out"] * w.double()).sum()) - float((exact["down"][0]["out"] * w.double()).sum())) / (2 * step)
    # difference quotient: the forward's rounding over the step, and the curvature that 64 bits show
    assert abs((up - down) / (2 * step) - along) <= noise / (2 * step) + 2 * abs(truth - true) + 1e-3 * abs(true)


def test_wide_offsets(cuda_device):
    """Element offsets past 2^31 in strided operands."""
    gen = torch.Generator(device="cuda").manual_seed(14)
    rows = 40000
    big = torch.empty(1, rows, 512, 128, dtype=BF16, device="cuda")   # 2.6e9 elements
    k, v = big[:, :, 500:501], big[:, :, 511:512]
    k.copy_(normal(gen, 1, rows, 1, 128))
    v.copy_(normal(gen, 1, rows, 1, 128))
    q = normal(gen, 1, 3, 2, 128)
    compare(q, k, v, normal(gen, 1, 3, 2, 128), grad=False)
    wide = big[:, :, 4:6]
    wide[:, -130:].copy_(normal(gen, 1, 130, 2, 128))
    compare(wide[:, -130:], k[:, -130:], v[:, -130:], normal(gen, 1, 130, 2, 128))


def test_many_short_sequences(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(15)
    lengths = [1 + (i * 37) % 23 for i in range(300)]
    total = sum(lengths)
    q, k, v = normal(gen, 1, total, 2, 64), *(normal(gen, 1, total, 1, 64) for _ in range(2))
    compare(q, k, v, normal(gen, 1, total, 2, 64), lengths)


def test_first_call_of_a_thread(cuda_device):
    """A host thread without any CUDA call before: forward, backward and decode."""
    import threading

    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(16)
    q, k, v, dout = normal(gen, 1, 200, 4, 128), *(normal(gen, 1, 200, 2, 128) for _ in range(2)), normal(gen, 1, 200, 4, 128)
    lengths = torch.tensor([200], dtype=torch.int32, device="cuda")
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = P.full_attention(*leaves)
    want = (out.detach(), P.prefix_attention(q[:, :1], k, v, lengths, prefix_k=k[0], prefix_v=v[0]).clone(),
            *torch.autograd.grad(out, leaves, dout))
    torch.cuda.synchronize()
    calls = [lambda: P.full_attention(q.detach(), k.detach(), v.detach()),
             lambda: P.prefix_attention(q[:, :1], k, v, lengths, prefix_k=k[0], prefix_v=v[0])]
    got = []
    for call in calls:
        worker = threading.Thread(target=lambda: got.append(call()))
        worker.start()
        worker.join()
    assert len(got) == 2
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(cuda_device):
    import nlogn_pisa_b200 as P

    q, k = torch.zeros(1, 8, 4, 64, dtype=BF16, device="cuda"), torch.zeros(1, 8, 2, 64, dtype=BF16, device="cuda")
    cu = cumulative([8])
    with pytest.raises(ValueError, match="dtype"):
        P.full_attention(q, k.float(), k.float())
    with pytest.raises(ValueError, match="multiple of 8"):
        P.full_attention(q[..., :20], k[..., :20], k)
    with pytest.raises(ValueError, match="at most 256"):
        P.full_attention(*(torch.zeros(1, 8, 2, 264, dtype=BF16, device="cuda") for _ in range(3)))
    with pytest.raises(ValueError, match="positions"):
        P.full_attention(q, k[:, :4], k[:, :4])
    with pytest.raises(ValueError, match="positions"):
        P.full_attention(q[:, :2], k, k, query_offset=7)
    with pytest.raises(ValueError, match="scale"):
        P.full_attention(q, k, k, scale=0.0)
    with pytest.raises(ValueError, match="scale"):
        P.full_attention(q, k, k, scale=math.inf)
    with pytest.raises(ValueError, match="batch size one"):
        P.full_attention(q.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), cu_seqlens=cu)
    with pytest.raises(ValueError, match="cu_seqlens"):
        P.full_attention(q, k, k, cu_seqlens_k=cu)
    with pytest.raises(ValueError, match="integer tensor"):
        P.full_attention(q, k, k, cu_seqlens=cu.float())
    with pytest.raises(ValueError, match="number of sequences"):
        P.full_attention(q, k, k, cu_seqlens=cu, cu_seqlens_k=cumulative([4, 4]))
    with pytest.raises(ValueError, match="rise"):
        P.full_attention(q, k, k, cu_seqlens=torch.tensor([0, 5]))
    with pytest.raises(ValueError, match="floating"):
        P.full_attention(q.int(), k.int(), k.int())
    with pytest.raises(ValueError, match="support"):
        P.full_attention(q.double(), k.double(), k.double())
