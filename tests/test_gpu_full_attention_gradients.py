"""Gradients of full_attention over the types' ranges, by the norm of their error.

The element bounds of dense_reference allow each of many roundings its worst
case; here the error's norm is held to what random roundings of the same size
give, so a gradient that lost its bits (or is zero) fails.
"""

import pytest
import torch

import dense_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def normal(gen, *shape, dtype=BF16, size=1.0):
    return (size * torch.randn(shape, generator=gen, device="cuda")).to(dtype)


def cumulative(lengths):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def room(value, dtype):
    """Norm of the error that a result may have: the rounding of the result
    itself, once more the size of that for each of its two 16-bit operands, and
    sums in fp32 (a random walk of a few hundred roundings)."""
    once = float((value.to(dtype).double() - value).norm())
    unit = 64 * R.EPS if dtype == F32 else R.UNIT[dtype]
    return 2 * once + unit * float(value.norm())


def compare(q, k, v, dout, lengths, scale=None, names=("dq", "dk", "dv")):
    import nlogn_pisa_b200 as P

    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = P.full_attention(*leaves, cu_seqlens=cumulative(lengths), scale=scale)
    grads = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout)))
    value, _ = R.attention(q, k, v, queries=lengths, scale=scale, dout=dout)
    begin = 0
    for n in lengths:       # sequence by sequence: one may be far smaller than another
        for name in names:
            got, want = (x[0, begin:begin + n].double() for x in (grads[name], value[name]))
            assert torch.isfinite(want.to(q.dtype)).all() and float(want.to(q.dtype).abs().max()) > 0
            off = float((got - want).norm())
            assert off <= room(want, q.dtype), (name, n, off / float(want.norm()), room(want, q.dtype) / float(want.norm()))
        begin += n


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (4, 2, 128), (4, 1, 80), (2, 1, 160)])
@pytest.mark.parametrize("size,v_size", [(1.0, 1.0), (1e-2, 1.0), (1e-3, 1.0), (1e-4, 1.0), (1e-2, 1e-2), (300.0, 20.0), (0.01, 1000.0)])
def test_sizes(cuda_device, dtype, heads, kv_heads, dim, size, v_size):
    """dout of a mean over many tokens, of a scaled loss, and values of other sizes."""
    gen = torch.Generator(device="cuda").manual_seed(dim)
    lengths = [1100, 333]
    q, k = normal(gen, 1, 1433, heads, dim, dtype=dtype), normal(gen, 1, 1433, kv_heads, dim, dtype=dtype)
    v, dout = normal(gen, 1, 1433, kv_heads, dim, dtype=dtype, size=v_size), normal(gen, 1, 1433, heads, dim, dtype=dtype, size=size)
    compare(q, k, v, dout, lengths)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
def test_sequences_of_different_sizes(cuda_device, dtype, dim):
    """A packed sequence whose gradient is 10^5 times another's takes no bits from it; nor does another head's."""
    gen = torch.Generator(device="cuda").manual_seed(dim + 1)
    lengths = [700, 500]
    q, k, v, dout = normal(gen, 1, 1200, 4, dim, dtype=dtype), *(normal(gen, 1, 1200, 2, dim, dtype=dtype) for _ in range(2)), \
        normal(gen, 1, 1200, 4, dim, dtype=dtype)
    loud = dout.clone()
    loud[:, :700] *= 100
    loud[:, 700:] *= 1e-3
    compare(q, k, v, loud, lengths)
    import nlogn_pisa_b200 as P

    def grads(g):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        return torch.autograd.grad(P.full_attention(*leaves, cu_seqlens=cumulative(lengths)), leaves, g)

    quiet = dout.clone()
    quiet[:, 700:] *= 1e-3
    for x, y in zip(grads(loud), grads(quiet)):
        assert torch.equal(x[:, 700:], y[:, 700:])
    tall = dout.clone()
    tall[:, :, 2:] *= 100        # the query heads of the second KV head
    for (x, y), n in zip(zip(grads(tall), grads(dout)), (2, 1, 1)):
        assert torch.equal(x[:, :, :n], y[:, :, :n])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_small_weights(cuda_device, dtype):
    """Weights near 1 / keys over many keys: dv keeps their bits."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(21)
    keys, rows = 262144, 128
    q, k = normal(gen, 1, rows, 1, 64, dtype=dtype, size=0.3), normal(gen, 1, keys, 1, 64, dtype=dtype)
    v, dout = normal(gen, 1, keys, 1, 64, dtype=dtype), normal(gen, 1, rows, 1, 64, dtype=dtype, size=100.0)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    dv = torch.autograd.grad(P.full_attention(*leaves, causal=False), leaves, dout)[2]
    weights = torch.softmax(q[0, :, 0].detach().double() @ k[0, :, 0].detach().double().T / 8, -1)
    want = weights.T @ dout[0, :, 0].double()
    assert float((dv[0, :, 0].double() - want).norm()) <= room(want, dtype)


@pytest.mark.parametrize("dtype,scale,size", [(F32, 1e-4, 1.0), (F32, 1e-33, 1.0), (BF16, 1e-4, 1.0), (BF16, 1e-33, 1.0),
                                              (F16, 1e-4, 1.0), (F16, 1e-4, 100.0), (F16, 1e-6, 1000.0), (F32, 3.0, 1.0),
                                              (BF16, 3.0, 1.0), (F16, 3.0, 1.0)])
@pytest.mark.parametrize("dim", [64, 128])
def test_scales(cuda_device, dtype, scale, size, dim):
    gen = torch.Generator(device="cuda").manual_seed(dim + 2)
    q, k, v = normal(gen, 1, 520, 4, dim, dtype=dtype, size=0.2 if scale > 1 else 1.0), *(normal(gen, 1, 520, 2, dim, dtype=dtype) for _ in range(2))
    compare(q, k, v, normal(gen, 1, 520, 4, dim, dtype=dtype, size=size), [300, 220], scale=scale)


def test_against_differences(cuda_device):
    """Differences of the fp32 forward along each operand's own gradient: zero, flipped or missing ones fail."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(13)
    lengths = [37, 70]
    x = {n: normal(gen, 1, 107, h, 64, dtype=F32) for n, h in (("q", 4), ("k", 2), ("v", 2))}
    w = normal(gen, 1, 107, 4, 64, dtype=F32)
    leaves = [t.clone().requires_grad_(True) for t in x.values()]
    grads = torch.autograd.grad(P.full_attention(*leaves, cu_seqlens=cumulative(lengths)), leaves, w)
    value, _ = R.attention(*x.values(), queries=lengths, dout=w)
    step = 2.0 ** -4
    for name, grad in zip(x, grads):
        way = value["d" + name] / value["d" + name].abs().max()
        ends = [{**x, name: (x[name].double() + sign * step * way).float()} for sign in (1, -1)]
        moved = (ends[0][name].double() - ends[1][name].double())        # what the rounded ends are apart
        got = [float((P.full_attention(*e.values(), cu_seqlens=cumulative(lengths)).double() * w.double()).sum()) for e in ends]
        exact = [float((R.attention(*e.values(), queries=lengths)[0]["out"] * w.double()).sum()) for e in ends]
        along = float((grad.double() * moved).sum())
        true = float((value["d" + name] * moved).sum())
        # rounding of the two forwards (sixteen units per output, random signs), and the curvature that 64 bits show
        slack = 2 * 16 * R.EPS * float(w.norm()) + abs(exact[0] - exact[1] - true)
        assert slack <= 0.1 * abs(true)
        assert abs(got[0] - got[1] - along) <= slack + 64 * R.EPS * abs(true)
        assert abs(along - true) <= 64 * R.EPS * abs(true)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("keys,rows,dim", [(8192, 200, 64), (16384, 128, 128), (65536, 300, 64), (65536, 128, 128), (262144, 128, 64)])
def test_cancelling_sums_over_many_keys(cuda_device, dtype, keys, rows, dim):
    """dq of near-equal weights and k, v with a mean: an output that is off by e moves dq by e times delta and the mean key."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(keys + dim)
    q = normal(gen, 1, rows, 2, dim, dtype=dtype, size=0.1)
    k, v = ((0.5 + torch.randn(1, keys, 1, dim, generator=gen, device="cuda")).to(dtype) for _ in range(2))
    dout = normal(gen, 1, rows, 2, dim, dtype=dtype, size=100.0)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    dq = torch.autograd.grad(P.full_attention(*leaves, causal=False), leaves, dout)[0]
    kd, vd, scale = k[0, :, 0].detach().double(), v[0, :, 0].detach().double(), dim ** -0.5
    for h in range(2):
        p = torch.softmax(q[0, :, h].detach().double() @ kd.T * scale, -1)
        d = dout[0, :, h].double()
        out = p @ vd
        delta = (d * out).sum(-1, keepdim=True)
        want = scale * (p * (d @ vd.T - delta)) @ kd
        # outputs short by 2^-16 of themselves (sums of 8192 keys in a truncating accumulator of 24 bits)
        off = 2.0 ** -16 * (2 * delta.abs() + (d * out).norm(dim=-1, keepdim=True))
        slack = float((scale * off * (p @ kd).abs()).norm())
        assert float((dq[0, :, h].double() - want).norm()) <= room(want, dtype) + slack
