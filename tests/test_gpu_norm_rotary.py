"""qk_norm_rotary against its 64-bit form, forward and backward."""

import pytest
import torch

import dense_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-6


def normal(gen, *shape, dtype=BF16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def inputs(gen, batch, tokens, heads, kv_heads, dim, dtype, weight_dtype):
    q, k = normal(gen, batch, tokens, heads, dim, dtype=dtype), normal(gen, batch, tokens, kv_heads, dim, dtype=dtype)
    qw, kw = ((1 + 0.2 * torch.randn(dim, generator=gen, device="cuda")).to(weight_dtype) for _ in range(2))
    frequency = 10000.0 ** (-2 * torch.arange(dim // 2, dtype=torch.float64, device="cuda") / dim)
    frequency[dim // 2 * 3 // 4:] = 0
    return q, k, qw, kw, frequency.float()


def compare(q, k, qw, kw, frequency, positions=None, offset=0, grads=None, eps=EPS):
    import nlogn_pisa_b200 as P

    leaves = [x.detach().requires_grad_(True) for x in (q, k, qw, kw)]
    out = P.qk_norm_rotary(*leaves, frequency, positions=positions, position_offset=offset, eps=eps)
    at = positions if positions is not None else (torch.arange(q.shape[1], device="cuda") + offset)[None]
    angle = at.float()[..., None] * frequency
    gen = torch.Generator(device="cuda").manual_seed(99)
    douts = [normal(gen, *x.shape, dtype=x.dtype) for x in out] if grads is None else grads
    dq, dk, dqw, dkw = torch.autograd.grad(out, leaves, douts)
    for x, w, y, g, dx, dw in ((q, qw, out[0], douts[0], dq, dqw), (k, kw, out[1], douts[1], dk, dkw)):
        found = R.norm_rotary(x, w, angle, eps, g)
        R.check("y", y, *found["y"])
        R.check("dx", dx, *found["dx"])
        R.check("dw", dw, *found["dw"])
        assert y.dtype == x.dtype and dx.dtype == x.dtype and dw.dtype == w.dtype


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (3, 3, 64), (5, 1, 80), (7, 2, 40), (1, 1, 8), (4, 2, 256),
                                                (16, 4, 96), (2, 1, 248)])
@pytest.mark.parametrize("batch,tokens", [(1, 1), (3, 7), (2, 450)])
def test_matches(cuda_device, dtype, heads, kv_heads, dim, batch, tokens):
    gen = torch.Generator(device="cuda").manual_seed(dim + tokens)
    compare(*inputs(gen, batch, tokens, heads, kv_heads, dim, dtype, dtype), offset=1234)
    compare(*inputs(gen, batch, tokens, heads, kv_heads, dim, dtype, F32),
            positions=torch.randint(0, 150000, (batch, tokens), generator=gen, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_tokens(cuda_device, dtype):
    """More tokens than CTAs: weight gradients over many turns."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    compare(*inputs(gen, 3, 4001, 4, 2, 64, dtype, F32))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch,tokens,heads,kv_heads,dim", [(3, 4001, 4, 2, 64), (1, 1000, 32, 8, 128), (7, 333, 5, 1, 80),
                                                             (1, 5, 3, 3, 40)])
def test_nothing_is_written_past_the_rows(cuda_device, dtype, batch, tokens, heads, kv_heads, dim):
    """Both entry points on slices of larger buffers: the rows after the last stay as they were."""
    from nlogn_pisa_b200 import _lib

    gen = torch.Generator(device="cuda").manual_seed(7)
    rows, spare = batch * tokens, 512
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    frequency, weight = torch.rand(dim // 2, device="cuda"), torch.ones(dim, device="cuda")

    def buffers():
        return [torch.full((rows + 2 * spare, h, dim), 7.0, dtype=dtype, device="cuda") for h in (heads, kv_heads)]

    def at(t):
        return t[spare:].data_ptr()

    x, g, y, dx = ([normal(gen, rows + 2 * spare, h, dim, dtype=dtype) for h in (heads, kv_heads)], buffers(), buffers(), buffers())
    common = (weight.data_ptr(), weight.data_ptr(), _lib.F32, frequency.data_ptr(), None, 0, 0, _lib.DTYPES[dtype], batch,
              tokens, heads, kv_heads, dim, EPS)
    views = [v for t, h in zip(x, (heads, kv_heads)) for v in (at(t), tokens * h * dim, h * dim, dim)]
    _lib.check(lib.pisa_qk_norm_rotary(*views, *common, at(y[0]), at(y[1]), stream))
    dw = torch.zeros(2, dim, device="cuda")
    size = lib.pisa_qk_norm_rotary_bwd_workspace_bytes(batch, tokens, dim)
    workspace = torch.full((size + 4096,), 85, dtype=torch.uint8, device="cuda")
    _lib.check(lib.pisa_qk_norm_rotary_bwd(*views, at(g[0]), at(g[1]), *common, at(dx[0]), at(dx[1]), dw[0].data_ptr(),
                                           dw[1].data_ptr(), workspace.data_ptr(), size, stream))
    for t in (*y, *dx):
        assert bool((t[:spare] == 7).all()) and bool((t[spare + rows:] == 7).all())
        assert bool((t[spare:spare + rows] != 7).any(-1).all())
    assert bool((workspace[size:] == 85).all())


def test_layouts(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, qw, kw, frequency = inputs(gen, 2, 50, 4, 2, 64, BF16, BF16)
    fused = normal(gen, 2, 50, 8, 64)
    compare(fused[:, :, :4], fused[:, :, 4:6], qw, kw, frequency)
    compare(q.transpose(1, 2).contiguous().transpose(1, 2), k, qw, kw, frequency,
            positions=torch.arange(50, device="cuda", dtype=torch.int32)[None])
    odd = normal(gen, 2 * 50 * 4 * 64 + 1)[1:].view(2, 50, 4, 64)
    compare(odd, k, qw, kw, frequency, grads=(odd, k.transpose(0, 1).contiguous().transpose(0, 1)))
    compare(q[:1].expand(2, -1, -1, -1), k, qw, kw, frequency)


def test_zero_rows_and_wild_rows_keep_to_themselves(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, qw, kw, frequency = inputs(gen, 1, 9, 4, 2, 128, BF16, BF16)
    q[0, 3] = 0
    compare(q, k, qw, kw, frequency)
    clean = P.qk_norm_rotary(q, k, qw, kw, frequency)
    q[0, 5, 1] = float("nan")
    k[0, 6, 0] = float("inf")
    wild = P.qk_norm_rotary(q, k, qw, kw, frequency)
    keep_q, keep_k = torch.ones(9, 4, dtype=torch.bool, device="cuda"), torch.ones(9, 2, dtype=torch.bool, device="cuda")
    keep_q[5, 1] = keep_k[6, 0] = False
    assert torch.equal(wild[0][0][keep_q], clean[0][0][keep_q]) and torch.equal(wild[1][0][keep_k], clean[1][0][keep_k])
    assert wild[0][0, 5, 1].isnan().all() and wild[1][0, 6, 0].isnan().all()


def test_repeats_bit_for_bit(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(4)
    args = inputs(gen, 2, 3000, 8, 2, 64, BF16, F32)
    leaves = [x.requires_grad_(True) for x in args[:4]]
    douts = normal(gen, 2, 3000, 8, 64), normal(gen, 2, 3000, 2, 64)
    runs = [torch.autograd.grad(P.qk_norm_rotary(*leaves, args[4]), leaves, douts) for _ in range(2)]
    for x, y in zip(*runs):
        assert torch.equal(x, y)


def test_gradient_against_differences(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, qw, kw, frequency = inputs(gen, 1, 20, 3, 2, 64, F32, F32)
    x = [q, k, qw, kw]
    way = [0.1 * normal(gen, *t.shape, dtype=F32) for t in x]
    w = normal(gen, 1, 20, 3, 64, dtype=F32), normal(gen, 1, 20, 2, 64, dtype=F32)
    step = 2.0 ** -5
    angle = torch.arange(20, device="cuda").float()[None, :, None] * frequency

    def loss(sign):
        moved = [(a.double() + sign * step * d.double()).float() for a, d in zip(x, way)]
        got = sum(float((y.double() * g.double()).sum()) for y, g in zip(P.qk_norm_rotary(*moved, frequency, eps=EPS), w))
        exact = [R.norm_rotary(moved[i], moved[2 + i], angle, EPS)["y"] for i in range(2)]
        return (got, sum(float((e[0] * g.double()).sum()) for e, g in zip(exact, w)),
                sum(float((e[1] * g.double().abs()).sum()) for e, g in zip(exact, w)))

    (up, up64, nu), (down, down64, nd) = loss(1), loss(-1)
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(P.qk_norm_rotary(*leaves, frequency, eps=EPS), leaves, w)
    along = sum(float((g.double() * d.double()).sum()) for g, d in zip(grads, way))
    exact = [R.norm_rotary(x[i], x[2 + i], angle, EPS, w[i]) for i in range(2)]
    true = sum(float((exact[i]["dx"][0] * way[i].double()).sum() + (exact[i]["dw"][0] * way[2 + i].double()).sum()) for i in range(2))
    assert abs((up - down) / (2 * step) - along) <= (nu + nd) / (2 * step) + 2 * abs((up64 - down64) / (2 * step) - true) + 1e-3 * abs(true)


def test_refusals(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k, qw, kw, frequency = inputs(gen, 1, 4, 4, 2, 64, BF16, BF16)
    with pytest.raises(ValueError, match="share batch"):
        P.qk_norm_rotary(q, k[:, :3], qw, kw, frequency)
    with pytest.raises(ValueError, match="q_weight"):
        P.qk_norm_rotary(q, k, qw[:32], kw, frequency)
    with pytest.raises(ValueError, match="share a dtype"):
        P.qk_norm_rotary(q, k, qw.float(), kw, frequency)
    with pytest.raises(ValueError, match="frequency"):
        P.qk_norm_rotary(q, k, qw, kw, frequency[:5])
    with pytest.raises(ValueError, match="positions"):
        P.qk_norm_rotary(q, k, qw, kw, frequency, positions=torch.zeros(2, 4, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError, match="multiple of 8"):
        P.qk_norm_rotary(q[..., :12], k[..., :12], qw[:12], kw[:12], frequency[:6])
    with pytest.raises(ValueError, match="support"):
        P.qk_norm_rotary(q.double(), k.double(), qw.double(), kw.double(), frequency)
