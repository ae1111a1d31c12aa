"""swiglu, its 8-bit checkpoints and swiglu_ffn against their 64-bit forms."""

import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def normal(gen, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def kept(x):
    return R.restored(*R.quantized(x.detach().float(), 128), 128)


def compare(gate, up, dout, bits):
    import nlogn_pisa_b200 as P

    leaves = [x.detach().requires_grad_(True) for x in (gate, up)]
    out = P.swiglu(*leaves, checkpoint_bits=bits)
    assert torch.equal(out, P.swiglu(gate, up))
    dgate, dup = torch.autograd.grad(out, leaves, dout)
    want = R.swiglu(gate, up, dout, None if bits is None else (kept(gate), kept(up)))
    R.check("out", out, *want["out"])
    R.check("dgate", dgate, *want["dgate"])
    R.check("dup", dup, *want["dup"])
    assert out.dtype == dgate.dtype == dup.dtype == gate.dtype


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", [1, 8, 127, 128, 129, 136, 1000, 1001, 2816])
@pytest.mark.parametrize("bits", [None, 8])
def test_matches(cuda_device, dtype, width, bits):
    gen = torch.Generator(device="cuda").manual_seed(width)
    for shape in ((1,), (37,), (3, 301)):
        compare(*(normal(gen, *shape, width, dtype=dtype, scale=s) for s in (3.0, 1.0, 1.0)), bits)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bits", [None, 8])
def test_many_groups(cuda_device, dtype, bits):
    """Teams with several groups, the last ones without any; aligned rows and others."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    for rows, width in ((1733, 2816), (1733, 2817), (40003, 40)):
        compare(*(normal(gen, rows, width, dtype=dtype) for _ in range(3)), bits)


@pytest.mark.parametrize("bits", [None, 8])
def test_layouts(cuda_device, bits):
    gen = torch.Generator(device="cuda").manual_seed(1)
    both = normal(gen, 2, 33, 2 * 264)
    dout = normal(gen, 2, 33, 264)
    compare(both[..., :264], both[..., 264:], dout, bits)
    compare(both[..., 1:265], both[..., 264:], dout[:, :1].expand(-1, 33, -1), bits)
    compare(both.transpose(0, 1)[..., :264], both.transpose(0, 1)[..., 264:], dout.transpose(0, 1), bits)
    columns = normal(gen, 2, 264, 33).transpose(1, 2)
    compare(columns, both[..., :264], dout, bits)
    compare(both[0, 0, :264], both[0, 0, 264:], dout[0, 0], bits)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", [8, 130, 1024, 2816, 4097, 16384, 20000])
def test_bytes(cuda_device, dtype, width):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(width)
    gate, up = (normal(gen, 3, 5, width, dtype=dtype) for _ in range(2))
    values, scale = P.swiglu(gate, up, quantize=True)
    assert values.dtype == torch.int8 and values.shape == gate.shape and scale.shape == (3, 5)
    out, bound = R.swiglu(gate, up)["out"]
    bound = bound - R.UNIT[dtype] * out.abs()
    R.check("bytes", values.double() * scale.double()[..., None], out,
            bound + scale.double()[..., None] * (0.5 + 1e-4) + bound.amax(-1, keepdim=True))
    assert bool((values.abs().amax(-1) == 127).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", [1, 16, 100, 256, 1024, 1025, 4096, 16384, 16400, 70001])
def test_quantize_and_checkpoint(cuda_device, dtype, width):
    """Bytes and scales equal the definition's, bit for bit; groups read back."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(width)
    for x in (normal(gen, 2, 3, width, dtype=dtype), normal(gen, 5, width + 3, dtype=dtype)[:, 3:],
              normal(gen, width, 4, dtype=dtype).T):
        values, scale = P.quantize_int8(x)
        want = R.quantized(x.float())
        assert torch.equal(values, want[0]) and torch.equal(scale, want[1])
        values, scale = P.checkpoint_int8(x)
        want = R.quantized(x.float(), 128)
        assert torch.equal(values, want[0]) and torch.equal(scale, want[1])
        back = P.restore_int8(values, scale, dtype)
        assert back.dtype == dtype and torch.equal(back, (R.restored(*want, 128).float()).to(dtype))
        back = P.restore_int8(values.contiguous(), scale, F32)
        assert torch.equal(back, R.restored(*want, 128).float())


def test_ties_small_values_and_wild_values(cuda_device):
    import nlogn_pisa_b200 as P

    x = torch.zeros(8, 128, device="cuda")
    x[0, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -3.5])             # steps of one: ties go to even
    x[1, 0] = 1e-38                                                         # below what a scale follows
    x[2, 0], x[2, 1] = 2.0 ** -99, -(2.0 ** -100)
    x[3, 5] = float("inf")
    x[4, 6] = float("nan")
    x[5, 7] = -float("inf")
    x[6] = torch.finfo(F32).max
    values, scale = P.quantize_int8(x)
    assert values[0, :6].tolist() == [127, 0, 2, 2, 0, -4]
    assert bool((values[1] == 0).all()) and bool((values[3:6] == 0).all()) and bool(scale[3:6].isnan().all())
    want = R.quantized(x)
    assert torch.equal(values, want[0]) and torch.equal(scale.nan_to_num(-1), want[1].nan_to_num(-1))
    assert bool((values[6] == 127).all()) and float(scale[7]) > 0 and bool((values[7] == 0).all())
    kept_values, kept_scale = P.checkpoint_int8(x)
    back = P.restore_int8(kept_values, kept_scale, BF16)
    assert bool(back[3:6].isnan().all()) and bool(back[[0, 1, 2, 7]].isfinite().all())


def test_wild_values_reach_their_groups_gradient_only(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(2)
    gate, up, dout = (normal(gen, 4, 300) for _ in range(3))
    clean = torch.autograd.grad(P.swiglu(*(g := [gate.clone().requires_grad_(True), up.clone().requires_grad_(True)]),
                                         checkpoint_bits=8), g, dout)
    gate[1, 130] = float("nan")
    wild = torch.autograd.grad(P.swiglu(*(g := [gate.requires_grad_(True), up.requires_grad_(True)]), checkpoint_bits=8), g, dout)
    hit = torch.zeros(4, 300, dtype=torch.bool, device="cuda")
    hit[1, 128:256] = True
    for x, y in zip(clean, wild):
        assert torch.equal(x[~hit], y[~hit]) and bool(y[hit].isnan().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(1, 8), (7, 136), (33, 1001)])
def test_nothing_is_written_past_the_rows(cuda_device, dtype, rows, width):
    from nlogn_pisa_b200 import _lib

    gen = torch.Generator(device="cuda").manual_seed(3)
    lib, stream, code = _lib.lib(), torch.cuda.current_stream().cuda_stream, _lib.DTYPES[dtype]
    step, groups, spare = -(-width // 16) * 16, -(-width // 128), 64
    g, u, d = (normal(gen, rows, width, dtype=dtype) for _ in range(3))

    def buffer():
        return torch.full(((rows + 2 * spare) * width,), 7.0, dtype=dtype, device="cuda")

    def at(t):
        return t.data_ptr() + spare * width * t.element_size()

    out, dg, du, again = (buffer() for _ in range(4))
    q = [torch.full((rows + 2, step), 85, dtype=torch.int8, device="cuda") for _ in range(3)]
    scale = [torch.full((rows * groups + 8,), 7.0, device="cuda") for _ in range(3)]
    _lib.check(lib.pisa_swiglu(g.data_ptr(), width, u.data_ptr(), width, code, rows, width, at(out), q[0][1:].data_ptr(),
                               q[1][1:].data_ptr(), step, scale[0].data_ptr(), scale[1].data_ptr(), None, 0, None, stream))
    _lib.check(lib.pisa_swiglu(g.data_ptr(), width, u.data_ptr(), width, code, rows, width, None, None, None, 0, None, None,
                               q[2][1:].data_ptr(), step, scale[2].data_ptr(), stream))
    _lib.check(lib.pisa_swiglu_bwd(d.data_ptr(), width, None, 0, None, 0, q[0][1:].data_ptr(), q[1][1:].data_ptr(), step,
                                   scale[0].data_ptr(), scale[1].data_ptr(), code, rows, width, at(dg), at(du), at(again), stream))
    edge = spare * width
    for t in (out, dg, du, again):
        assert bool((t[:edge] == 7).all()) and bool((t[-edge:] == 7).all()) and bool((t[edge:-edge] != 7).any())
    for t in q:
        assert bool((t[0] == 85).all()) and bool((t[-1] == 85).all()) and bool((t[:, width:] == 85).all())
    assert all(bool((t[rows * groups:] == 7).all()) for t in scale[:2]) and bool((scale[2][rows:] == 7).all())


@pytest.mark.parametrize("bits", [None, 8])
def test_gradient_against_differences(cuda_device, bits):
    """Along every direction of values that 8 bits hold exactly, both forms follow the loss."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(4)
    x = [torch.randint(-127, 128, (6, 256), generator=gen, device="cuda").float() / 32 for _ in range(2)]
    for t in x:
        t[:, ::128] = 127 / 32
    w = normal(gen, 6, 256, dtype=F32)
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(P.swiglu(*leaves, checkpoint_bits=bits), leaves, w)

    def loss(g, u):
        return float((torch.nn.functional.silu(g) * u * w.double()).sum())

    for i in range(2):
        way = torch.randn(x[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        base, found = [t.double() for t in x], []
        for s in (2.0 ** -8, 2.0 ** -9):
            ends = [loss(*[b + (sign * s * way if j == i else 0) for j, b in enumerate(base)]) for sign in (1, -1)]
            found.append((ends[0] - ends[1]) / (2 * s))
        along, size = float((grads[i].double() * way).sum()), float((grads[i].double() * way).abs().sum())
        assert abs(found[1] - along) <= 2 * abs(found[1] - found[0]) + 1e-5 * size
        assert abs(along) > 1e-3 * size


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bias", [True, False])
def test_ffn_keeps_its_activations_in_8_bits(cuda_device, dtype, bias):
    """The forward is the plain layer's; the gradients are those of the kept values."""
    import torch.nn.functional as F

    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(5)
    x = normal(gen, 2, 40, 256, dtype=dtype)
    w = [normal(gen, *s, dtype=dtype, scale=s[1] ** -0.5) for s in ((384, 256), (384, 256), (256, 384))]
    b = [normal(gen, n, dtype=dtype, scale=0.3) for n in (384, 384, 256)] if bias else []
    leaves = [t.requires_grad_(True) for t in (x, *w, *b)]
    y = P.swiglu_ffn(*leaves)
    dy = normal(gen, 2, 40, 256, dtype=dtype)
    bs = b if bias else (None,) * 3
    with torch.no_grad():
        gate, up = F.linear(x, w[0], bs[0]), F.linear(x, w[1], bs[1])
        assert torch.equal(y, F.linear(P.swiglu(gate, up), w[2], bs[2]))
        assert torch.equal(y, P.swiglu_ffn(*leaves))
    grads = torch.autograd.grad(y, leaves, dy)
    # the same in 64 bits from what was kept
    g, u, xk = kept(gate), kept(up), kept(x)
    s = torch.sigmoid(g)
    d = dy.double() @ w[2].double()
    dg, du, out = d * u * s * (1 + g * (1 - s)), d * g * s, g * s * u
    rows = [t.reshape(-1, t.shape[-1]) for t in (dg, du, dy.double(), out, xk)]
    want = [dg @ w[0].double() + du @ w[1].double(), rows[0].T @ rows[4], rows[1].T @ rows[4], rows[2].T @ rows[3]]
    if bias:
        want += [rows[0].sum(0), rows[1].sum(0), rows[2].sum(0)]
    # roundings of dproduct, dgate and dup (or the rebuilt product) and of the result, worst case relative to sums of magnitudes
    unit = R.UNIT[dtype] + 2e-6
    terms = [dg.abs() @ w[0].double().abs() + du.abs() @ w[1].double().abs(), rows[0].abs().T @ rows[4].abs(),
             rows[1].abs().T @ rows[4].abs(), rows[2].abs().T @ rows[3].abs(), rows[0].abs().sum(0), rows[1].abs().sum(0),
             rows[2].abs().sum(0)]
    for got, value, size in zip(grads, want, terms):
        # dgate crosses zero where its two terms cancel: an element's error then exceeds its own share
        R.check("grad", got, value, 8 * unit * (size + size.mean()))


def test_ffn_computes_the_gradients_that_are_asked_for(cuda_device):
    """Any subset of the inputs, with the same bits; under autocast the products' type is its own."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(10)
    shapes = ((3, 5, 96), (160, 96), (160, 96), (96, 160), (160,), (160,), (96,))
    leaves = [normal(gen, *s, dtype=F32, scale=0.2).requires_grad_(True) for s in shapes]
    dy = normal(gen, 3, 5, 96, dtype=F32)
    full = torch.autograd.grad(P.swiglu_ffn(*leaves), leaves, dy)
    for i in range(7):
        some = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        got, = torch.autograd.grad(P.swiglu_ffn(*some), some[i], dy)
        assert torch.equal(got, full[i])
    with torch.autocast("cuda", dtype=BF16):
        y = P.swiglu_ffn(*leaves)
    assert y.dtype == BF16
    half = torch.autograd.grad(y, leaves, dy.to(BF16))
    for x, z in zip(half, full):
        # products of bf16 operands: each of three in a row is off by some 2^-8 of its norm, and a value next
        # to the border of an 8-bit step moves by 1/127 of its group's largest (at most 4.5% of the norm in all)
        assert x.dtype == F32 and float((x - z).norm() / z.norm()) < 0.06


def test_ffn_memory(cuda_device):
    """Between forward and backward the layer holds about a third of the plain layer's activations."""
    import torch.nn.functional as F

    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(6)
    x = normal(gen, 4096, 512).requires_grad_(True)
    w = [normal(gen, *s, scale=0.05).requires_grad_(True) for s in ((1408, 512), (1408, 512), (512, 1408))]

    def held(layer):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = layer(x.clone())
        return torch.cuda.memory_allocated() - before - y.numel() * 2

    plain = held(lambda t: F.linear(F.silu(F.linear(t, w[0])) * F.linear(t, w[1]), w[2]))
    assert held(lambda t: P.swiglu_ffn(t, *w)) < 0.45 * plain


def test_captured_and_replayed(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(7)
    gate, up = (normal(gen, 70, 1000).requires_grad_(True) for _ in range(2))
    dout = normal(gen, 70, 1000)

    def step():
        out = P.swiglu(gate, up, checkpoint_bits=8)
        with torch.no_grad():
            return (out.detach(), *torch.autograd.grad(out, (gate, up), dout), *P.swiglu(gate, up, quantize=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        with torch.no_grad():
            for t in (gate, up, dout):
                t.copy_(normal(gen, 70, 1000))
        graph.replay()
        for x, y in zip(got, step()):
            assert torch.equal(x, y)


def test_refusals(cuda_device):
    import nlogn_pisa_b200 as P
    from torch.autograd import forward_ad

    gen = torch.Generator(device="cuda").manual_seed(8)
    x = normal(gen, 4, 64)
    with pytest.raises(ValueError, match="inference"):
        P.swiglu(x.clone().requires_grad_(True), x, quantize=True)
    with pytest.raises(ValueError, match="32768"):
        P.swiglu(normal(gen, 1, 32776), normal(gen, 1, 32776), quantize=True)
    with pytest.raises(ValueError, match="inference"):
        P.quantize_int8(x.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="support"):
        P.swiglu(x.double(), x.double())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="jvp"):
            P.swiglu(dual, x)
        with pytest.raises(RuntimeError, match="forward"):
            P.swiglu_ffn(dual, *(normal(gen, *s) for s in ((8, 64), (8, 64), (64, 8))))
