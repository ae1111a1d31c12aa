"""residual_norm against its 64-bit form, forward and backward."""

import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-6


def normal(gen, *shape, dtype=BF16, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale + mean).to(dtype)


def inputs(gen, batch, tokens, width, dtype, gate="none", post=True, param=F32):
    x, branch = normal(gen, batch, tokens, width, dtype=dtype, scale=2.0), normal(gen, batch, tokens, width, dtype=dtype)
    weight, post_weight = (normal(gen, width, dtype=param, scale=0.2, mean=1.0) for _ in range(2))
    shape = {"none": None, "width": (width,), "sequence": (batch, 1, width), "token": (batch, tokens, width)}[gate]
    g = None if shape is None else normal(gen, *shape, dtype=dtype if gate == "token" else param)
    return {"x": x, "branch": branch, "weight": weight, "post_weight": post_weight if post else None, "gate": g}


def call(t, a=1.0, b=1.0, **kw):
    import nlogn_pisa_b200 as P

    return P.residual_norm(t["x"], t["branch"], t["weight"], post_weight=t["post_weight"], gate=t["gate"], residual_scale=a,
                           branch_scale=b, eps=EPS, **kw)


def compare(t, a=1.0, b=1.0, grads=None, seed=99):
    t = {k: None if v is None else v.detach().requires_grad_(True) for k, v in t.items()}
    h, n = call(t, a, b)
    with torch.no_grad():   # without a graph: the same values
        again = call(t, a, b)
    assert torch.equal(again[0], h) and torch.equal(again[1], n)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dh, dn = (normal(gen, *h.shape, dtype=h.dtype) for _ in range(2)) if grads is None else grads
    names = [k for k, v in t.items() if v is not None]
    got = dict(zip(names, torch.autograd.grad((h, n), [t[k] for k in names], (dh, dn))))
    want = R.residual_norm(t["x"], t["branch"], t["weight"], t["post_weight"], t["gate"], a, b, EPS, dh, dn)
    R.check("h", h, *want["h"])
    R.check("n", n, *want["n"])
    for k in names:
        assert got[k].dtype == t[k].dtype
        R.check("d" + k, got[k], *want["d" + k])


WIDTHS = [1, 7, 8, 64, 72, 128, 136, 255, 256, 257, 264, 512, 1000, 1024, 1025, 2048, 2056, 4096, 4097, 8192, 8200, 16383, 16384]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(cuda_device, dtype, width):
    gen = torch.Generator(device="cuda").manual_seed(width)
    compare(inputs(gen, 2, 5, width, dtype, "width", True, F32), 0.75, 1.5)
    compare(inputs(gen, 3, 3, width, dtype, "token", False, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gate", ["none", "width", "sequence", "token"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("batch,tokens", [(1, 1), (3, 1), (1, 7), (5, 130)])
def test_gates(cuda_device, dtype, gate, post, batch, tokens):
    gen = torch.Generator(device="cuda").manual_seed(batch + tokens)
    for width, param in ((320, dtype), (1111, F32)):
        compare(inputs(gen, batch, tokens, width, dtype, gate, post, param), 1.0, 0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [40, 61, 104, 200, 520, 1536, 2560, 4800])
@pytest.mark.parametrize("gate", ["width", "sequence", "token"])
def test_many_rows(cuda_device, dtype, width, gate):
    """More rows than teams: parameter gradients over many turns, shares of unequal teams."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    compare(inputs(gen, 3, 1501, width, dtype, gate))


def test_many_short_sequences(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(2)
    compare(inputs(gen, 3001, 2, 72, BF16, "sequence"))
    compare(inputs(gen, 3001, 3, 24, BF16, "sequence", True, BF16))
    compare(inputs(gen, 7, 5, 24, F32, "sequence", False))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_without_branch(cuda_device, dtype):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(3)
    for width in (96, 1025):
        x, w = normal(gen, 4, 9, width, dtype=dtype).requires_grad_(True), normal(gen, width, dtype=F32).requires_grad_(True)
        dn, dh = normal(gen, 4, 9, width, dtype=dtype), normal(gen, 4, 9, width, dtype=dtype)
        h, n = P.residual_norm(x, None, w, eps=EPS)
        assert h is x
        want = R.residual_norm(x, None, w, eps=EPS, dn=dn)
        R.check("n", n, *want["n"])
        dx, dw = torch.autograd.grad(n, (x, w), dn)
        R.check("dx", dx, *want["dx"])
        R.check("dw", dw, *want["dweight"])
        # both outputs are used: autograd adds their parts
        h, n = P.residual_norm(x, None, w, eps=EPS)
        both, = torch.autograd.grad((h, n), x, (dh, dn))
        assert torch.equal(both, dx + dh)


def test_one_output_used(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(4)
    t = inputs(gen, 2, 33, 200, BF16, "width")
    zero = torch.zeros_like(t["x"])
    d = normal(gen, *zero.shape)
    leaves = [v.requires_grad_(True) for v in t.values()]
    h, n = call(t)
    for which, full in ((n, (zero, d)), (h, (d, zero))):
        alone = torch.autograd.grad(which, leaves, d, retain_graph=True, allow_unused=True)
        both = torch.autograd.grad((h, n), leaves, full, retain_graph=True)
        for x, y in zip(alone, both):
            assert torch.equal(x, y)


def test_layouts(cuda_device):
    """Strided, unaligned, broadcast and transposed tensors."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    wide = normal(gen, 2, 21, 3 * 128)
    t = inputs(gen, 2, 21, 128, BF16, "token")
    compare({**t, "x": wide[..., :128], "branch": wide[..., 128:256], "gate": wide[..., 256:]})
    odd = normal(gen, 2 * 21 * 128 + 1)[1:].view(2, 21, 128)
    compare({**t, "branch": odd}, grads=(odd, odd.transpose(0, 1).contiguous().transpose(0, 1)))
    compare({**t, "x": t["x"].transpose(0, 1).contiguous().transpose(0, 1), "gate": t["gate"][:1].expand(2, -1, -1)})
    compare({**t, "x": normal(gen, 2, 128, 21).transpose(1, 2), "branch": t["branch"][:, :1].expand(-1, 21, -1)})
    compare({**t, "gate": normal(gen, 257)[1::2]})
    compare({**t, "gate": normal(gen, 1, 1, 128), "weight": normal(gen, 129, dtype=F32)[1:]})
    compare({**t, "gate": normal(gen, 2, 3, 128)[:, 1:2]})
    single = {k: v[:, :1] if v is not None and v.dim() == 3 else v for k, v in t.items()}
    compare({**single, "gate": normal(gen, 2, 1, 128, dtype=F32)})     # one token, fp32: one gate per sequence


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(1, 64), (37, 72), (700, 1000), (5, 1001), (3, 8200), (5000, 48), (3000, 57), (900, 6001)])
def test_nothing_is_written_past_the_rows(cuda_device, dtype, rows, width):
    """Both entry points on slices of larger buffers: what lies around the outputs stays as it was."""
    from nlogn_pisa_b200 import _lib

    gen = torch.Generator(device="cuda").manual_seed(6)
    spare = 64
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    code, step = _lib.DTYPES[dtype], -(-width // 16) * 16

    def buffer():
        return torch.full(((rows + 2 * spare) * width,), 7.0, dtype=dtype, device="cuda")

    def at(t):
        return t.data_ptr() + spare * width * t.element_size()

    x, y, dh, dn = (normal(gen, (rows + 2 * spare) * width, dtype=dtype) for _ in range(4))
    w = normal(gen, width, dtype=F32)
    h, n, dx, dy, dg = (buffer() for _ in range(5))
    stats = torch.full((rows + 8, 2), 7.0, device="cuda")
    q = torch.full((rows + 2, step), 85, dtype=torch.int8, device="cuda")
    scale = torch.full((rows + 8,), 7.0, device="cuda")
    gate = normal(gen, (rows + 2 * spare) * width, dtype=dtype)
    common = (at(gate), width, 0, code, w.data_ptr(), _lib.F32, w.data_ptr(), _lib.F32, code, rows, width)
    _lib.check(lib.pisa_residual_norm(at(x), width, at(y), width, *common, 1.0, 1.0, EPS, at(h), at(n), None, 0, None,
                                      stats.data_ptr(), stream))
    h2 = buffer()
    _lib.check(lib.pisa_residual_norm(at(x), width, at(y), width, *common, 1.0, 1.0, EPS, at(h2), None, q[1:].data_ptr(), step,
                                      scale.data_ptr(), None, stream))
    assert torch.equal(h, h2)
    size = lib.pisa_residual_norm_bwd_workspace_bytes(rows, width, 0)
    workspace = torch.full((size + 4096,), 85, dtype=torch.uint8, device="cuda")
    dw = torch.full((2, width + 32), 7.0, device="cuda")
    _lib.check(lib.pisa_residual_norm_bwd(at(dh), at(dn), at(x), width, at(y), width, *common, 1.0, 1.0, stats.data_ptr(), at(dx),
                                          at(dy), at(dg), dw[0].data_ptr(), dw[1].data_ptr(), workspace.data_ptr(), size, stream))
    edge = spare * width
    for t in (h, n, dx, dy, dg):
        assert bool((t[:edge] == 7).all()) and bool((t[-edge:] == 7).all())
        assert bool((t[edge:-edge].view(rows, width) != 7).any(-1).all())
    assert bool((stats[rows:] == 7).all()) and bool((scale[rows:] == 7).all()) and bool((dw[:, width:] == 7).all())
    assert bool((q[0] == 85).all()) and bool((q[-1] == 85).all()) and bool((q[:, width:] == 85).all())
    assert bool((workspace[size:] == 85).all())


def test_zero_rows_and_wild_rows_keep_to_themselves(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(7)
    for width in (64, 333, 2048):
        t = inputs(gen, 1, 9, width, BF16, "token")
        t["x"][0, 3] = t["branch"][0, 3] = 0
        compare(t)
        clean = call(t)
        bytes_clean = call(t, quantize=True)
        t["branch"][0, 5, 1] = float("nan")
        t["x"][0, 6, width - 1] = float("inf")
        wild = call(t)
        keep = torch.ones(9, dtype=torch.bool, device="cuda")
        keep[5] = keep[6] = False
        for x, y in zip(clean, wild):
            assert torch.equal(x[0][keep], y[0][keep])
        assert wild[1][0, 5].isnan().all() and wild[1][0, 6, width - 1].isnan()
        _, values, scale = call(t, quantize=True)
        assert torch.equal(values[0][keep], bytes_clean[1][0][keep]) and torch.equal(scale[0][keep], bytes_clean[2][0][keep])
        assert scale[0, 5].isnan() and scale[0, 6].isnan() and bool((values[0, 5:7] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", [8, 100, 1024, 1031, 4096, 11000])
def test_bytes(cuda_device, dtype, width):
    gen = torch.Generator(device="cuda").manual_seed(8)
    t = inputs(gen, 2, 17, width, dtype, "width")
    h, values, scale = call(t, quantize=True)
    assert values.shape == h.shape and scale.shape == h.shape[:-1] and values.stride(-2) % 16 == 0
    want = R.residual_norm(t["x"], t["branch"], t["weight"], t["post_weight"], t["gate"], eps=EPS)
    R.check("h", h, *want["h"])
    n, bound = want["n"]
    bound = bound - R.UNIT[dtype] * n.abs()              # rounded from its fp32 value, not from the tensors' type
    # half a step, and the error of the largest value through the scale
    R.check("n", values.double() * scale.double()[..., None], n,
            bound + scale.double()[..., None] * (0.5 + 1e-4) + bound.amax(-1, keepdim=True))
    assert bool((values.abs().amax(-1) == 127).all())


def test_repeats_bit_for_bit(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(9)
    t = {k: v.requires_grad_(True) for k, v in inputs(gen, 2, 3000, 768, BF16, "sequence").items()}
    dh, dn = normal(gen, 2, 3000, 768), normal(gen, 2, 3000, 768)
    runs = [torch.autograd.grad(call(t), list(t.values()), (dh, dn)) for _ in range(2)]
    for x, y in zip(*runs):
        assert torch.equal(x, y)


@pytest.mark.parametrize("gate", ["width", "sequence", "token"])
def test_gradient_against_differences(cuda_device, gate):
    """A step along each operand alone moves the loss as its gradient says."""
    gen = torch.Generator(device="cuda").manual_seed(10)
    t = {k: v.double() for k, v in inputs(gen, 2, 6, 96, F32, gate).items()}
    w = [normal(gen, 2, 6, 96, dtype=F32) for _ in range(2)]
    leaves = {k: v.float().requires_grad_(True) for k, v in t.items()}
    grads = dict(zip(leaves, torch.autograd.grad(call(leaves, 0.8, 1.3), list(leaves.values()), w)))
    step = 2.0 ** -7

    def loss(moved):
        want = R.residual_norm(moved["x"], moved["branch"], moved["weight"], moved["post_weight"], moved["gate"], 0.8, 1.3, EPS)
        return sum(float((want[k][0] * g.double()).sum()) for k, g in zip(("h", "n"), w))

    def third(k, way):
        """The loss's change by the central difference at two step sizes: their gap bounds its error."""
        found = []
        for s in (step, step / 2):
            up, down = loss({**t, k: (t[k].float().double() + s * way)}), loss({**t, k: (t[k].float().double() - s * way)})
            found.append((up - down) / (2 * s))
        return found

    t = {k: v.float().double() for k, v in t.items()}
    for k, g in grads.items():
        way = torch.randn(g.shape, generator=gen, device="cuda", dtype=torch.float64)
        coarse, fine = third(k, way)
        along = float((g.double() * way).sum())
        size = float((g.double().abs() * way.abs()).sum())
        assert abs(fine - along) <= 2 * abs(fine - coarse) + 1e-4 * size, k
        assert abs(along) > 1e-3 * size or size < 1e-6


def test_captured_and_replayed(cuda_device):
    """A training step and a serving step in a graph, replayed on other data; another stream."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    t = {k: v.requires_grad_(True) for k, v in inputs(gen, 3, 50, 640, BF16, "sequence").items()}
    dh, dn = normal(gen, 3, 50, 640), normal(gen, 3, 50, 640)

    def step():
        h, n = call(t)
        grads = torch.autograd.grad((h, n), list(t.values()), (dh, dn))
        with torch.no_grad():
            return (h.detach(), n.detach(), *grads, *call(t, quantize=True))

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
            for v in (*t.values(), dh, dn):
                v.copy_(normal(gen, *v.shape, dtype=v.dtype))
        graph.replay()
        for x, y in zip(got, step()):
            assert torch.equal(x, y)


def test_refusals(cuda_device):
    import nlogn_pisa_b200 as P
    from torch.autograd import forward_ad

    gen = torch.Generator(device="cuda").manual_seed(12)
    t = inputs(gen, 1, 4, 64, BF16)
    with pytest.raises(ValueError, match="inference"):
        call({**t, "x": t["x"].clone().requires_grad_(True)}, quantize=True)
    with pytest.raises(ValueError, match="16384"):
        P.residual_norm(normal(gen, 1, 1, 16392), None, torch.ones(16392, device="cuda"))
    with pytest.raises(ValueError, match="support"):
        P.residual_norm(t["x"].double(), t["x"].double(), t["weight"].double())
    with pytest.raises(ValueError, match="scales"):
        call(t, float("nan"))
    with pytest.raises(ValueError, match="numbers"):
        call(t, 1.0, torch.ones((), device="cuda", requires_grad=True))
    with forward_ad.dual_level():
        dual = {**t, "branch": forward_ad.make_dual(t["branch"], torch.ones_like(t["branch"]))}
        with pytest.raises(RuntimeError, match="jvp"):
            call(dual)
