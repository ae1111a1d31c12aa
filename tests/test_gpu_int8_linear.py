"""int8_linear against exact integer sums."""

import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def bytes_of(gen, *shape):
    return torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)


def scales(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda") * 0.01 + 1e-4


def case(gen, tokens, inner, outer):
    return bytes_of(gen, tokens, inner), scales(gen, tokens), bytes_of(gen, outer, inner), scales(gen, outer)


def compare(x, x_scale, w, w_scale, bias=None, dtype=BF16):
    import nlogn_pisa_b200 as P

    out = P.int8_linear(x, w, w_scale, bias=bias, x_scale=x_scale, out_dtype=dtype)
    assert out.dtype == dtype and out.shape == (*x.shape[:-1], w.shape[0]) and out.is_contiguous()
    R.check("out", out, *R.int8_linear(x, x_scale, w, w_scale, bias, dtype))
    return out


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 600])
@pytest.mark.parametrize("inner,outer", [(1, 1), (16, 7), (100, 128), (128, 129), (129, 255), (1000, 64), (1024, 1001), (2064, 300)])
def test_sizes(cuda_device, tokens, inner, outer):
    gen = torch.Generator(device="cuda").manual_seed(tokens + inner)
    x, xs, w, ws = case(gen, tokens, inner, outer)
    compare(x, xs, w, ws, dtype=BF16)
    compare(x, xs, w, ws, scales(gen, outer) * 1000, F32)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,inner,outer", [(3, 4096, 6144), (64, 2816, 1024), (200, 1024, 5632), (1500, 512, 2817), (2100, 768, 2048)])
def test_types_and_bias(cuda_device, dtype, tokens, inner, outer):
    gen = torch.Generator(device="cuda").manual_seed(outer)
    x, xs, w, ws = case(gen, tokens, inner, outer)
    compare(x, xs, w, ws, None, dtype)
    compare(x, xs, w, ws, scales(gen, outer) * 100, dtype)
    compare(x, xs, w, ws, (scales(gen, outer) * 100).to(dtype), dtype)


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_long_sums_are_exact(cuda_device, tokens):
    """Sums near 2^31: every byte -128 or 127, and a K that fills no block."""
    inner = (1 << 17) - 1
    x = torch.full((tokens, inner), -128, dtype=torch.int8, device="cuda")
    w = torch.full((130, inner), -128, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    ones = torch.ones(130, device="cuda")
    out = compare(x, ones[:1].expand(tokens).contiguous(), w, ones, dtype=F32)
    assert float(out[0, 0]) == float(torch.tensor(inner * 16384, dtype=torch.float32))


def test_large(cuda_device):
    """Many tiles per CTA, in both directions; long K, where pairs of CTAs share tiles."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    compare(*case(gen, 4099, 640, 3000), dtype=BF16)
    compare(*case(gen, 4099, 2820, 865), dtype=F16)
    compare(*case(gen, 2500, 4096, 3001), scales(gen, 3001), F32)
    compare(*case(gen, 700, 9000, 1030), dtype=BF16)
    compare(*case(gen, 9000, 200, 1100), scales(gen, 1100), F16)
    compare(*case(gen, 20, 300, 70000), dtype=F32)


def test_layouts(cuda_device):
    """Strided and unaligned rows; the bytes between rows are not used; leading dimensions."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(2)
    x, xs, w, ws = case(gen, 24, 208, 96)
    want = compare(x, xs, w, ws)
    wide_x, wide_w = (torch.full((t.shape[0], 256), 99, dtype=torch.int8, device="cuda") for t in (x, w))
    wide_x[:, 16:224], wide_w[:, 32:240] = x, w
    assert torch.equal(compare(wide_x[:, 16:224], xs, wide_w[:, 32:240], ws), want)
    wide_x[:, 3:211], wide_w[:, 5:213] = x, w
    assert torch.equal(compare(wide_x[:, 3:211], xs, wide_w[:, 5:213], ws), want)
    assert torch.equal(compare(x.T.contiguous().T, xs, w.T.contiguous().T, ws), want)
    folded = compare(x.view(2, 3, 4, 208), xs.view(2, 3, 4), w, ws)
    assert torch.equal(folded.view(24, 96), want)
    assert torch.equal(compare(x[0], xs[0], w, ws), want[0])
    assert torch.equal(compare(x[:1].expand(5, -1), xs[:1].expand(5), w, ws), want[:1].expand(5, -1))
    assert torch.equal(P.int8_linear(x, w, torch.stack((ws, ws), 1)[:, 0], x_scale=xs), want)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,inner", [(1, 64), (50, 1000), (300, 4099), (1, 1), (1, 5000), (1, 16384), (2, 8192), (3, 5461), (5, 777),
                                          (7, 2048), (9, 1820), (16, 1024), (16, 1023), (15, 128), (17, 512), (4, 4100)])
def test_floating_tokens_are_rounded_in_the_call(cuda_device, dtype, tokens, inner):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(inner)
    x = torch.randn(tokens, inner, generator=gen, device="cuda").to(dtype)
    w, ws = P.quantize_int8(torch.randn(70, inner, generator=gen, device="cuda"))
    values, scale = R.quantized(x.float())
    out = P.int8_linear(x, w, ws)
    assert out.dtype == dtype
    R.check("out", out, *R.int8_linear(values, scale, w, ws, None, dtype))
    # the same bytes as tokens rounded before, other layouts, many tiles
    assert torch.equal(out, P.int8_linear(values, w, ws, x_scale=scale, out_dtype=dtype))
    wide = torch.randn(tokens, inner + 9, generator=gen, device="cuda").to(dtype)
    wide[:, 3:inner + 3] = x
    assert torch.equal(out, P.int8_linear(wide[:, 3:inner + 3], w, ws))
    w, ws = P.quantize_int8(torch.randn(20003, inner, generator=gen, device="cuda"))
    bias = torch.randn(20003, generator=gen, device="cuda")
    out = P.int8_linear(x, w, ws, bias=bias)
    R.check("out", out, *R.int8_linear(values, scale, w, ws, bias, dtype))


def test_wild_rows_keep_to_themselves(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(3)
    w, ws = P.quantize_int8(torch.randn(100, 256, generator=gen, device="cuda"))
    for tokens in (40, 11):
        x = torch.randn(tokens, 256, generator=gen, device="cuda")
        clean = P.int8_linear(x, w, ws)
        x[7, 3], x[9, 100], x[4] = float("nan"), float("inf"), 0
        wild = P.int8_linear(x, w, ws)
        keep = torch.ones(tokens, dtype=torch.bool, device="cuda")
        keep[[4, 7, 9]] = False
        assert torch.equal(clean[keep], wild[keep]) and bool(wild[[7, 9]].isnan().all()) and bool((wild[4] == 0).all())


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("tokens,inner,outer", [(1, 64, 7), (17, 500, 130), (270, 128, 129), (700, 4096, 300)])
def test_nothing_is_written_past_the_rows(cuda_device, out, tokens, inner, outer):
    from nlogn_pisa_b200 import _lib

    gen = torch.Generator(device="cuda").manual_seed(4)
    step = -(-inner // 16) * 16
    x, w = (torch.zeros(n, step, dtype=torch.int8, device="cuda") for n in (tokens, outer))
    x[:, :inner], w[:, :inner] = bytes_of(gen, tokens, inner), bytes_of(gen, outer, inner)
    xs, ws = scales(gen, tokens), scales(gen, outer)
    spare = 4096
    got = torch.full((tokens * outer + 2 * spare,), 7.0, dtype=out, device="cuda")
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    size = lib.pisa_int8_linear_workspace_bytes(tokens, inner, outer, _lib.S8)
    workspace = torch.full((size + 4096,), 85, dtype=torch.uint8, device="cuda")
    _lib.check(lib.pisa_int8_linear(x.data_ptr(), step, _lib.S8, xs.data_ptr(), w.data_ptr(), step, ws.data_ptr(), None, 0, _lib.DTYPES[out],
                                    tokens, inner, outer, got.data_ptr() + spare * got.element_size(), workspace.data_ptr(), size,
                                    stream))
    assert bool((got[:spare] == 7).all()) and bool((got[-spare:] == 7).all())
    assert bool((workspace[size:] == 85).all())
    _lib.check_workspace(workspace, x.device)
    R.check("out", got[spare:-spare].view(tokens, outer), *R.int8_linear(x[:, :inner], xs, w[:, :inner], ws, None, out))
    # floating tokens, rounded in the workspace
    f = torch.randn(tokens, inner, generator=gen, device="cuda").to(BF16)
    size = lib.pisa_int8_linear_workspace_bytes(tokens, inner, outer, _lib.BF16)
    workspace = torch.full((size + 4096,), 85, dtype=torch.uint8, device="cuda")
    got.fill_(7.0)
    _lib.check(lib.pisa_int8_linear(f.data_ptr(), inner, _lib.BF16, None, w.data_ptr(), step, ws.data_ptr(), None, 0,
                                    _lib.DTYPES[out], tokens, inner, outer, got.data_ptr() + spare * got.element_size(),
                                    workspace.data_ptr(), size, stream))
    assert bool((got[:spare] == 7).all()) and bool((got[-spare:] == 7).all()) and bool((workspace[size:] == 85).all())
    _lib.check_workspace(workspace, x.device)
    R.check("out", got[spare:-spare].view(tokens, outer), *R.int8_linear(*R.quantized(f.float()), w[:, :inner], ws, None, out))


def test_repeats_and_status(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(5)
    x, xs, w, ws = case(gen, 300, 2048, 1500)
    first = P.int8_linear(x, w, ws, x_scale=xs)
    P.set_status_checks(True)
    try:
        assert torch.equal(P.int8_linear(x, w, ws, x_scale=xs), first)
        assert torch.equal(P.int8_linear(x.float(), w, ws), P.int8_linear(x.float(), w, ws))
    finally:
        P.set_status_checks(False)


def test_two_streams_and_graphs(cuda_device):
    """Calls that overlap on two streams, and two captured graphs replayed in turn, share nothing."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(6)
    cases = [case(gen, 5, 4096, 1200), case(gen, 300, 1024, 900)]

    def step(c):
        return P.int8_linear(c[0], c[2], c[3], x_scale=c[1])

    want = [step(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(step(c))
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    graphs = []
    for s, c in zip(streams, cases):
        with torch.cuda.stream(s):
            step(c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(c)
        graphs.append((graph, out))
    for c in cases:
        c[0].copy_(bytes_of(gen, *c[0].shape))
    for s, (graph, _) in zip(streams, graphs):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for (_, out), c in zip(graphs, cases):
        assert torch.equal(out, step(c))


def test_layer(cuda_device):
    import nlogn_pisa_b200 as P
    from torch import nn

    gen = torch.Generator(device="cuda").manual_seed(7)
    a, b = nn.Linear(100, 48, device="cuda", dtype=BF16), nn.Linear(100, 30, device="cuda", dtype=BF16)
    layer = P.Int8Linear.from_linear(a, b)
    x = torch.randn(3, 7, 100, generator=gen, device="cuda").to(BF16)
    out = layer(x)
    w, ws = R.quantized(torch.cat((a.weight, b.weight)).detach().float())
    values, scale = R.quantized(x.float())
    R.check("out", out, *R.int8_linear(values, scale, w, ws, torch.cat((a.bias, b.bias)).detach().float(), BF16))
    assert torch.equal(layer(values, x_scale=scale), out)
    half = layer.half()
    assert half.weight_scale.dtype == F32 and half.weight.dtype == torch.int8
    assert torch.equal(P.Int8Linear.from_linear(nn.Linear(64, 8, bias=False, device="cuda"))(x[..., :64]).isfinite(),
                       torch.ones(3, 7, 8, dtype=torch.bool, device="cuda"))
    other = P.Int8Linear(100, 78).to("cuda")
    other.load_state_dict(P.Int8Linear.from_linear(a, b).state_dict())
    assert torch.equal(other(x), out)
    with pytest.raises(ValueError, match="share their input"):
        P.Int8Linear.from_linear(a, nn.Linear(64, 8, device="cuda", dtype=BF16))


def test_refusals(cuda_device):
    import nlogn_pisa_b200 as P
    from torch.autograd import forward_ad

    gen = torch.Generator(device="cuda").manual_seed(8)
    x, xs, w, ws = case(gen, 4, 64, 8)
    with pytest.raises(ValueError, match="inference"):
        P.int8_linear(x.float().requires_grad_(True), w, ws)
    with pytest.raises(ValueError, match="inference"):
        P.int8_linear(x, w, ws, x_scale=xs, bias=torch.zeros(8, device="cuda", requires_grad=True))
    with pytest.raises(ValueError, match="support"):
        P.int8_linear(x.double(), w, ws)
    with pytest.raises(ValueError, match="CUDA"):
        P.int8_linear(x, w, ws.cpu(), x_scale=xs)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="inference"):
        P.int8_linear(forward_ad.make_dual(x.float(), x.float()), w, ws)
