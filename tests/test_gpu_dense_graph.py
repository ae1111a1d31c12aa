"""The dense operators captured in a CUDA graph and replayed on other data."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def captured(call):
    """A graph of one call after warm-up on a side stream, and its outputs."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = call()
    return graph, outputs


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("prefix", [0, 100, 5000])
@pytest.mark.parametrize("batch", [1, 24])
def test_decode_step_at_later_positions(cuda_device, dtype, prefix, batch):
    """One captured step serves every later one: lengths, positions and the cache change on the device."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(prefix + batch)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    q, k, new = normal(batch, 1, 8, 64), normal(batch, 700, 2, 64), normal(batch, 1, 2, 64)
    v = normal(batch, 700, 2, 64)
    pk, pv = (normal(prefix, 2, 64), normal(prefix, 2, 64)) if prefix else (None, None)
    w, frequency = torch.ones(64, device="cuda"), torch.rand(32, generator=gen, device="cuda")
    lengths = torch.ones(batch, dtype=torch.int32, device="cuda")
    positions = torch.zeros(batch, 1, dtype=torch.int64, device="cuda")

    def step():
        q_out, k_out = P.qk_norm_rotary(q, new, w, w, frequency, positions=positions)
        return k_out, P.prefix_attention(q_out, k, v, lengths, prefix_k=pk, prefix_v=pv)

    graph, got = captured(step)
    for at in (1, 64, 65, 333, 700):
        q.copy_(normal(batch, 1, 8, 64))
        new.copy_(normal(batch, 1, 2, 64))
        k.copy_(normal(batch, 700, 2, 64))
        lengths.copy_((torch.arange(batch, device="cuda") * 29 + at) % 701)
        positions.copy_(lengths[:, None])
        graph.replay()
        for x, y in zip(got, step()):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128])
def test_training_step_of_other_documents(cuda_device, dtype, dim):
    """Forward and backward of packed documents whose lengths change between replays."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(dim)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    q, k, v = (normal(1, 900, h, dim).requires_grad_(True) for h in (4, 2, 2))
    dout = normal(1, 900, 4, dim)
    cu = torch.tensor([0, 300, 900, 900], dtype=torch.int32, device="cuda")

    def step():
        out = P.full_attention(q, k, v, cu_seqlens=cu)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))

    graph, got = captured(step)
    for bounds in ([0, 300, 900, 900], [0, 1, 130, 900], [0, 899, 899, 900], [0, 256, 512, 900]):
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        with torch.no_grad():
            for x in (q, k, v, dout):
                x.copy_(normal(*x.shape))
        graph.replay()
        for x, y in zip(got, step()):
            assert torch.equal(x, y)
