"""The decoder block's operators on tensors of more than 2^31 elements: rows are
their own, so the last ones equal a call on them alone, bit for bit."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
TAIL = 1000      # rows of the small call: enough for the same kernels


@pytest.fixture
def room(cuda_device):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    yield
    torch.cuda.empty_cache()


def filled(rows, width):
    """Cheap values that differ from row to row: a tile of random ones, shifted."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    tile = torch.randn(1 << 14, width, generator=gen, device="cuda").to(BF16)
    out = torch.empty(rows, width, dtype=BF16, device="cuda")
    for at in range(0, rows, 1 << 14):
        n = min(1 << 14, rows - at)
        out[at:at + n] = tile.roll(at >> 14, 1)[:n]
    return out


def test_residual_norm(room):
    import nlogn_pisa_b200 as P

    rows, width = (1 << 31) // 1024 + 5000, 1024
    x, branch = filled(rows, width), filled(rows, width)
    branch[-TAIL:] *= 0.5
    w, gate = torch.rand(width, device="cuda"), torch.rand(width, device="cuda").to(BF16)

    def call(x, branch):
        leaves = [x.requires_grad_(True), branch.requires_grad_(True)]
        h, n = P.residual_norm(*leaves, w, post_weight=w, gate=gate)
        dx, dbranch = torch.autograd.grad((h, n), leaves, (branch.detach(), x.detach()))
        return h.detach()[-TAIL:].clone(), n.detach()[-TAIL:].clone(), dx[-TAIL:].clone(), dbranch[-TAIL:].clone()

    big = call(x, branch)
    small = call(*(t.detach()[-TAIL:].clone() for t in (x, branch)))
    for a, b in zip(big, small):
        assert torch.equal(a, b)
    with torch.no_grad():
        big = [t[-TAIL:] for t in P.residual_norm(x, branch, w, quantize=True)]
        for a, b in zip(big, P.residual_norm(x[-TAIL:].clone(), branch[-TAIL:].clone(), w, quantize=True)):
            assert torch.equal(a, b)


def test_swiglu(room):
    import nlogn_pisa_b200 as P

    rows, width = (1 << 31) // 2816 + 5000, 2816
    gate, up = filled(rows, width), filled(rows, width)
    up[-TAIL:] *= 0.5

    def call(gate, up):
        leaves = [gate.requires_grad_(True), up.requires_grad_(True)]
        out = P.swiglu(*leaves, checkpoint_bits=8)
        return [t.detach()[-TAIL:].clone() for t in (out, *torch.autograd.grad(out, leaves, gate.detach()))]

    big = call(gate, up)
    small = call(*(t.detach()[-TAIL:].clone() for t in (gate, up)))
    for a, b in zip(big, small):
        assert torch.equal(a, b)
    with torch.no_grad():
        for a, b in zip(P.swiglu(gate, up, quantize=True), P.swiglu(gate[-TAIL:].clone(), up[-TAIL:].clone(), quantize=True)):
            assert torch.equal(a[-TAIL:], b)


def test_int8_linear(room):
    """More than 2^31 bytes of tokens, and more than 2^31 outputs."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(1)
    for tokens, inner, outer in (((1 << 31) // 2048 + 3000, 2048, 128), ((1 << 31) // 20000 + 1000, 64, 20000)):
        x = torch.randint(-127, 128, (tokens, inner), generator=gen, device="cuda", dtype=torch.int8)
        w = torch.randint(-127, 128, (outer, inner), generator=gen, device="cuda", dtype=torch.int8)
        xs, ws = torch.rand(tokens, generator=gen, device="cuda"), torch.rand(outer, generator=gen, device="cuda")
        out = P.int8_linear(x, w, ws, x_scale=xs)[-TAIL:].clone()
        assert torch.equal(out, P.int8_linear(x[-TAIL:].clone(), w, ws, x_scale=xs[-TAIL:].clone()))
        del x
        torch.cuda.empty_cache()
