"""The full-attention token mixer end to end: training, packed documents, decode caches, a shared prefix."""

import math
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

# sums of bf16 products through four projections and the attention between
# them: five roundings of 2^-8 relative to magnitudes of the same size
BF16_TOL, F32_TOL = 5 * 2.0 ** -8, 1e-4


def make(dtype, **kw):
    from nlogn_pisa_b200.mixer import FullAttention

    base = dict(hidden_size=256, num_attention_heads=8, num_key_value_heads=2, head_dim=64, attention_method="full",
                rope_theta=10000.0, rope_fraction=0.5, rope_position_mode="document", bias=False, rms_norm_eps=1e-6)
    base.update(kw)
    torch.manual_seed(0)
    mixer = FullAttention(SimpleNamespace(**base)).cuda()
    with torch.no_grad():
        for w in (mixer.q_norm, mixer.k_norm):
            w.add_(0.1 * torch.randn_like(w))
    return mixer.to(dtype)


def plain(mixer, x, documents=None):
    """The layer in float64 with torch operations."""
    cfg = mixer.config
    x = x.double()
    weight = {n: p.detach().double() for n, p in mixer.named_parameters()}
    batch, length, _ = x.shape

    def heads(name, n):
        return (x @ weight[name + ".weight"].T).view(batch, length, n, cfg.head_dim)

    q, k, v = heads("q_proj", cfg.num_attention_heads), heads("k_proj", cfg.num_key_value_heads), heads("v_proj", cfg.num_key_value_heads)
    documents = [length] if documents is None else documents
    position = torch.cat([torch.arange(n, device=x.device) for n in documents]).double()
    number = torch.cat([torch.full((n,), i, device=x.device) for i, n in enumerate(documents)])
    angle = (position[:, None] * mixer.theta.double())[:, None]

    def rotate(y, w):
        y = y / (y.square().mean(-1, keepdim=True) + mixer.eps).sqrt() * w
        a, b = y.chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1)

    q, k = rotate(q, weight["q_norm"]), rotate(k, weight["k_norm"])
    group = cfg.num_attention_heads // cfg.num_key_value_heads
    k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) * cfg.head_dim ** -0.5
    hidden = (number[:, None] != number[None]) | (torch.arange(length, device=x.device)[:, None] < torch.arange(length, device=x.device))
    p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
    out = torch.einsum("bhqk,bkhd->bqhd", p, v).reshape(batch, length, -1)
    return out @ weight["o_proj.weight"].T


def near(got, want, dtype):
    tol = F32_TOL if dtype == torch.float32 else BF16_TOL
    scale = float(want.double().square().mean().sqrt())
    assert float((got.double() - want.double()).abs().max()) <= 4 * tol * scale + 1e-12


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_and_documents(cuda_device, dtype):
    mixer = make(dtype)
    x = torch.randn(2, 300, 256, device="cuda").to(dtype)
    near(mixer(x)[0], plain(mixer, x), dtype)
    cu = torch.tensor([0, 100, 101, 300], device="cuda")
    near(mixer(x[:1], cu_seqlens=cu)[0], plain(mixer, x[:1], [100, 1, 199]), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_follows_the_prompt(cuda_device, dtype):
    mixer = make(dtype)
    x = torch.randn(3, 180, 256, device="cuda").to(dtype)
    want = plain(mixer, x)
    with torch.no_grad():
        out, cache = mixer(x[:, :100], use_cache=True)
        near(out, want[:, :100], dtype)
        for begin, end in ((100, 101), (101, 105), (105, 150), (150, 151)):
            look, none = mixer(x[:, begin:end], cache=cache)
            assert none is None and cache["k"].shape[1] == begin
            out, cache = mixer(x[:, begin:end], cache=cache, use_cache=True)
            assert torch.equal(look, out)
            near(out, want[:, begin:end], dtype)
    layers = [None]
    out, layers = mixer(x[:, :50], past_key_values=layers, use_cache=True)
    out, layers = mixer(x[:, 50:51], past_key_values=layers, use_cache=True)
    near(out, want[:, 50:51], dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_answers_share_a_prompt(cuda_device, dtype):
    from nlogn_pisa_b200.mixer import FullAttention

    mixer = make(dtype)
    prompt = torch.randn(1, 200, 256, device="cuda").to(dtype)
    answers = torch.randn(5, 40, 256, device="cuda").to(dtype)
    want = plain(mixer, torch.cat((prompt.expand(5, -1, -1), answers), 1))[:, 200:]
    with torch.no_grad():
        _, cache = mixer(prompt, use_cache=True)
        cache = FullAttention.share_prefix(cache)
        for begin, end in ((0, 1), (1, 2), (2, 30), (30, 40)):
            out, cache = mixer(answers[:, begin:end], cache=cache, use_cache=True)
            near(out, want[:, begin:end], dtype)


def test_training_step(cuda_device):
    """Gradients of every parameter against autograd through the float64 layer."""
    mixer = make(torch.float32)
    x = torch.randn(1, 150, 256, device="cuda")
    cu = torch.tensor([0, 60, 150], dtype=torch.int32, device="cuda")
    w = torch.randn(1, 150, 256, device="cuda")
    (mixer(x, cu_seqlens=cu)[0] * w).sum().backward()
    got = {n: p.grad for n, p in mixer.named_parameters()}
    twin = make(torch.float32).double()
    # the same layer with differentiable float64 parameters
    params = {n: p for n, p in twin.named_parameters()}
    twin_named = lambda: ((n, SimpleNamespace(detach=lambda p=p: p)) for n, p in params.items())  # noqa: E731
    (plain(SimpleNamespace(config=twin.config, theta=mixer.theta, eps=mixer.eps, named_parameters=twin_named), x, [60, 90])
     * w.double()).sum().backward()
    for n, p in params.items():
        near(got[n], p.grad, torch.float32)


def test_decoder_block_trains(cuda_device):
    from nlogn_pisa_b200.model import BlockConfig, DecoderBlock

    torch.manual_seed(1)
    block = DecoderBlock(BlockConfig(vocab_size=100, hidden_size=256, intermediate_size=512, num_attention_heads=4,
                                     num_key_value_heads=2, head_dim=64, attention_method="full")).cuda().to(torch.bfloat16)
    tokens = torch.randint(0, 100, (1, 500), device="cuda")
    target = torch.randn(1, 500, 256, device="cuda")
    optim = torch.optim.SGD(block.parameters(), lr=0.05)
    cu = torch.tensor([0, 200, 500], dtype=torch.int32, device="cuda")
    losses = []
    for _ in range(8):
        optim.zero_grad()
        loss = (block(tokens, cu_seqlens=cu).float() - target).square().mean()
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in block.parameters())
        optim.step()
        losses.append(float(loss))
    assert losses[-1] < losses[0]


def test_refusals(cuda_device):
    from nlogn_pisa_b200.mixer import FullAttention

    mixer = make(torch.bfloat16)
    x = torch.randn(2, 20, 256, device="cuda").to(torch.bfloat16)
    _, cache = mixer(x, use_cache=True)
    with pytest.raises(ValueError, match="without a cache"):
        mixer(x[:1], cache=cache, cu_seqlens=torch.tensor([0, 20], device="cuda"))
    with pytest.raises(ValueError, match="single prompt"):
        FullAttention.share_prefix(cache)
    with pytest.raises(ValueError, match="padding"):
        mixer(x, attention_mask=torch.tensor([[True, False]]))
    with pytest.raises(ValueError, match="full attention"):
        make(torch.bfloat16, attention_method="pisa")


def test_status_checks_pass_on_the_dense_operators(cuda_device):
    """With checks on, every call reads its status word back: set, and clean."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(3)
    junk = torch.full((1 << 24,), 255, dtype=torch.uint8, device="cuda")   # what the workspaces' memory held before
    del junk
    P.set_status_checks(True)
    try:
        for dtype, dim in ((torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 64), (torch.bfloat16, 256)):
            q, k, v = (torch.randn(2, 300, h, dim, generator=gen, device="cuda").to(dtype).requires_grad_(True) for h in (4, 2, 2))
            P.full_attention(q, k, v).sum().backward()
            n = torch.tensor([300, 7], device="cuda")
            for rows, prefix in ((1, None), (3, None), (1, k[0]), (40, k[0])):
                P.prefix_attention(q[:, :rows], k, v, n, prefix_k=prefix, prefix_v=prefix)
    finally:
        P.set_status_checks(False)


def test_frequencies_stay_fp32(cuda_device):
    from nlogn_pisa_b200.mixer import rotary_frequencies

    mixer = make(torch.bfloat16)
    assert mixer.theta.dtype == torch.float32
    assert torch.equal(mixer.theta.cpu(), rotary_frequencies(64, 10000.0, 0.5))
