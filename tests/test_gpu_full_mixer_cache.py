"""The full-attention token mixer with caches: long continuations over a shared prompt, gradients."""

import pytest
import torch

from test_gpu_full_mixer import make, near, plain

pytestmark = pytest.mark.gpu


def answers(mixer, prompt, x, steps):
    """Outputs of x's tokens after a shared prompt, in steps of the given lengths."""
    from nlogn_pisa_b200.mixer import FullAttention

    with torch.no_grad():
        _, cache = mixer(prompt, use_cache=True)
        cache = FullAttention.share_prefix(cache)
        out, begin = [], 0
        for n in steps:
            y, cache = mixer(x[:, begin:begin + n], cache=cache, use_cache=True)
            out.append(y)
            begin += n
    return torch.cat(out, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (4, 4, 128), (8, 1, 96), (2, 1, 160)])
@pytest.mark.parametrize("prompt,steps", [(200, [1, 500, 1, 300]), (1, [17, 16, 129]), (700, [256]), (333, [15, 400, 3])])
def test_long_answers_share_a_prompt(cuda_device, dtype, heads, kv_heads, head_dim, prompt, steps):
    mixer = make(dtype, num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=head_dim)
    first = torch.randn(1, prompt, 256, device="cuda").to(dtype)
    x = torch.randn(3, sum(steps), 256, device="cuda").to(dtype)
    want = plain(mixer, torch.cat((first.expand(3, -1, -1), x), 1))[:, prompt:]
    near(answers(mixer, first, x, steps), want, dtype)


def test_many_rows(cuda_device):
    """More query rows per KV head than the decode kernels take."""
    mixer = make(torch.bfloat16, num_attention_heads=16, num_key_value_heads=1, head_dim=64)
    first = torch.randn(1, 300, 256, device="cuda").to(torch.bfloat16)
    x = torch.randn(64, 1100, 256, device="cuda").to(torch.bfloat16)
    got = answers(mixer, first, x, [1, 1099])
    for b in (0, 31, 63):
        near(got[b:b + 1], plain(mixer, torch.cat((first, x[b:b + 1]), 1))[:, 300:], torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_continued_attention_is_prefix_attention(cuda_device, dtype):
    """The same operation as the decode kernels', within what either rounds (the output, and its weights)."""
    import nlogn_pisa_b200 as P
    from nlogn_pisa_b200 import dense

    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(2, n, h, 64, generator=gen, device="cuda").to(dtype) for n, h in ((90, 4), (200, 2), (200, 2)))
    pk, pv = (torch.randn(500, 2, 64, generator=gen, device="cuda").to(dtype) for _ in range(2))
    want = P.prefix_attention(q, k, v, torch.tensor([200, 200], device="cuda"), prefix_k=pk, prefix_v=pv)
    tight = dense.JOIN_ELEMENTS
    got = dense.continued_attention(q, k, v, pk, pv)
    try:
        dense.JOIN_ELEMENTS = 1      # a sequence at a time
        assert torch.equal(got, dense.continued_attention(q, k, v, pk, pv))
    finally:
        dense.JOIN_ELEMENTS = tight
    unit = {torch.float32: 64 * 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    assert float((got.double() - want.double()).norm()) <= 2 * unit * float(want.double().norm())


def reference_step(mixer, params, history, x):
    """One cached call in float64: ``history`` is every token before it, whose keys and values are constants."""
    cfg, theta = mixer.config, mixer.theta.double()
    group = cfg.num_attention_heads // cfg.num_key_value_heads

    def heads(y, name, n):
        return (y @ params[name + ".weight"].T).view(*y.shape[:2], n, cfg.head_dim)

    def rotate(y, w, offset):
        y = y / (y.square().mean(-1, keepdim=True) + mixer.eps).sqrt() * w
        angle = ((torch.arange(y.shape[1], device=y.device) + offset).double()[:, None] * theta)[:, None]
        a, b = y.chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1)

    past, new = history.shape[1], x.shape[1]
    q = rotate(heads(x, "q_proj", cfg.num_attention_heads), params["q_norm"], past)
    k = rotate(heads(x, "k_proj", cfg.num_key_value_heads), params["k_norm"], past)
    v = heads(x, "v_proj", cfg.num_key_value_heads)
    old_k = rotate(heads(history, "k_proj", cfg.num_key_value_heads), params["k_norm"], 0).detach()
    old_v = heads(history, "v_proj", cfg.num_key_value_heads).detach()
    k, v = (torch.cat(pair, 1).repeat_interleave(group, 2) for pair in ((old_k, k), (old_v, v)))
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) * cfg.head_dim ** -0.5
    hidden = torch.arange(past + new, device=x.device)[None] > past + torch.arange(new, device=x.device)[:, None]
    p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
    return torch.einsum("bhqk,bkhd->bqhd", p, v).reshape(*x.shape[:2], -1) @ params["o_proj.weight"].T


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("steps", [[1, 1], [5, 30], [30, 5], [16, 17]])
@pytest.mark.parametrize("look", [False, True])
def test_gradients_with_a_cache(cuda_device, shared, steps, look):
    """The same gradient rule at every length: this call's tokens get theirs, cached ones are constant."""
    from nlogn_pisa_b200.mixer import FullAttention

    mixer = make(torch.float32)
    batch, prompt = 3, 70
    first = torch.randn(1 if shared else batch, prompt, 256, device="cuda")
    x = torch.randn(batch, sum(steps), 256, device="cuda").requires_grad_(True)
    w = torch.randn(batch, sum(steps), 256, device="cuda")
    with torch.no_grad():
        _, cache = mixer(first, use_cache=True)
    if shared:
        cache = FullAttention.share_prefix(cache)
    params = {n: p.detach().double().requires_grad_(True) for n, p in mixer.named_parameters()}
    x64 = x.detach().double().requires_grad_(True)
    history = first.detach().double().expand(batch, -1, -1)
    loss, want, begin = 0, 0, 0
    for i, n in enumerate(steps):
        at = slice(begin, begin + n)
        if look and i + 1 == len(steps):
            out, _ = mixer(x[:, at], cache=cache)
        else:
            out, cache = mixer(x[:, at], cache=cache, use_cache=True)
        loss = loss + (out * w[:, at]).sum()
        want = want + (reference_step(mixer, params, history, x64[:, at]) * w[:, at].double()).sum()
        history = torch.cat((history, x64[:, at].detach()), 1)
        begin += n
    # the first step's graph is followed after the second step grew the cache in place
    loss.backward()
    want.backward()
    near(x.grad, x64.grad, torch.float32)
    for n, p in mixer.named_parameters():
        near(p.grad, params[n].grad, torch.float32)


@pytest.mark.parametrize("compute", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kept", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_weights_keep_their_bits(cuda_device, compute, kept):
    """Under autocast the norms take the parameters themselves, not a rounded copy."""
    import nlogn_pisa_b200 as P

    mixer = make(torch.float32)
    mixer.q_norm.data, mixer.k_norm.data = mixer.q_norm.data.to(kept), mixer.k_norm.data.to(kept)
    x = torch.randn(2, 130, 256, device="cuda")
    with torch.autocast("cuda", dtype=compute):
        got, _ = mixer(x)
        q, k, v = (getattr(mixer, n)(x).view(2, 130, h, 64) for n, h in (("q_proj", 8), ("k_proj", 2), ("v_proj", 2)))
        assert q.dtype == compute
        q, k = P.qk_norm_rotary(q, k, mixer.q_norm.float(), mixer.k_norm.float(), mixer.theta)
        want = mixer.o_proj(P.full_attention(q, k, v).reshape(2, 130, -1))
    assert torch.equal(got, want)
    got.float().square().sum().backward()
    assert mixer.q_norm.grad.dtype == kept and mixer.k_norm.grad.dtype == kept
    assert torch.isfinite(mixer.q_norm.grad).all() and bool(mixer.q_norm.grad.any())
