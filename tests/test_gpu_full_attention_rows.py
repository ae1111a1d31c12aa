"""Gradients of full_attention summed over very many query rows or keys."""

import pytest
import torch

from test_gpu_full_attention_gradients import cumulative, room

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def by_chunks(q, k, v, dout, causal, shift, rows=4096):
    """dq [T,G,D], dk, dv of one KV head in 64 bits, some rows at a time."""
    k, v, scale = k.double(), v.double(), k.shape[-1] ** -0.5
    dq, dk, dv = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros_like(k), torch.zeros_like(v)
    cols = torch.arange(k.shape[0], device="cuda")
    for g in range(q.shape[1]):
        for a in range(0, q.shape[0], rows):
            x, d = q[a:a + rows, g].double(), dout[a:a + rows, g].double()
            s = x @ k.T * scale
            if causal:
                s.masked_fill_(cols[None] > torch.arange(a, a + x.shape[0], device="cuda")[:, None] + shift, float("-inf"))
            p = torch.softmax(s, -1).masked_fill(torch.isneginf(s).all(-1, keepdim=True), 0.0)   # rows without keys weigh nothing
            ds = scale * p * (d @ v.T - (d * (p @ v)).sum(-1, keepdim=True))
            dq[a:a + rows, g] = ds @ k
            dk += ds.T @ x
            dv += p.T @ d
    return dq, dk, dv


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("queries,keys,heads,dim,causal", [
    ([131072], [128], 8, 64, False), ([70001], [300], 16, 128, False), ([20000], [20000], 8, 64, True), ([17000], [17003], 4, 128, True),
    ([100, 30001, 1], [70, 33000, 500], 4, 80, True), ([300], [200001], 2, 64, False), ([130, 129], [131073, 70000], 2, 128, True)])
def test_one_kv_head(cuda_device, dtype, queries, keys, heads, dim, causal):
    """Items of more tiles than one part, that begin and end inside a head and in ragged tiles."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(sum(queries))

    def normal(n, h, size=1.0, mean=0.0):
        return torch.empty(1, n, h, dim, device="cuda").normal_(mean, size, generator=gen).to(dtype).requires_grad_(True)

    q, k, v = normal(sum(queries), heads, 0.3), normal(sum(keys), 1), normal(sum(keys), 1)
    dout = normal(sum(queries), heads, 30.0, 10.0).detach()
    out = P.full_attention(q, k, v, cu_seqlens=cumulative(queries), cu_seqlens_k=cumulative(keys), causal=causal)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    again = torch.autograd.grad(P.full_attention(q, k, v, cu_seqlens=cumulative(queries), cu_seqlens_k=cumulative(keys), causal=causal),
                                (q, k, v), dout)
    for x, y in zip(grads, again):
        assert torch.equal(x, y)
    q0 = k0 = 0
    for n, m in zip(queries, keys):
        want = by_chunks(q[0, q0:q0 + n].detach(), k[0, k0:k0 + m, 0].detach(), v[0, k0:k0 + m, 0].detach(), dout[0, q0:q0 + n],
                         causal, m - n)
        got = grads[0][0, q0:q0 + n], grads[1][0, k0:k0 + m, 0], grads[2][0, k0:k0 + m, 0]
        for name, x, y in zip(("dq", "dk", "dv"), got, want):
            off, most = float((x.double() - y).norm()), room(y, dtype)
            assert off <= most, (name, n, m, off / float(y.norm()), most / float(y.norm()))
        q0, k0 = q0 + n, k0 + m
