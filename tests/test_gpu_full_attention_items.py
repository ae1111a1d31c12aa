"""full_attention over so many keys that one work item outlasts half a second."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_every_item_is_written(cuda_device):
    """Waits for a whole item allow for its length: none expires, and the status word says so."""
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(1)
    keys, dim = 1 << 26, 8
    q = torch.randn(1, 1, 1, dim, generator=gen, device="cuda").to(torch.bfloat16)
    k = torch.empty(1, keys, 1, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    v = torch.ones(1, keys, 1, dim, dtype=torch.bfloat16, device="cuda")
    P.set_status_checks(True)
    try:
        out, lse = P.full_attention(q, k, v, return_lse=True)
    finally:
        P.set_status_checks(False)
    assert torch.isfinite(out).all()
    logits = (k[0, :, 0].float() @ q[0, 0, 0].float()).double() * dim ** -0.5
    # 2^19 sums of 128 weights in fp32, at random; half a unit each at most
    assert abs(float(lse[0, 0, 0]) - float(torch.logsumexp(logits, 0))) <= 2.0 ** -10
