"""qk_norm_rotary with eps 0, and eps that are refused."""

import math

import pytest
import torch

from test_gpu_norm_rotary import compare, inputs

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("batch,tokens,heads,kv_heads,dim", [(1, 1, 1, 1, 64), (2, 7, 5, 3, 128), (1, 333, 5, 1, 80),
                                                             (3, 1001, 3, 2, 64), (1, 50, 7, 1, 8)])
def test_eps_zero(cuda_device, dtype, batch, tokens, heads, kv_heads, dim):
    """Rows that fill up a warp's step are no rows of length zero."""
    gen = torch.Generator(device="cuda").manual_seed(dim + tokens)
    q, k, qw, kw, frequency = inputs(gen, batch, tokens, heads, kv_heads, dim, dtype, F32)
    compare(q, k, qw, kw, frequency, eps=0.0)


@pytest.mark.gpu
def test_zero_rows_with_eps_zero_keep_to_themselves(cuda_device):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, qw, kw, frequency = inputs(gen, 1, 9, 5, 3, 64, BF16, BF16)
    clean = P.qk_norm_rotary(q, k, qw, kw, frequency, eps=0.0)
    q[0, 3, 2] = 0
    out = P.qk_norm_rotary(q, k, qw, kw, frequency, eps=0.0)
    keep = torch.ones(9, 5, dtype=torch.bool, device="cuda")
    keep[3, 2] = False
    assert torch.equal(out[0][0][keep], clean[0][0][keep]) and torch.equal(out[1], clean[1])
    assert out[0][0, 3, 2].isnan().all()      # 0 / 0


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [-1e-6, math.nan, math.inf])
def test_refused(cuda_device, eps):
    import nlogn_pisa_b200 as P

    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, qw, kw, frequency = inputs(gen, 1, 4, 4, 2, 64, BF16, BF16)
    with pytest.raises(ValueError, match="eps"):
        P.qk_norm_rotary(q, k, qw, kw, frequency, eps=eps)


@pytest.mark.parametrize("eps", [-1e-6, math.nan, math.inf])
def test_entry_points_refuse(eps):
    from nlogn_pisa_b200 import _lib

    lib, p = _lib.lib(), 256
    views = (p, 0, 256, 64, p, 0, 128, 64)
    common = (p, p, _lib.BF16, p, None, 0, 0, _lib.BF16, 1, 4, 4, 2, 64, eps)
    for rc in (lib.pisa_qk_norm_rotary(*views, *common, p, p, None),
               lib.pisa_qk_norm_rotary_bwd(*views, p, p, *common, p, p, p, p, p, 1 << 20, None)):
        assert rc == _lib.ERR_INVALID and "eps" in lib.pisa_last_error().decode()
