"""Host-side contract of the dense-attention operators (no GPU)."""

import pytest
import torch


def test_cpu_tensors_are_refused():
    import nlogn_pisa_b200 as P

    q, k = torch.zeros(1, 4, 4, 64), torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        P.full_attention(q, k, k)
    with pytest.raises(ValueError, match="CUDA"):
        P.prefix_attention(q, k, k, torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        P.qk_norm_rotary(q, k, torch.ones(64), torch.ones(64), torch.ones(32))


def test_entry_checks_run_on_the_host():
    """Bad shapes are refused before any device work."""
    from nlogn_pisa_b200 import _lib

    lib = _lib.lib()

    def full(B=1, T=4, Hq=4, H=2, D=64, Dv=64, N=4, scale=0.125, offset=0, dtype=_lib.BF16, align=256):
        p = align
        return lib.pisa_full_attn_fwd(p, 0, Hq * D, D, p, 0, H * D, D, p, 0, H * Dv, Dv, None, None, 0, 0, offset, dtype, B,
                                      T, Hq, H, D, Dv, N, scale, 1, None, None, None, None, 0, None)

    for kw, word in (({"Hq": 3}, "whole number"), ({"D": 12}, "multiple of 8"), ({"Dv": 512}, "at most 256"),
                     ({"T": 0}, "nonempty"), ({"scale": 0.0}, "scale"), ({"scale": float("nan")}, "scale"),
                     ({"offset": 3}, "positions"), ({"offset": -1}, "positions"), ({"dtype": 7}, "support"),
                     ({"align": 8}, "aligned"), ({"N": 1 << 31}, "too large"), ({}, "out is required")):
        rc = full(**kw)
        assert rc in (_lib.ERR_INVALID, _lib.ERR_UNSUPPORTED), kw
        assert word in lib.pisa_last_error().decode(), (kw, lib.pisa_last_error())
    # a row of 12 bytes apart
    rc = lib.pisa_full_attn_fwd(256, 0, 250, 62, 256, 0, 128, 64, 256, 0, 128, 64, None, None, 0, 0, 0, _lib.BF16, 1, 4, 4,
                                2, 64, 64, 4, 0.1, 1, 256, None, None, None, 0, None)
    assert rc == _lib.ERR_UNSUPPORTED and "aligned" in lib.pisa_last_error().decode()


def test_workspace_sizes_are_pure_host_functions():
    from nlogn_pisa_b200 import _lib

    lib = _lib.lib()
    assert lib.pisa_full_attn_fwd_workspace_bytes(1, 100, 4, 2, 64, 64, 100, 0, _lib.BF16) >= 256
    assert lib.pisa_full_attn_bwd_workspace_bytes(1, 100, 4, 2, 64, 64, 100, 3, _lib.BF16) >= 256 + 1600
    assert lib.pisa_full_attn_bwd_workspace_bytes(0, 100, 4, 2, 64, 64, 100, 3, _lib.BF16) == -1
    assert lib.pisa_prefix_attn_workspace_bytes(2, 1, 8, 2, 64, 64, 100, 0, _lib.BF16) >= 256
    assert lib.pisa_prefix_attn_workspace_bytes(2, 1, 8, 3, 64, 64, 100, 0, _lib.BF16) == -1
    assert lib.pisa_qk_norm_rotary_bwd_workspace_bytes(1, 1, 64) == 512
    assert lib.pisa_qk_norm_rotary_bwd_workspace_bytes(0, 1, 64) == -1
