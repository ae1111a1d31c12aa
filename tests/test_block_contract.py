"""Host-side contract of the decoder block's operators (no GPU)."""

import pytest
import torch


def test_cpu_tensors_are_refused():
    import nlogn_pisa_b200 as P

    x, w = torch.zeros(2, 3, 64), torch.ones(64)
    q = torch.zeros(2, 64, dtype=torch.int8)
    with pytest.raises(ValueError, match="CUDA"):
        P.residual_norm(x, x, w)
    with pytest.raises(ValueError, match="CUDA"):
        P.swiglu(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        P.swiglu_ffn(x, torch.zeros(8, 64), torch.zeros(8, 64), torch.zeros(64, 8))
    with pytest.raises(ValueError, match="CUDA"):
        P.quantize_int8(x)
    with pytest.raises(ValueError, match="CUDA"):
        P.checkpoint_int8(x)
    with pytest.raises(ValueError, match="CUDA"):
        P.restore_int8(q, torch.zeros(2, 1), torch.float32)
    with pytest.raises(ValueError, match="CUDA"):
        P.int8_linear(x, q, torch.zeros(2))


def test_arguments_are_checked():
    import nlogn_pisa_b200 as P

    x, w = torch.zeros(2, 3, 64), torch.ones(64)
    q, s = torch.zeros(5, 64, dtype=torch.int8), torch.ones(5)
    for args, kw, word in (((x, x[:1], w), {}, "share x's shape"), ((x, x, w[:8]), {}, "weight must have"),
                           ((x, x, w.double()), {}, "weight must have"), ((x, x, w), {"post_weight": w[1:]}, "post_weight"),
                           ((x, x, w), {"gate": torch.zeros(2, 64)}, "gate must have"),
                           ((x, x, w), {"gate": torch.zeros(2, 3, 64, dtype=torch.float16)}, "gate must have"),
                           ((x, x, w), {"gate": w.double()}, "gate must be in"), ((x, None, w), {"gate": w}, "belong to a branch"),
                           ((x, None, w), {"residual_scale": 2.0}, "belong to a branch"), ((w, w, w), {}, "must have shape"),
                           ((x[:, :0], x[:, :0], w), {}, "nonempty"), ((x.int(), x.int(), w), {}, "floating")):
        with pytest.raises(ValueError, match=word):
            P.residual_norm(*args, **kw)
    for args, kw, word in (((x, x[:1]), {}, "share a shape"), ((x, x.half()), {}, "share a shape"),
                           ((x, x), {"checkpoint_bits": 4}, "checkpoint_bits"), ((x[:0], x[:0]), {}, "nonempty")):
        with pytest.raises(ValueError, match=word):
            P.swiglu(*args, **kw)
    for args, kw, word in (((x, q.float(), s), {}, "weight must be int8"), ((x[..., :8], q, s), {}, "last dimension"),
                           ((x, q, s[:2]), {}, "weight_scale"), ((x, q, s), {"x_scale": s}, "comes with x_scale"),
                           ((x.to(torch.int8), q, s), {}, "comes with x_scale"),
                           ((x.to(torch.int8), q, s), {"x_scale": torch.zeros(2)}, "x_scale must"),
                           ((x, q, s), {"bias": s[:2]}, "bias must"), ((x, q, s), {"out_dtype": torch.int32}, "support"),
                           ((x[:0], q, s), {}, "nonempty"),
                           ((torch.zeros(1, 1 << 17), torch.zeros(1, 1 << 17, dtype=torch.int8), s[:1]), {}, "may not fit")):
        with pytest.raises(ValueError, match=word):
            P.int8_linear(*args, **kw)
    with pytest.raises(ValueError, match="nonempty"):
        P.quantize_int8(x[:0])
    with pytest.raises(ValueError, match="floating"):
        P.quantize_int8(q)
    with pytest.raises(ValueError, match="one element per 128"):
        P.restore_int8(q, s, torch.float32)
    with pytest.raises(ValueError, match="share a floating dtype"):
        P.swiglu_ffn(x, torch.zeros(8, 64).half(), torch.zeros(8, 64), torch.zeros(64, 8))


def test_entry_checks_run_on_the_host():
    """Bad shapes are refused before any device work."""
    from nlogn_pisa_b200 import _lib

    lib = _lib.lib()

    def refused(rc, word):
        assert rc in (_lib.ERR_INVALID, _lib.ERR_UNSUPPORTED)
        assert word in lib.pisa_last_error().decode(), lib.pisa_last_error()

    def norm(rows=4, D=64, dtype=_lib.BF16, w=_lib.F32, gate=None, gate_rows=0, gate_dtype=_lib.BF16, y=256, h=256, n=256, q=None,
             q_st=64, a=1.0, b=1.0, eps=1e-6):
        return lib.pisa_residual_norm(256, D, y, D, gate, D, gate_rows, gate_dtype, None, 0, 256, w, dtype, rows, D, a, b, eps, h, n,
                                      q, q_st, 256 if q else None, None, None)

    for kw, word in (({"rows": 0}, "nonempty"), ({"D": 0}, "nonempty"), ({"D": 16385}, "16384"), ({"dtype": 5}, "support"),
                     ({"w": _lib.F16}, "weights must be"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
                     ({"a": float("inf")}, "scales"), ({"gate": 256, "gate_rows": 3}, "divide"), ({"h": None}, "outputs"),
                     ({"gate": 256, "gate_dtype": _lib.F32}, "rows share"), ({"y": None, "gate": 256}, "belong to a branch"),
                     ({"n": None}, "outputs"), ({"q": 256}, "or in 8 bits"), ({"n": None, "q": 256, "q_st": 60}, "16 bytes"),
                     ({"rows": 1 << 31}, "too large")):
        refused(norm(**kw), word)
    refused(lib.pisa_residual_norm_bwd(None, 256, 256, 64, 256, 64, None, 0, 0, 0, None, 0, 256, _lib.F32, _lib.BF16, 4, 64, 1.0, 1.0,
                                       256, 256, 256, None, None, 256, 256, 16, None), "workspace")
    refused(lib.pisa_swiglu(256, 64, 256, 64, _lib.BF16, 4, 64, 256, 256, None, 64, 256, 256, None, 0, None, None), "come together")
    refused(lib.pisa_swiglu(256, 64, 256, 64, _lib.BF16, 4, 64, None, None, None, 64, None, None, None, 0, None, None), "written")
    refused(lib.pisa_swiglu(256, 64, 256, 64, _lib.BF16, 4, 40000, None, None, None, 0, None, None, 256, 40000, 256, None), "32768")
    refused(lib.pisa_swiglu_bwd(256, 64, None, 0, None, 0, None, None, 0, None, None, _lib.BF16, 4, 64, 256, 256, None, None),
            "required")
    refused(lib.pisa_quantize_int8(256, 64, _lib.BF16, 4, 64, 0, 8, 64, 256, None), "16 bytes")
    refused(lib.pisa_restore_int8(256, 64, None, _lib.BF16, 4, 64, 256, None), "required")

    def linear(T=4, K=64, O=8, x=256, x_st=64, x_dtype=_lib.S8, w_st=64, out=_lib.BF16, size=0, workspace=None, bias=None,
               bias_dtype=0):
        return lib.pisa_int8_linear(x, x_st, x_dtype, 256, 256, w_st, 256, bias, bias_dtype, out, T, K, O, 256, workspace, size, None)

    for kw, word in (({"T": 0}, "nonempty"), ({"K": 1 << 17}, "32 bits"), ({"O": 0}, "nonempty"), ({"x": 8}, "16 bytes"),
                     ({"x_st": 72}, "16 bytes"), ({"w_st": 48}, "overlap"), ({"out": 9}, "support"), ({"T": 1 << 31}, "too large"),
                     ({"workspace": 256, "size": 16}, "workspace"), ({"x_dtype": _lib.BF16, "T": 17}, "workspace"), ({"x_dtype": 4}, "support"),
                     ({"x_dtype": _lib.BF16, "workspace": 8, "size": 4096}, "16 bytes"), ({"bias": 256, "bias_dtype": _lib.F16}, "bias")):
        refused(linear(**kw), word)


def test_workspace_sizes_are_pure_host_functions():
    from nlogn_pisa_b200 import _lib

    lib = _lib.lib()
    assert lib.pisa_residual_norm_bwd_workspace_bytes(1, 64, 0) == 3 * 64 * 4
    assert lib.pisa_residual_norm_bwd_workspace_bytes(12, 64, 4) % (3 * 3 * 64 * 4) == 0
    assert lib.pisa_residual_norm_bwd_workspace_bytes(12, 64, 5) == -1
    assert lib.pisa_residual_norm_bwd_workspace_bytes(0, 64, 0) == -1
    assert lib.pisa_int8_linear_workspace_bytes(4, 64, 8, _lib.S8) == 256
    assert lib.pisa_int8_linear_workspace_bytes(4, 65, 8, _lib.BF16) == 256       # rounded by the product's kernel
    assert lib.pisa_int8_linear_workspace_bytes(17, 65, 8, _lib.BF16) == 512 + 17 * 80
    assert lib.pisa_int8_linear_workspace_bytes(1, 16385, 8, _lib.BF16) == 512 + 16400
    assert lib.pisa_int8_linear_workspace_bytes(4, 0, 8, _lib.S8) == -1
