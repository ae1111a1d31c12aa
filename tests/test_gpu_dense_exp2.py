"""The polynomial 2^x of the full-attention backward against 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_polynomial_exp2(cuda_device):
    """Relative error 2.7e-6 of the fit and a few fp32 roundings (argument, five steps of Horner's rule, product)."""
    from nlogn_pisa_b200 import _lib

    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.cat([torch.linspace(-126.0, 100.0, 2_000_001, device="cuda"),
                   -40 * torch.rand(1_000_000, generator=gen, device="cuda"),
                   torch.tensor([0.0, -0.0, 0.5, -0.5, -0.49999997, 15.0, -126.0, 100.0], device="cuda")])
    y = torch.empty_like(x)
    _lib.check(_lib.lib().pisa_ex2_pair_selftest(_lib.ptr(x), _lib.ptr(y), x.numel(), _lib.stream_of(cuda_device)))
    exact = torch.exp2(x.double())
    assert float(((y.double() - exact).abs() / exact).max()) <= 2.72e-6 + 8 * 2.0 ** -24
    edge = torch.tensor([-127.0, -1e30, -math.inf, math.nan], device="cuda")
    y = torch.empty_like(edge)
    _lib.check(_lib.lib().pisa_ex2_pair_selftest(_lib.ptr(edge), _lib.ptr(y), 4, _lib.stream_of(cuda_device)))
    assert ((y[:3].double() / 2.0 ** -126 - 1).abs() <= 2.72e-6 + 8 * 2.0 ** -24).all() and y[3].isnan()
