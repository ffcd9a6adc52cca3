"""RMS norm with 8-bit output on CPU tensors where squares or products pass fp32's range."""

import pytest
import torch

from dsv4_flash_deployment_b200.ops import norm as Q


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "mx8"])
def test_rows_past_the_range_cpu(fmt):
    d = 256
    x = torch.ones(6, d)
    x[0] = 3e38
    x[1] = 1e25 * torch.arange(1, d + 1)
    x[2] = 2.0
    x[3, 17] = 100.0                        # its y is past the range
    x[4, 3] = float("inf")
    w = torch.linspace(0.5, 1.5, d)
    w[17] = 2.5e38
    got = Q.rms_norm_quant(x, w, 1e-6, fmt)
    v = Q.dequantize_rows(*got, 6).double()
    assert torch.isnan(v[3:5]).all() and torch.isfinite(v[[0, 1, 2, 5]]).all()
    y = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    # half a step of the code, then of bf16; the fp32 scale and y are off by under 2^-20
    top = y.abs().amax(-1, keepdim=True)
    tol = {"i8": top * (0.502 / 127) + y.abs() * 2.0 ** -8,
           "e4m3": y.abs() * (2.0 ** -4 + 2.0 ** -7) + top / 448 * 2.0 ** -10,
           "mx8": y.abs() * (2.0 ** -4 + 2.0 ** -7) + y.view(6, -1, 32).abs().amax(-1).repeat_interleave(32, 1) / 224 * 2.0 ** -10}
    assert ((v - y).abs() <= tol[fmt])[[0, 1, 2, 5]].all()
