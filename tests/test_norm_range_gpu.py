"""RMS norm with 8-bit output where a partial result leaves fp32's range: products of a
value and its weight, and squares.  Rows whose y is finite come out as the formula in
64 bits says, whichever kernel takes them; rows whose y is not come out as NaN."""

import pytest
import torch

from dsv4_flash_deployment_b200.ops import norm as Q
from dsv4_flash_deployment_b200.ops.layout import chunks_to_sf

from test_step_tail_ops_gpu import BF, E_Y, F32, U, _done, _gen, _y64

pytestmark = pytest.mark.gpu

TOP = torch.finfo(torch.float32).max
# (rows, width, first column in a wider buffer): a block's registers, with two groups of
# columns a thread, a warp a row, shared memory, and off 16-byte boundaries a block and a warp a row
SHAPES = [(6, 256, 0), (6, 6272, 0), (1302, 256, 0), (6, 8320, 0), (6, 640, 1), (2400, 512, 1)]


def _values(got, fmt, t, d):
    """What the codes stand for in 64 bits (NaN where the scale says so), and the step of a code."""
    q, scale = got[0], got[1]
    if fmt != "mx8":
        s = scale.double()[:, None].expand(t, d)
        return q.double() * s, s
    sb = chunks_to_sf(scale, t, d // 32)
    s = torch.exp2(sb.double() - 127)
    s[sb == 255] = float("nan")
    s = s.repeat_interleave(32, 1)
    return q[:t].view(torch.float8_e4m3fn).double() * s, s


def _check(got, x, w, eps, fmt, res=None):
    t, d = x.shape
    _, y = _y64(x, w, eps, res)
    v, s = _values(got, fmt, t, d)
    fine = (y.abs() <= TOP).all(-1)
    assert torch.isnan(v[~fine]).all() and not got[0][:t][~fine].view(torch.uint8).any()
    v, s, y = v[fine], s[fine], y[fine]
    if fmt == "i8":      # half a code, and 127 codes times the error of y and of the scale
        tol = s * (0.5 + 127 * 3 * E_Y)
    else:                # half a step of e4m3, or of its smallest codes
        tol = y.abs() * (2.0 ** -4 + 3 * E_Y) + s * 2.0 ** -10
    assert ((v - y).abs() <= tol).all()
    if fmt != "mx8":
        want = y.abs().amax(-1, keepdim=True).clamp(min=1e-30) / (127 if fmt == "i8" else 448)
        assert ((s - want).abs() <= want * (E_Y + 4 * U)).all()
    return fine


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "mx8"])
@pytest.mark.parametrize("t,d,off", SHAPES)
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("eps", [1e-6, 4.0])
def test_products_past_the_range(t, d, off, dt, eps, fmt):
    g = _gen(d)
    w = torch.rand(d, device="cuda", generator=g) + 0.5
    w[17], w[d - 9] = 2.5e38, 1e38
    sign = 1.0 - 2.0 * (torch.rand(d, device="cuda", generator=g) < 0.5).float()
    mix = torch.linspace(0.5, 2.0, d, device="cuda")
    mix[17] = 1e-30
    peak = torch.ones(d, device="cuda")
    peak[17] = 100.0                                       # its y is past the range
    kinds = torch.stack([2 * sign, 1.5 * sign, 3e38 * sign, peak, mix, 1e-3 * sign])
    x = torch.zeros(t, d + 8, device="cuda", dtype=dt)[:, off:off + d]
    x.copy_(kinds.repeat(t // 6, 1))
    w = w.to(dt)
    got = Q.rms_norm_quant(x, w, eps, fmt)
    _done()
    fine = _check(got, x, w, eps, fmt)
    assert fine[:6].tolist() == [True, True, True, False, True, True]


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "mx8"])
@pytest.mark.parametrize("t,d,off", SHAPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_weights_that_are_not_finite(t, d, off, bad, fmt):
    """Every row is NaN, all of it, as on the CPU; a weight that is fine again leaves no trace."""
    g = _gen(d + 1)
    x = torch.randn(t, d + 8, device="cuda", generator=g)[:, off:off + d]
    x[t - 1, d - 5] = 0.0                                  # 0 times infinity
    w = torch.ones(d, device="cuda")
    w[d - 5] = bad
    got = Q.rms_norm_quant(x, w, 1e-6, fmt)
    _done()
    assert not _check(got, x, w, 1e-6, fmt).any()
    cpu = Q.rms_norm_quant(x[-3:].cpu(), w.cpu(), 1e-6, fmt)
    assert torch.isnan(Q.dequantize_rows(*cpu, 3)).all()
    w[d - 5] = 0.5
    got = Q.rms_norm_quant(x, w, 1e-6, fmt)
    _done()
    assert _check(got, x, w, 1e-6, fmt).all()


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "mx8"])
@pytest.mark.parametrize("t,d,off", SHAPES)
def test_sum_before_its_rounding_past_the_range(t, d, off, fmt):
    """The norm takes x + residual before residual_out's rounding also where the squares
    overflow; residual_out in place of an input holds the rounded sum there, and the
    codes are then those of the rounded sum (documented)."""
    g = _gen(d + 2)
    x, res = ((1e25 * torch.randn(t, d + 8, device="cuda", generator=g)).to(BF)[:, off:off + d] for _ in range(2))
    w = torch.rand(d, device="cuda", generator=g) + 0.5
    got = Q.rms_norm_quant(x, w, 1e-6, fmt, residual=res)
    _done()
    assert _check(got, x, w, 1e-6, fmt, res).all()
    x1 = x.clone(memory_format=torch.contiguous_format)
    again = Q.rms_norm_quant(x1, w, 1e-6, fmt, residual=res, residual_out=x1)
    _done()
    assert torch.equal(x1, got[2])
    assert _check(again, x1, w, 1e-6, fmt).all()
