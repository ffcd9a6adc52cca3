"""The operators at the tail of a decoding step on CPU tensors (the oracle math that
the device kernels are tested against): RMS norm with residual and 8-bit output,
int8 matrix product, rules on logits, against their definitions in 64 bits; and
what the entry points refuse."""

import pytest
import torch

from dsv4_flash_deployment_b200.ops import gemm as G
from dsv4_flash_deployment_b200.ops import logits as L
from dsv4_flash_deployment_b200.ops import norm as Q
from dsv4_flash_deployment_b200.ref import numerics as N

U = 2.0 ** -24          # half a step of fp32, relative


def test_pack_bits_round_trip():
    g = torch.Generator().manual_seed(0)
    for n in (1, 31, 32, 33, 100):
        b = torch.rand(3, n, generator=g) < 0.5
        w = N.pack_bits(b)
        assert w.dtype == torch.int32 and w.shape == (3, (n + 31) // 32)
        assert torch.equal(N.unpack_bits(w, n), b)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "mx8"])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_quant_cpu(fmt, residual):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 256, generator=g).to(torch.bfloat16)
    r = torch.randn(5, 256, generator=g).to(torch.bfloat16) if residual else None
    w = 1 + 0.1 * torch.randn(256, generator=g)
    got = Q.rms_norm_quant(x, w, 1e-6, fmt, residual=r)
    s = x.double() + (r.double() if residual else 0)
    y = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    v = Q.dequantize_rows(got[0], got[1], 5).double()
    # half a step of the code, then of bf16 (2^-8), and the fp32 arithmetic before (2^-17)
    if fmt == "i8":
        tol = got[1].double()[:, None] * 0.502 + v.abs() * 2 ** -8
    else:
        sc = got[1].double()[:, None] if fmt == "e4m3" else y.abs().amax(-1, keepdim=True) / 224
        tol = y.abs() * (2 ** -4 + 2 ** -8 + 2 ** -17) * 1.01 + sc * 2 ** -10
    assert ((v - y).abs() <= tol).all()
    if residual:
        assert ((got[2].double() - s).abs() <= s.abs() * 2 ** -8 * 1.001).all()


def test_rms_norm_quant_rows_with_nothing_finite():
    x = torch.zeros(4, 32)
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3] = 1.0
    q, s = Q.rms_norm_quant(x, torch.ones(32), 1e-20, "i8")
    assert s[0] > 0 and not q[0].any()
    assert torch.isnan(s[1]) and torch.isnan(s[2]) and not q[1:3].any()
    v = Q.dequantize_rows(q, s)
    assert torch.equal(v[0], torch.zeros(32, dtype=torch.bfloat16)) and torch.isnan(v[1:3]).all()
    assert torch.equal(v[3], torch.ones(32, dtype=torch.bfloat16))


def test_norm_refusals():
    x = torch.randn(2, 64)
    w = torch.ones(64)
    with pytest.raises(ValueError):
        Q.rms_norm_quant(x, w, 1e-6, "i4")
    with pytest.raises(ValueError):
        Q.quantize_rows(x, "fp8")
    for bad in (dict(x=x, w=w, eps=0.0), dict(x=x, w=w, eps=1e-6, fmt="mx8"), dict(x=x, w=torch.ones(63), eps=1e-6),
                dict(x=x, w=w.half(), eps=1e-6), dict(x=x, w=w, eps=1e-6, residual=x.half()),
                dict(x=x, w=w, eps=1e-6, residual_out=x.clone()),
                dict(x=torch.ones(1, 32784), w=torch.ones(32784), eps=1e-6)):
        kw = {k: v for k, v in bad.items() if k not in ("x", "w", "eps")}
        with pytest.raises(RuntimeError):
            Q.rms_norm_quant(bad["x"], bad["w"], bad["eps"], **kw)
    with pytest.raises(ValueError):
        Q.dequantize_rows(torch.zeros(2, 4), torch.ones(2))
    with pytest.raises(ValueError):
        Q.dequantize_rows(torch.zeros(2, 4, dtype=torch.int8), torch.ones(2), rows=3)


@pytest.mark.parametrize("t,n,k", [(1, 1, 1), (3, 5, 17), (4, 130, 300)])
def test_gemm_i8_cpu(t, n, k):
    g = torch.Generator().manual_seed(t + n)
    x = torch.randn(t, k, generator=g)
    w = torch.randn(n, k, generator=g)
    wq = G.I8Weight.from_float(w)
    assert wq.q.stride(0) % 16 == 0
    xq, xs = Q.quantize_rows(x)
    want = (xq.double() @ wq.q.double().t()) * xs.double()[:, None] * wq.scale.double()[None]
    for dt, half in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        out = G.gemm_i8(xq, xs, wq, out_dtype=dt)
        assert ((out.double() - want).abs() <= want.abs() * (half + 4 * U) * 1.001).all()
    assert torch.equal(G.linear_i8(x, wq), G.gemm_i8(xq, xs, wq))


def test_gemm_i8_refusals():
    w = G.I8Weight.from_float(torch.randn(4, 8))
    with pytest.raises(RuntimeError):
        G.gemm_i8(torch.zeros(2, 8), torch.ones(2), w)
    with pytest.raises(RuntimeError):
        G.gemm_i8(torch.zeros(2, 9, dtype=torch.int8), torch.ones(2), w)
    with pytest.raises(ValueError):
        G.I8Weight.from_quantized(torch.zeros(4, 8), torch.ones(4))
    with pytest.raises(ValueError):
        G.I8Weight.from_quantized(torch.zeros(4, 8, dtype=torch.int8), torch.ones(3))


def test_history_counts_prompt_and_output():
    h = L.TokenHistory.empty(2, 70, "cpu")
    i = lambda v: torch.tensor(v, dtype=torch.int32)
    h.add(i([3, 31, 63, 31, 69, 5]), i([0, 0, 0, 0, 1, -1]), i([0, 1, 0, 1, -1, 1]))
    seen = N.unpack_bits(h.seen, 70)
    assert seen[0].nonzero()[:, 0].tolist() == [3, 31, 63] and not seen[1].any()
    assert h.counts[0].nonzero()[:, 0].tolist() == [31] and int(h.counts[0, 31]) == 2
    with pytest.raises(RuntimeError):
        h.add(i([70]), i([0]), i([1]))
    h.reset(0)
    assert not h.seen.any() and not h.counts.any()
    for slot in (-1, 2):
        with pytest.raises(IndexError):
            h.reset(slot)


def test_rules_cpu_against_the_formula():
    v = 40
    lg = torch.tensor([[2.0, -2.0, 0.5, 3.0] + [0.0] * (v - 4), [1.0] * v])
    h = L.TokenHistory.empty(1, v, "cpu")
    i = lambda x: torch.tensor(x, dtype=torch.int32)
    h.add(i([0, 1, 1, 2]), i([0, 0, 0, 0]), i([1, 1, 1, 0]))
    r = L.RowRules().penalties(i([0, -1]), torch.tensor([2.0, 2.0]), torch.tensor([0.25, 9.0]), torch.tensor([0.5, 9.0]))
    r.biases(i([0, 3, 4]), i([0, 3, 3, 7]), torch.tensor([1.0, 0.5, 0.25, float("-inf")]))
    allowed = torch.ones(1, v, dtype=torch.bool)
    allowed[0, 2] = False
    r.masks(i([-1, 0]), N.pack_bits(allowed))
    z = L.apply_logits_rules(lg.clone(), r, h)
    want0 = [2 / 2 - 0.25 - 0.5 + 1.0, -2 * 2 - 0.5 - 0.5, 0.25, 3.75]
    assert torch.allclose(z[0, :4], torch.tensor(want0)) and not z[0, 4:].any()
    assert z[1, 7] == float("-inf") and z[1, 2] == float("-inf")
    assert torch.equal(z[1][[0, 1, 3, 4]], torch.ones(4))
    keep = lg.clone()
    out = torch.empty_like(lg)
    assert L.apply_logits_rules(lg, r, h, out=out) is out
    assert torch.equal(lg, keep) and torch.equal(out, z)


def test_rules_masked_places_hold_anything():
    lg = torch.tensor([[float("nan"), float("inf"), float("-inf"), 1.0]])
    r = L.RowRules().masks(torch.zeros(1, dtype=torch.int32), torch.tensor([[8]], dtype=torch.int32))
    assert L.apply_logits_rules(lg, r).tolist() == [[float("-inf")] * 3 + [1.0]]
    r.masks(torch.zeros(1, dtype=torch.int32), torch.tensor([[0]], dtype=torch.int32))
    assert L.apply_logits_rules(torch.ones(1, 4), r).tolist() == [[float("-inf")] * 4]


def test_rules_refusals():
    i = lambda x: torch.tensor(x, dtype=torch.int32)
    one = torch.ones(1)
    r = L.RowRules().penalties(i([0]), one, one, one)
    with pytest.raises(ValueError):
        L.apply_logits_rules(torch.zeros(1, 8), r)
    with pytest.raises(RuntimeError):
        L.apply_logits_rules(torch.zeros(1, 9), r, L.TokenHistory.empty(1, 8, "cpu"))
    with pytest.raises(RuntimeError):
        L.apply_logits_rules(torch.zeros(1, 8), L.RowRules().penalties(i([1]), one, one, one),
                             L.TokenHistory.empty(1, 8, "cpu"))
    with pytest.raises(RuntimeError):
        L.apply_logits_rules(torch.zeros(1, 40), L.RowRules().masks(i([0]), i([[1]])))
    with pytest.raises(RuntimeError):
        L.apply_logits_rules(torch.zeros(1, 8), L.RowRules().masks(i([1]), i([[1]])))
