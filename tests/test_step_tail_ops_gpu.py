"""The operators at the tail of a decoding step on the GPU, against their definitions
in 64 bits: RMS norm with residual and 8-bit output, int8 matrix product, rules on
logits; the run of them together, captured and replayed; and what they refuse.

Tolerances are counted in roundings: half a step of fp32 is 2^-24 of the value, of
bf16 2^-8, of fp16 2^-11, of e4m3 2^-4."""

import pytest
import torch

from dsv4_flash_deployment_b200.ops import _ext
from dsv4_flash_deployment_b200.ops import gemm as G
from dsv4_flash_deployment_b200.ops import logits as L
from dsv4_flash_deployment_b200.ops import norm as Q
from dsv4_flash_deployment_b200.ops.layout import chunks_to_sf
from dsv4_flash_deployment_b200.ref import numerics as N

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
# y before its code: the sum of squares has under 100 rounded additions in a row, the
# root halves their 100 U, and six more roundings follow: under 64 U = 2^-18
E_Y = 2.0 ** -18


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _done():
    torch.cuda.synchronize()
    G.ErrorWord.check("cuda")


# ------------------------------------------------------------------------- norm
def _y64(x, w, eps, res):
    s = x.double() + (res.double() if res is not None else 0)
    y = s
    if w is not None:
        y = s / (s.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return s, y


def _check_norm(got, x, w, eps, fmt, res):
    t, d = x.shape
    s, y = _y64(x, w, eps, res)
    q, scale = got[0], got[1]
    if fmt == "mx8":
        sb = chunks_to_sf(scale, t, d // 32)
        b = y.view(t, d // 32, 32)
        amax = b.abs().amax(-1).clamp(min=1e-4)
        lo = torch.ceil(torch.log2(amax * (1 - 2 * E_Y) / 448)) + 127
        hi = torch.ceil(torch.log2(amax * (1 + 2 * E_Y) / 448)) + 127
        assert ((sb >= lo) & (sb <= hi)).all()
        sc = torch.exp2(sb.double() - 127)[..., None].expand(-1, -1, 32).reshape(t, d)
        v = q[:t].view(torch.float8_e4m3fn).double() * sc
        tol = y.abs() * (2.0 ** -4 + 2 * E_Y) + sc * 2.0 ** -10      # the smallest codes are 2^-9 apart
    else:
        top = 127 if fmt == "i8" else 448
        sc = y.abs().amax(-1).clamp(min=1e-30) / top
        assert ((scale.double() - sc).abs() <= sc * (E_Y + 4 * U)).all()
        v = q.double() * scale.double()[:, None]
        if fmt == "i8":    # half a code, and at most 127 codes times the error of y and of the scale
            tol = sc[:, None] * (0.5 + 127 * 3 * E_Y)
        else:
            tol = y.abs() * (2.0 ** -4 + 3 * E_Y) + sc[:, None] * 2.0 ** -10
    assert ((v - y).abs() <= tol).all(), float(((v - y).abs() - tol).max())
    if res is not None:
        half = HALF[x.dtype]
        assert ((got[2].double() - s).abs() <= s.abs() * (half + U) + (2.0 ** -25 if x.dtype == HF else 0)).all()
    # the values come back as the product of code and scale, rounded to bf16 once
    back = Q.dequantize_rows(q, scale, t)
    want = v.to(F32) if fmt == "mx8" else q.float() * scale[:, None]
    assert torch.equal(back, want.to(BF))


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "mx8"])
@pytest.mark.parametrize("t,d", [(1, 1), (2, 8), (1, 4096), (3, 33), (7, 128), (130, 1024), (5, 5003), (300, 5120),
                                 (300, 4224), (5, 6144), (5, 6272), (300, 8192), (9, 8200), (2, 16384), (2, 32768),
                                 (3, 32767)])
def test_norm_widths(t, d, fmt):
    if fmt == "mx8" and d % 128:
        d = -(-d // 128) * 128
    g = _gen(t * 31 + d)
    x = torch.randn(t, d, device="cuda", generator=g).to(BF)
    x[:, d // 2] *= 30
    res = (2 * torch.randn(t, d, device="cuda", generator=g)).to(BF)
    w = (1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(BF)
    got = Q.rms_norm_quant(x, w, 1e-6, fmt, residual=res)
    _done()
    _check_norm(got, x, w, 1e-6, fmt, res)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "mx8"])
@pytest.mark.parametrize("t,d,off", [(5003, 37, 0), (4097, 256, 1), (2500, 511, 0), (2369, 1024, 3), (1300, 256, 0),
                                     (2369, 512, 0), (1201, 1024, 0), (1200, 1536, 0)])
@pytest.mark.parametrize("dt,wt", [(BF, BF), (F32, F32)])
def test_norm_many_narrow_rows(t, d, off, dt, wt, fmt):
    """Rows that a warp each takes, on 16-byte boundaries and off them; two of them are not finite."""
    if fmt == "mx8" and d % 128:
        d = 128
    g = _gen(t + d)
    x = torch.randn(t, d + 8, device="cuda", generator=g).to(dt)[:, off:off + d]
    res = (2 * torch.randn(t, d, device="cuda", generator=g)).to(dt)
    w = (1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(wt)
    got = Q.rms_norm_quant(x, w, 1e-6, fmt, residual=res)
    _done()
    _check_norm(got, x, w, 1e-6, fmt, res)
    x[t - 1, d - 1], x[t // 2, 0] = float("nan"), float("inf")
    again = Q.rms_norm_quant(x, w, 1e-6, fmt, residual=res)
    v, want = (Q.dequantize_rows(*r[:2], t) for r in (again, got))
    _done()
    want[[t - 1, t // 2]] = float("nan")
    assert torch.equal(v.isnan(), want.isnan()) and torch.equal(v.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "mx8"])
@pytest.mark.parametrize("dt,wt", [(BF, BF), (BF, F32), (HF, HF), (HF, F32), (F32, F32)])
@pytest.mark.parametrize("res", [False, True])
def test_norm_types_strides_and_offsets(dt, wt, fmt, res):
    """Rows apart from each other, at 16-byte boundaries and off them."""
    t, d = 37, 640
    g = _gen(3)
    w = (1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(wt)
    for ld, off in ((d, 0), (d + 8, 0), (d + 8, 3), (d + 1, 1)):
        x = torch.randn(t, ld, device="cuda", generator=g).to(dt)[:, off:off + d] if off + d <= ld else None
        if x is None:
            continue
        r = torch.randn(t, ld, device="cuda", generator=g).to(dt)[:, :d] if res else None
        ro = torch.zeros(t, ld, device="cuda", dtype=dt) if res else None
        kw = dict(residual=r, residual_out=ro[:, :d]) if res else {}
        got = Q.rms_norm_quant(x, w, 1e-5, fmt, **kw)
        _done()
        _check_norm(got, x, w, 1e-5, fmt, r)
        if res and ld > d:
            assert not ro[:, d:].any()        # what lies between the rows stays
    got = Q.quantize_rows(x, fmt)
    _done()
    _check_norm(got, x, None, 0.0, fmt, None)


@pytest.mark.parametrize("fmt", ["i8", "mx8"])
def test_norm_residual_updated_in_place(fmt):
    g = _gen(5)
    x = torch.randn(70, 1024, device="cuda", generator=g).to(BF)
    r = torch.randn(70, 1024, device="cuda", generator=g).to(BF)
    w = torch.ones(1024, device="cuda", dtype=BF)
    want = Q.rms_norm_quant(x, w, 1e-6, fmt, residual=r)
    for into in ("residual", "x"):
        x1, r1 = x.clone(), r.clone()
        got = Q.rms_norm_quant(x1, w, 1e-6, fmt, residual=r1, residual_out=r1 if into == "residual" else x1)
        _done()
        assert torch.equal(got[0][:70], want[0][:70]) and torch.equal(got[2], want[2])
        assert torch.equal(x if into == "residual" else r, x1 if into == "residual" else r1)


@pytest.mark.parametrize("fmt", ["i8", "e4m3", "mx8"])
@pytest.mark.parametrize("d", [256, 384 + 128])
def test_norm_rows_of_nothing_and_of_everything(fmt, d):
    """Zeros under a tiny eps, the largest finite values, infinities and NaN."""
    x = torch.zeros(6, d, device="cuda")
    x[1] = 3e38
    x[2] = 1e25 * torch.arange(1, d + 1, device="cuda")
    x[3, d - 1] = float("inf")
    x[4, 0] = float("nan")
    x[5] = 1e-18 * torch.arange(1, d + 1, device="cuda")
    w = torch.linspace(0.5, 1.5, d, device="cuda")
    q, s = Q.rms_norm_quant(x, w, 1e-20, fmt)
    v = Q.dequantize_rows(q, s, 6).double()
    _done()
    fine = [0, 1, 2, 5]
    assert torch.isnan(v[3:5]).all() and torch.isfinite(v[fine]).all() and not v[0].any()
    _, y = _y64(x, w, 1e-20, None)
    tol = {"i8": y.abs().amax(-1, keepdim=True) * (0.502 / 127) + y.abs() * 2.0 ** -8,
           "e4m3": y.abs() * (2.0 ** -4 + 2.0 ** -7) + y.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10,
           "mx8": y.abs() * (2.0 ** -4 + 2.0 ** -7) + y.abs().amax(-1, keepdim=True) / 224 * 2.0 ** -10 + 1e-7}[fmt]
    assert ((v - y).abs() <= tol)[fine].all()
    # without the norm, finite rows stay finite whatever their squares are
    q, s = Q.quantize_rows(x.clamp(-1e30, 1e30), fmt)
    v = Q.dequantize_rows(q, s, 6)
    _done()
    assert torch.isnan(v[4]).all() and torch.isfinite(v[[0, 1, 2, 3, 5]]).all()


def test_norm_no_rows_and_padded_rows_stay():
    w = torch.ones(128, device="cuda", dtype=BF)
    q, s = Q.rms_norm_quant(torch.empty(0, 128, device="cuda", dtype=BF), w, 1e-6)
    assert q.shape == (0, 128) and s.shape == (0,)
    q, s = Q.empty_rows(3, 128, "mx8", "cuda")
    q.fill_(7)
    s.fill_(9)
    Q.rms_norm_quant(torch.ones(3, 128, device="cuda", dtype=BF), w, 1e-6, "mx8", q_out=q, scale_out=s)
    _done()
    assert (q[3:] == 7).all() and (chunks_to_sf(s, 128, 4)[3:] == 9).all()


def test_norm_refusals_on_the_device():
    x = torch.ones(2, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    bad = [dict(weight=w.half()), dict(weight=w[:63]), dict(weight=w.cpu()), dict(eps=0.0), dict(fmt="mx8"),
           dict(residual=x.half()), dict(residual=x[:1]), dict(residual_out=x.clone()),
           dict(q_out=torch.zeros(2, 64, device="cuda")), dict(scale_out=torch.zeros(3, device="cuda")),
           dict(residual=torch.ones(1, 64, device="cuda").expand(2, 64)), dict(x=x.double()), dict(x=x.t()),
           dict(x=torch.ones(1, 32776, device="cuda"), weight=torch.ones(32776, device="cuda")),
           dict(x=x[:, :0], weight=w[:0])]
    for b in bad:
        kw = dict(dict(x=x, weight=w, eps=1e-6), **b)
        with pytest.raises(RuntimeError):
            Q.rms_norm_quant(**kw)
    _done()


def test_norm_weights_that_are_not_finite():
    x = torch.randn(3, 256, device="cuda")
    for bad in (float("nan"), float("inf")):
        w = torch.ones(256, device="cuda")
        w[17] = bad
        for xx in (x, x[:, :255]):      # aligned and odd rows
            q, s = Q.rms_norm_quant(xx, w[: xx.shape[1]].contiguous(), 1e-6)
            assert torch.isnan(s).all() and not q.any()
    _done()


def test_norm_wrong_scale_chunks_are_refused():
    x = torch.ones(3, 256, device="cuda")
    q = torch.empty(128, 256, device="cuda", dtype=torch.uint8)
    for shape in ((1, 1, 512), (1, 4, 512), (1024,), (0, 2, 512)):
        with pytest.raises(RuntimeError):
            Q.quantize_rows(x, "mx8", q_out=q, scale_out=torch.empty(shape, device="cuda", dtype=torch.uint8))
        with pytest.raises(RuntimeError):
            Q.dequantize_rows(q, torch.empty(shape, device="cuda", dtype=torch.uint8), 3)
    _done()


# ------------------------------------------------------------------------- gemm
def _check_gemm(out, xq, xs, w):
    want = (xq.double() @ w.q.double().t()) * xs.double()[:, None] * w.scale.double()[None]
    half = HALF[out.dtype] if out.dtype != F32 else 0.0
    # the sum is exact; its conversion, the scales' product and the result round once each
    tol = want.abs() * (half + 4 * U) + (2.0 ** -25 if out.dtype == HF else 0.0)
    err = (out.double() - want).abs()
    assert (err <= tol).all(), float((err - tol).max())


def _i8_case(t, n, k, seed):
    g = _gen(seed)
    x = torch.randn(t, k, device="cuda", generator=g)
    if k <= Q.MAX_WIDTH:
        xq, xs = Q.quantize_rows(x)
    else:
        xw = G.I8Weight.from_float(x)
        xq, xs = xw.q, xw.scale
    w = G.I8Weight.from_float(torch.randn(n, k, device="cuda", generator=g) * k ** -0.5)
    return xq, xs, w


@pytest.mark.parametrize("t", [1, 2, 5, 8, 9, 17, 32, 33, 64, 65, 128, 129, 256, 257, 600])
@pytest.mark.parametrize("n,k", [(1, 1), (127, 33), (130, 129), (640, 1024), (2305, 1279)])
def test_gemm_i8_sizes(t, n, k):
    xq, xs, w = _i8_case(t, n, k, t + n)
    for dt in (BF, F32):
        out = torch.full((t, n), float("nan"), device="cuda", dtype=dt)
        assert G.gemm_i8(xq, xs, w, out) is out
        _done()
        _check_gemm(out, xq, xs, w)


@pytest.mark.parametrize("t,n,k", [(1, 1280, 5120), (4, 20000, 4096), (40, 512, 16384), (100, 384, 8192),
                                   (200, 4096, 512), (1100, 5120, 1280), (3000, 300, 256), (2, 3, 131071)])
def test_gemm_i8_larger(t, n, k):
    xq, xs, w = _i8_case(t, n, k, t)
    for dt in (BF, HF, F32):
        out = G.gemm_i8(xq, xs, w, out_dtype=dt)
        _done()
        _check_gemm(out, xq, xs, w)


@pytest.mark.parametrize("path", [G.I8_ROWS, G.I8_TILES, G.I8_PAIRS])
@pytest.mark.parametrize("t", [1, 2, 3, 40, 130, 300, 520])
@pytest.mark.parametrize("n,k", [(1, 1), (129, 33), (640, 4096), (1030, 1279), (20000, 520)])
def test_gemm_i8_every_kernel(t, n, k, path):
    """Each kernel at sizes that the rule would give to another: the same bits."""
    xq, xs, w = _i8_case(t, n, k, t + n)
    if path == G.I8_ROWS and t > 2:
        with pytest.raises(RuntimeError):
            G.gemm_i8(xq, xs, w, path=path)
        return
    for dt in (BF, F32):
        out = torch.full((t + 1, n), float("nan"), device="cuda", dtype=dt)
        G.gemm_i8(xq, xs, w, out[:t], path=path)
        _done()
        _check_gemm(out[:t], xq, xs, w)
        assert torch.isnan(out[t]).all() and torch.equal(out[:t], G.gemm_i8(xq, xs, w, out_dtype=dt))


@pytest.mark.parametrize("bn", [32, 64, 128, 256])
@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8])
def test_gemm_i8_tile_widths_and_splits(bn, splits):
    for t, n, k in ((1, 129, 1100), (70, 300, 1279), (290, 513, 4097)):
        xq, xs, w = _i8_case(t, n, k, t + n)
        for dt in (BF, F32):
            out = torch.full((t + 1, n), float("nan"), device="cuda", dtype=dt)
            G.gemm_i8(xq, xs, w, out[:t], path=G.I8_TILES, bn=bn, splits=splits)
            _done()
            _check_gemm(out[:t], xq, xs, w)
            assert torch.isnan(out[t]).all()


def test_gemm_i8_many_tiles_per_block():
    """More tiles than SMs, in both tensor-core kernels, twice in a row."""
    xq, xs, w = _i8_case(700, 12000, 640, 1)
    for path in (G.I8_TILES, G.I8_PAIRS):
        for _ in range(2):
            out = G.gemm_i8(xq, xs, w, out_dtype=F32, path=path)
        _done()
        _check_gemm(out, xq, xs, w)


@pytest.mark.parametrize("t", [1, 3, 40, 300])
def test_gemm_i8_extreme_codes(t):
    """The largest sums: every product 2^14 over the longest K."""
    k = 131071
    x = torch.full((t, k + 1), -128, device="cuda", dtype=torch.int8)[:, :k]
    q = torch.full((3, k), -128, dtype=torch.int8)
    q[1] = 127
    q[2, ::2] = 127
    w = G.I8Weight.from_quantized(q, torch.tensor([1.0, 0.5, 2.0]), "cuda")
    out = G.gemm_i8(x, torch.full((t,), 0.25, device="cuda"), w, out_dtype=F32)
    _done()
    _check_gemm(out, x, torch.full((t,), 0.25, device="cuda"), w)


@pytest.mark.parametrize("t", [1, 3, 77, 300])
def test_gemm_i8_strides_and_what_lies_between(t):
    g = _gen(t)
    n, k = 260, 200
    big = torch.randint(-127, 128, (t + 2, 512), device="cuda", generator=g).to(torch.int8)
    x = big[1:t + 1, 16:16 + k]
    wb = torch.randint(-127, 128, (n, 224), device="cuda", generator=g).to(torch.int8)
    w = G.I8Weight(wb[:, :k], torch.rand(n, device="cuda", generator=g))
    xs = torch.rand(t, device="cuda", generator=g)
    for dt in (BF, F32):
        for off in (0, 1):
            buf = torch.full((t + 1, n + 13), 7.0, device="cuda", dtype=dt)
            out = buf[:t, off:off + n]
            G.gemm_i8(x, xs, w, out)
            _done()
            _check_gemm(out, x, xs, w)
            assert (buf[t] == 7).all() and (buf[:, off + n:] == 7).all() and (buf[:, :off] == 7).all()


def test_gemm_i8_refusals_on_the_device():
    xq, xs, w = _i8_case(4, 8, 32, 1)
    z = torch.zeros(4, 33, device="cuda", dtype=torch.int8)
    out = torch.empty(4, 8, device="cuda")
    bad = [(xq.float(), xs, w, out), (xq, xs[:3], w, out), (xq, xs.double(), w, out), (xq[:, :31], xs, w, out),
           (z[:, :32], xs, w, out), (z[:, 1:], xs, w, out), (xq, xs, w, out[:, :7]), (xq, xs, w, out.double()),
           (xq, xs, w, torch.empty(8, 4, device="cuda").t()), (xq, xs, w, out.cpu()),
           (xq, xs, G.I8Weight(w.q, w.scale[:7]), out), (xq, xs, G.I8Weight(w.q.cpu(), w.scale), out),
           (xq[:, :0], xs, G.I8Weight(w.q[:, :0], w.scale), out),
           (torch.zeros(1, 131072, device="cuda", dtype=torch.int8), xs[:1],
            G.I8Weight(torch.zeros(8, 131072, device="cuda", dtype=torch.int8), w.scale), out[:1])]
    for a in bad:
        with pytest.raises(RuntimeError):
            G.gemm_i8(*a)
    assert G.gemm_i8(xq[:0], xs[:0], w).shape == (0, 8)
    _done()


# ------------------------------------------------------------------------ rules
def _rules_case(s, v, dt, seed, slots=None):
    g = _gen(seed)
    lg = (3 * torch.randn(s, v, device="cuda", generator=g)).to(dt)
    h = L.TokenHistory.empty(s + 2, v, "cuda")
    n = 40 * s
    ids = torch.randint(0, v, (n,), device="cuda", generator=g).int()
    sl = torch.randint(0, s + 2, (n,), device="cuda", generator=g).int()
    gen = torch.randint(-1, 2, (n,), device="cuda", generator=g).int()
    h.add(ids, sl, gen)
    ref = L.TokenHistory.empty(s + 2, v, "cpu")
    ref.add(ids.cpu(), sl.cpu(), gen.cpu())
    _done()
    assert torch.equal(h.seen.cpu(), ref.seen) and torch.equal(h.counts.cpu(), ref.counts)
    slots = torch.randperm(s + 2, device="cuda", generator=g)[:s].int()
    slots[s // 2] = -1 if s > 1 else slots[0]
    r = L.RowRules().penalties(slots, 0.7 + torch.rand(s, device="cuda", generator=g),
                               torch.rand(s, device="cuda", generator=g) - 0.3,
                               torch.rand(s, device="cuda", generator=g) - 0.3)
    per = [int(x) for x in torch.randint(0, min(v, 50) + 1, (s,), device="cuda", generator=g)]
    per[-1] = min(v, 50)
    rows = [torch.randint(0, v, (p,), device="cuda", generator=g).sort().values.int() for p in per]   # repeats too
    vals = 2 * torch.randn(sum(per), device="cuda", generator=g)
    if len(vals):
        vals[::7] = float("-inf")
    off = torch.tensor([0] + per, device="cuda").cumsum(0).int()
    r.biases(off, torch.cat(rows), vals)
    bits = torch.rand(s + 1, v, device="cuda", generator=g) < 0.7
    bits[0] = False
    mr = torch.randint(-1, s + 1, (s,), device="cuda", generator=g).int()
    words = torch.zeros(s + 1, (v + 31) // 32 + 3, device="cuda", dtype=torch.int32)
    words[:, : (v + 31) // 32] = N.pack_bits(bits)
    r.masks(mr, words)
    return lg, r, h, bits


def _check_rules(z, lg, r, h, bits, kinds="pbm"):
    """The formula in 64 bits; each of at most six fp32 roundings is 2^-24 of a partial result."""
    s, v = lg.shape
    x = lg.double()
    size = x.abs()
    if "p" in kinds and r.slots is not None:
        at = r.slots.clamp(min=0).long()
        use = (r.slots >= 0)[:, None]
        seen = N.unpack_bits(h.seen[at], v) & use
        c = (h.counts[at] * use).double()
        rep = r.repetition.double()[:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        p = r.frequency.double()[:, None] * c + r.presence.double()[:, None] * (c > 0)
        size = torch.maximum(size, x.abs()) + (r.frequency.double()[:, None] * c).abs() + r.presence.double().abs()[:, None]
        x = x - p
    if "b" in kinds and r.bias_off is not None:
        rows = torch.repeat_interleave(torch.arange(s, device="cuda"), (r.bias_off[1:] - r.bias_off[:-1]).long())
        b = torch.zeros(s, v, device="cuda", dtype=torch.float64)
        b.index_put_((rows, r.bias_ids.long()), r.bias_vals.double(), accumulate=True)
        mag = torch.zeros_like(b).index_put_((rows, r.bias_ids.long()), r.bias_vals.double().abs(), accumulate=True)
        x = torch.where(b == float("-inf"), b, x + b)
        size = size + torch.where(torch.isinf(mag), torch.zeros_like(mag), 8 * mag)
    if "m" in kinds and r.mask is not None:
        ok = bits[r.mask_rows.clamp(min=0).long()] | (r.mask_rows < 0)[:, None]
        x = torch.where(ok, x, torch.full_like(x, float("-inf")))
    out = z.double()
    gone = torch.isinf(x)
    assert torch.equal(out[gone], x[gone])
    half = HALF[lg.dtype] if lg.dtype != F32 else 0.0
    tol = 6 * U * size + x.abs() * half * (1 + 8 * U) + (2.0 ** -25 if lg.dtype == HF else 0.0)
    assert ((out - x).abs() <= tol)[~gone].all()


@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("s,v", [(1, 1), (2, 31), (1, 33), (3, 1000), (5, 4096), (2, 4097), (4, 32003), (3, 129280)])
def test_rules_sizes(s, v, dt):
    lg, r, h, bits = _rules_case(s, v, dt, s * 7 + v)
    out = torch.full_like(lg, float("nan"))
    assert L.apply_logits_rules(lg, r, h, out=out) is out
    _done()
    _check_rules(out, lg, r, h, bits)
    same = lg.clone()
    assert L.apply_logits_rules(same, r, h) is same
    _done()
    assert torch.equal(same, out)


@pytest.mark.parametrize("kinds", ["", "p", "b", "m", "pb", "pm", "bm"])
@pytest.mark.parametrize("ld,off", [(1000, 0), (1008, 4), (1001, 1)])
def test_rules_kinds_and_strides(kinds, ld, off):
    s, v = 6, 990
    lg0, full, h, bits = _rules_case(s, v, F32, 11)
    r = L.RowRules()
    if "p" in kinds:
        r.penalties(full.slots, full.repetition, full.frequency, full.presence)
    if "b" in kinds:
        r.biases(full.bias_off, full.bias_ids, full.bias_vals)
    if "m" in kinds:
        r.masks(full.mask_rows, full.mask)
    buf = torch.full((s, ld), 5.0, device="cuda")
    lg = buf[:, off:off + v]
    lg.copy_(lg0)
    ob = torch.full((s, ld), 6.0, device="cuda")
    out = ob[:, off:off + v]
    L.apply_logits_rules(lg, r, h if "p" in kinds else None, out=out)
    _done()
    assert torch.equal(lg, lg0)
    _check_rules(out, lg0, full, h, bits, kinds)
    L.apply_logits_rules(lg, r, h if "p" in kinds else None)
    _done()
    assert torch.equal(lg, out)
    for b, k in ((buf, 5.0), (ob, 6.0)):
        assert (b[:, :off] == k).all() and (b[:, off + v:] == k).all()


@pytest.mark.parametrize("in_place", [False, True])
def test_rules_infinities_and_nan(in_place):
    v = 4500
    lg = torch.zeros(2, v, device="cuda")
    lg[:, 0], lg[:, 1], lg[:, 2] = float("nan"), float("inf"), float("-inf")
    lg[:, 4200] = float("nan")
    bits = torch.ones(2, v, dtype=torch.bool, device="cuda")
    bits[0, [0, 1, 4200]] = False
    bits[1] = False
    r = L.RowRules().masks(i32([0, 1]), N.pack_bits(bits)).biases(i32([0, 1, 1]), i32([3]),
                                                                 torch.tensor([float("-inf")], device="cuda"))
    z = L.apply_logits_rules(lg, r, out=None if in_place else torch.empty_like(lg))
    _done()
    ninf = float("-inf")
    assert z[0, [0, 1, 2, 3, 4200]].tolist() == [ninf] * 5 and not z[0, 4:4200].any()
    assert (z[1] == ninf).all()
    out = torch.full((2,), -1, dtype=torch.int32, device="cuda")
    _ext.load().argmax_rows(z, 2, v, out, None, None, 0)
    assert out.tolist() == [4, 0]


def test_rules_bad_rows_are_reported_and_left_out():
    lg = torch.ones(2, 64, device="cuda")
    one = torch.ones(2, device="cuda")
    h = L.TokenHistory.empty(2, 64, "cuda")
    h.add(i32([1]), i32([0]), i32([1]))
    for r, hist in ((L.RowRules().penalties(i32([2, 0]), 2 * one, one, one), h),
                    (L.RowRules().masks(i32([1, 0]), i32([[1, 0]])), None)):
        z = L.apply_logits_rules(lg, r, hist, out=torch.empty_like(lg))
        assert torch.equal(z[0], lg[0]) and not torch.equal(z[1], lg[1])
        with pytest.raises(RuntimeError):
            G.ErrorWord.check("cuda")
    for ids, slots in (([64], [0]), ([-1], [0]), ([0], [2])):
        h.add(i32(ids), i32(slots), i32([1]))
        with pytest.raises(RuntimeError):
            G.ErrorWord.check("cuda")
    assert int(h.counts.sum()) == 1
    # offsets that point past the lists read nothing there
    r = L.RowRules().biases(i32([-5, 1, 900]), i32([3]), torch.tensor([1.0], device="cuda"))
    z = L.apply_logits_rules(lg, r, out=torch.empty_like(lg))
    _done()
    assert float(z[0, 3]) == 2.0 and float(z.sum()) == 129.0


def test_rules_refusals_on_the_device():
    lg = torch.zeros(2, 64, device="cuda")
    one = torch.ones(2, device="cuda")
    h = L.TokenHistory.empty(2, 64, "cuda")
    p = lambda *a: L.RowRules().penalties(*a)
    bad = [(lg, p(i32([0]), one, one, one), h, None), (lg, p(i32([0, 1]).long(), one, one, one), h, None),
           (lg, p(i32([0, 1]), one[:1], one, one), h, None), (lg, p(i32([0, 1]), one, one.cpu(), one), h, None),
           (lg, p(i32([0, 1]), one, one, one), L.TokenHistory.empty(2, 65, "cuda"), None),
           (lg, p(i32([0, 1]), one, one, one), L.TokenHistory(h.seen[:1], h.counts), None),
           (lg, L.RowRules().biases(i32([0, 1]), i32([0]), one[:1]), None, None),
           (lg, L.RowRules().biases(i32([0, 1, 1]), i32([0]), one), None, None),
           (lg, L.RowRules().masks(i32([0, 0]), i32([[1]])), None, None),
           (lg, L.RowRules().masks(i32([0]), i32([[1, 1]])), None, None),
           (lg.double(), L.RowRules(), None, None), (lg.t(), L.RowRules(), None, None),
           (lg, L.RowRules(), None, torch.empty(2, 63, device="cuda")), (lg, L.RowRules(), None, lg.half()),
           (lg[:1].expand(2, 64), L.RowRules(), None, None)]
    for a in bad:
        with pytest.raises(RuntimeError):
            L.apply_logits_rules(a[0], a[1], a[2], out=a[3])
    with pytest.raises(ValueError):
        L.apply_logits_rules(lg, p(i32([0, 1]), one, one, one))
    for a in ((i32([0]), i32([0, 1]), i32([1])), (i32([0]).long(), i32([0]), i32([1])), (i32([0]).cpu(), i32([0]), i32([1]))):
        with pytest.raises(RuntimeError):
            h.add(*a)
    assert L.apply_logits_rules(lg[:0], L.RowRules()).shape == (0, 64)
    _done()


# ------------------------------------------------------- offsets past 32 bits
def test_offsets_past_32_bits():
    """The last rows of arrays with more than 2^31 elements."""
    t, d = 270000, 8192
    x = torch.zeros(t, d, device="cuda", dtype=BF)
    x[-3:] = torch.randn(3, d, device="cuda", generator=_gen(1)).to(BF)
    w = torch.ones(d, device="cuda", dtype=BF)
    q, s = Q.rms_norm_quant(x, w, 1e-6)
    _done()
    _check_norm((q[-3:], s[-3:].contiguous()), x[-3:], w, 1e-6, "i8", None)
    wt = G.I8Weight(torch.ones(16, d, device="cuda", dtype=torch.int8), torch.ones(16, device="cuda"))
    out = G.gemm_i8(q, s, wt, out_dtype=F32)
    _done()
    _check_gemm(out[-3:], q[-3:], s[-3:], wt)
    y = Q.dequantize_rows(q, s)
    assert torch.equal(y[-3:], (q[-3:].float() * s[-3:, None]).to(BF))
    del x, q, y, out
    n = 129280
    xq, xs, wn = _i8_case(17000, n, 64, 2)
    out = G.gemm_i8(xq, xs, wn)
    _done()
    _check_gemm(out[-40:], xq[-40:], xs[-40:], wn)
    keep = out[-2:].clone()
    bits = torch.rand(1, n, device="cuda", generator=_gen(3)) < 0.5
    r = L.RowRules().masks(torch.zeros(17000, device="cuda", dtype=torch.int32), N.pack_bits(bits))
    L.apply_logits_rules(out, r)
    _done()
    assert torch.equal(out[-2:], torch.where(bits, keep, torch.full_like(keep, float("-inf"))))


# ---------------------------------------------------------------- all of them
class _Tail:
    """Residual stream -> norm -> int8 head -> rules -> token, on buffers of its own."""

    def __init__(self, s, d, v, seed):
        g = _gen(seed)
        self.s, self.v = s, v
        self.x = torch.randn(s, d, device="cuda", generator=g).to(BF)
        self.res = torch.randn(s, d, device="cuda", generator=g).to(BF)
        self.norm = (1 + 0.1 * torch.randn(d, device="cuda", generator=g)).to(BF)
        self.head = G.I8Weight.from_float(torch.randn(v, d, device="cuda", generator=g) * d ** -0.5)
        self.q, self.qs = Q.empty_rows(s, d, "i8", "cuda")
        self.rout = torch.empty_like(self.x)
        self.raw = torch.empty(s, v, device="cuda")
        self.z = torch.empty(s, v, device="cuda")
        self.ids = torch.zeros(s, device="cuda", dtype=torch.int32)
        self.scratch = torch.zeros(2 * 296 + s, device="cuda", dtype=torch.int32)
        self.h = L.TokenHistory.empty(s, v, "cuda")
        self.slots = torch.arange(s, device="cuda", dtype=torch.int32)
        self.gen = torch.ones(s, device="cuda", dtype=torch.int32)
        self.bits = torch.rand(s, v, device="cuda", generator=g) < 0.5
        one = torch.ones(s, device="cuda")
        self.rules = L.RowRules().penalties(self.slots, 1.5 * one, 0.5 * one, 0.25 * one)
        self.rules.masks(self.slots, N.pack_bits(self.bits))

    def step(self):
        Q.rms_norm_quant(self.x, self.norm, 1e-6, "i8", residual=self.res, residual_out=self.rout, q_out=self.q,
                         scale_out=self.qs)
        G.gemm_i8(self.q, self.qs, self.head, self.raw)
        L.apply_logits_rules(self.raw, self.rules, self.h, out=self.z)
        _ext.load().argmax_rows(self.z, self.s, self.v, self.ids, self.scratch, None, 0)
        self.h.add(self.ids, self.slots, self.gen)

    def check(self, before):
        _check_norm((self.q, self.qs, self.rout), self.x, self.norm, 1e-6, "i8", self.res)
        _check_gemm(self.raw, self.q, self.qs, self.head)
        _check_rules(self.z, self.raw, self.rules, before, self.bits)
        assert torch.equal(self.ids.long(), self.z.argmax(-1))
        after = before.counts.clone()
        after[torch.arange(self.s, device="cuda"), self.ids.long()] += 1
        assert torch.equal(after, self.h.counts)


@pytest.mark.parametrize("s,d,v", [(1, 512, 4000), (70, 1024, 1999)])
def test_tail_runs_captured_and_replayed(s, d, v):
    """Two graphs of two tails, replayed in turn on another stream with new inputs."""
    a, b = _Tail(s, d, v, 1), _Tail(s, d, v, 2)
    st = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(st):
        for x in (a, b):
            x.step()                                   # the first step runs eagerly
            st.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=st):
                x.step()
            graphs.append(gr)
        for k in range(3):
            kept = [L.TokenHistory(x.h.seen.clone(), x.h.counts.clone()) for x in (a, b)]
            for x in (a, b):
                x.x.copy_(torch.randn(s, d, device="cuda", generator=_gen(50 + k)))
            for gr in graphs:
                gr.replay()
            st.synchronize()
            for x, h in zip((a, b), kept):
                x.check(h)
    _done()


def test_tail_on_two_streams_at_once():
    a, b = _Tail(5, 256, 3001, 3), _Tail(5, 256, 3001, 4)
    kept = [L.TokenHistory(x.h.seen.clone(), x.h.counts.clone()) for x in (a, b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for x, st in ((a, s1), (b, s2)):
        with torch.cuda.stream(st):
            x.step()
    torch.cuda.synchronize()
    for x, h in zip((a, b), kept):
        x.check(h)
    _done()


def test_i8_weight_written_just_before_its_use():
    """The product sees codes that the kernel right before it wrote."""
    g = _gen(9)
    xq, xs, _ = _i8_case(3, 16, 512, 9)
    q, s = Q.empty_rows(3000, 512, "i8", "cuda")
    for k in range(5):
        f = torch.randn(3000, 512, device="cuda", generator=g)
        w = G.I8Weight(*Q.quantize_rows(f, "i8", q_out=q, scale_out=s))
        q2, s2 = Q.quantize_rows(torch.randn(3, 512, device="cuda", generator=g))
        out = G.gemm_i8(q2, s2, w, out_dtype=F32)
        _done()
        _check_gemm(out, q2, s2, w)
