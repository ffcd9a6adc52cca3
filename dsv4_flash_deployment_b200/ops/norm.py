"""RMS norm with the residual's addition and an 8-bit output, per-row 8-bit
quantization, and the way back (``csrc/norm_quant.cu``).

``fmt`` names the output: ``"i8"`` (int8, one fp32 scale per row: the operand of
:func:`.gemm.gemm_i8`), ``"e4m3"`` (float8_e4m3fn, one fp32 scale per row) or
``"mx8"`` (MXFP8: e4m3 bytes and ue8m0 scale chunks, the operand of
:func:`.gemm.gemm_mx`, as :func:`.gemm.quantize` returns them).

CPU tensors run the torch oracle math instead; CUDA tensors always run the
extension, on the current stream of their device.
"""

from __future__ import annotations

import torch

from ..ref import numerics as N
from . import _ext
from .layout import ceil_to, chunks_to_sf, sf_to_chunks

Q8_FMT = {"i8": 0, "e4m3": 1, "mx8": 2}
MAX_WIDTH = 32768     # a row stays in one thread block's registers or shared memory


def empty_rows(t: int, d: int, fmt: str, device) -> tuple[torch.Tensor, torch.Tensor]:
    """Uninitialized (codes, scales) of a ``[t, d]`` result.  Rows of ``"i8"`` /
    ``"e4m3"`` codes start on 16-byte boundaries, as the GEMM's TMA loads need."""
    if fmt == "mx8":
        tp = ceil_to(max(t, 1), 128)
        return (torch.empty(tp, d, dtype=torch.uint8, device=device),
                torch.empty(tp // 128, d // 128, 512, dtype=torch.uint8, device=device))
    dt = torch.int8 if fmt == "i8" else torch.float8_e4m3fn
    return torch.empty(t, ceil_to(d, 16), dtype=dt, device=device)[:, :d], torch.empty(t, device=device)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float, fmt: str = "i8",
                   residual: torch.Tensor | None = None, residual_out: torch.Tensor | None = None,
                   q_out: torch.Tensor | None = None, scale_out: torch.Tensor | None = None):
    """``y = rmsnorm(x + residual) * weight`` in fp32, quantized to ``fmt``.

    ``x`` [T, D] bf16, fp16 or fp32 with contiguous rows (any row stride), D from 1 to
    32768 (``"mx8"``: a multiple of 128); ``residual`` of x's type; ``weight`` [D] of
    x's type or fp32; ``eps`` at least 1e-30.  Returns ``(q, scale)``, or with a
    residual ``(q, scale, residual_out)`` with the sum rounded to x's type
    (``residual_out`` may be ``residual`` or ``x`` itself; the norm takes the sum
    before its rounding, except that a row whose squares or products with the weight
    pass fp32's range takes the rounded sum where it replaced an input).  ``q_out`` /
    ``scale_out``: buffers to write (:func:`empty_rows`); apart from ``residual_out``
    being an input whole, no output may overlap an input.  Rows that hold an infinity
    or NaN, or whose y passes fp32's range, come out as NaN (their scale is NaN)."""
    f = Q8_FMT.get(fmt)
    if f is None:
        raise ValueError(f"fmt {fmt!r}: one of {sorted(Q8_FMT)}")
    if q_out is None or scale_out is None:
        q0, s0 = empty_rows(x.shape[0], x.shape[1], fmt, x.device)
        q_out = q0 if q_out is None else q_out
        scale_out = s0 if scale_out is None else scale_out
    if residual is not None and residual_out is None:
        residual_out = torch.empty_like(x)
    if x.is_cuda:
        _ext.load().norm_quant(x, residual, residual_out, weight, eps, f, q_out, scale_out)
    else:
        _cpu(x, residual, residual_out, weight, eps, fmt, q_out, scale_out)
    return (q_out, scale_out) if residual is None else (q_out, scale_out, residual_out)


def quantize_rows(x: torch.Tensor, fmt: str = "i8", q_out: torch.Tensor | None = None,
                  scale_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``x`` [T, D] quantized to ``fmt`` without a norm: ``(q, scale)``."""
    f = Q8_FMT.get(fmt)
    if f is None:
        raise ValueError(f"fmt {fmt!r}: one of {sorted(Q8_FMT)}")
    if q_out is None or scale_out is None:
        q0, s0 = empty_rows(x.shape[0], x.shape[1], fmt, x.device)
        q_out = q0 if q_out is None else q_out
        scale_out = s0 if scale_out is None else scale_out
    if x.is_cuda:
        _ext.load().norm_quant(x, None, None, None, 0.0, f, q_out, scale_out)
    else:
        _cpu(x, None, None, None, 0.0, fmt, q_out, scale_out)
    return q_out, scale_out


def dequantize_rows(q: torch.Tensor, scale: torch.Tensor, rows: int | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """The bf16 values ``[rows, D]`` that codes and scales stand for (the format is
    told by q's type: int8, float8_e4m3fn, or uint8 for MXFP8)."""
    fmt = {torch.int8: "i8", torch.float8_e4m3fn: "e4m3", torch.uint8: "mx8"}.get(q.dtype)
    if fmt is None:
        raise ValueError(f"no 8-bit row format has codes of type {q.dtype}")
    t = q.shape[0] if rows is None else rows
    if t > q.shape[0]:
        raise ValueError(f"{t} rows of {q.shape[0]}")
    if out is None:
        out = torch.empty(t, q.shape[1], dtype=torch.bfloat16, device=q.device)
    elif out.shape[0] != t:
        raise ValueError(f"out has {out.shape[0]} rows, {t} expected")
    if q.is_cuda:
        _ext.load().dequant_rows(q, scale, Q8_FMT[fmt], out)
    elif fmt == "mx8":
        s = chunks_to_sf(scale, t, q.shape[1] // 32)
        v = N.act_dequant(q[:t].view(torch.float8_e4m3fn), s)
        bad = (s == 255).repeat_interleave(32, 1)
        out.copy_(torch.where(bad, torch.full_like(v, float("nan")), v))
    else:
        out.copy_(q[:t].float() * scale[:t, None])
    return out


def _cpu(x, residual, residual_out, weight, eps, fmt, q_out, scale_out) -> None:
    """The operator on CPU tensors, with the device binding's checks."""
    t, d = x.shape
    if not 1 <= d <= MAX_WIDTH:
        raise RuntimeError(f"width {d}: 1 to {MAX_WIDTH}")
    if weight is not None and eps < 1e-30:
        raise RuntimeError("eps must be at least 1e-30")
    if weight is not None and (weight.shape != (d,) or weight.dtype not in (x.dtype, torch.float32)):
        raise RuntimeError("weight: [D] of x's type or fp32 expected")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise RuntimeError("residual: x's shape and type expected")
    if residual is None and residual_out is not None:
        raise RuntimeError("residual_out without residual")
    if fmt == "mx8" and d % 128:
        raise RuntimeError("MXFP8 rows: width must be a multiple of 128")
    if weight is None:
        y = x.float()
    else:
        y, s = N.add_rms_norm(x, weight, eps, residual)
        if residual_out is not None:
            residual_out.copy_(s)
    if fmt != "mx8":
        q, sc = N.row_quant(y, fmt)
        q_out.copy_(q)
        scale_out.copy_(sc)
        return
    bad = ~torch.isfinite(y).all(-1)
    q, s = N.act_quant(torch.where(bad[:, None], torch.zeros_like(y), y))
    s[bad] = 255
    q_out[:t] = q.view(torch.uint8)
    scale_out.copy_(sf_to_chunks(s, scale_out.shape[0] * 128))
