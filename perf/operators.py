"""The operators at the tail of a decoding step: RMS norm with the residual's
addition and an 8-bit output, the matrix product of 8-bit integers, and the rules
on logits (penalties for repeated tokens, biases, grammar masks).

``run`` computes a case in its plain form with elementary torch operations, or,
where ``own`` is true, with the calls a user makes of this package.
"""

import math

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_pkg = None


def _ops():
    """The package's operator modules (only where ``own`` is true)."""
    global _pkg
    if _pkg is None:
        from dsv4_flash_deployment_b200.ops import gemm, logits, norm

        _pkg = (norm, gemm, logits)
    return _pkg


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # one decoding token before its first projection: launch latency counts
        _norm("norm: one token, 4096 wide", 1, 4096, "bf16", "bf16", "i8", True),
        # a full decode batch into the block-scaled GEMMs
        _norm("norm: decode batch, MXFP8", 512, 5120, "bf16", "bf16", "mx8", True),
        # a long prefill into an int8 projection
        _norm("norm: prefill, int8", 16384, 4096, "bf16", "f32", "i8", True),
        # an odd width and odd rows in 32 bits, no residual, one e4m3 scale a token
        _norm("norm: odd width, e4m3", 777, 5003, "f32", "f32", "e4m3", False),
        # one token through a small low-rank projection: latency
        _gemm("gemm: one token, low rank", 1, 1280, 5120, "bf16"),
        # the output head for one sequence: the weights' bytes
        _gemm("gemm: one token, output head", 1, 129280, 4096, "f32"),
        # the output head for a full decode batch
        _gemm("gemm: batch, output head", 512, 129280, 4096, "f32"),
        # an output projection during prefill: operations
        _gemm("gemm: prefill projection", 4096, 5120, 8192, "bf16"),
        # odd sizes in every dimension
        _gemm("gemm: odd sizes", 333, 2305, 1279, "bf16"),
        # one chat turn with penalties
        _rules("rules: one row, penalties", 1, 129280, "f32", 2000, 0, True, False, False),
        # a full decode batch, every rule, the raw logits kept for log-probabilities
        _rules("rules: batch, every rule", 512, 129280, "f32", 1500, 64, True, True, False),
        # structured output for a batch: grammar masks written over the logits
        _rules("rules: batch, grammar in place", 256, 32003, "bf16", 0, 0, False, True, True),
    ]


def _norm(name, rows, width, dtype, weight, fmt, residual):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "weight": weight, "fmt": fmt,
            "residual": residual}


def _gemm(name, rows, out, inner, dtype):
    return {"name": name, "op": "gemm", "rows": rows, "out": out, "inner": inner, "dtype": dtype}


def _rules(name, rows, vocab, dtype, history, bias, penalties, mask, in_place):
    return {"name": name, "op": "rules", "rows": rows, "vocab": vocab, "dtype": dtype, "history": history,
            "bias": bias, "penalties": penalties, "mask": mask, "in_place": in_place}


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("norm", "gemm", "rules"))
    if op == "norm":
        fmt = rng.choice(("i8", "e4m3", "mx8"))
        width = 128 * _log(rng, 1, 64) if fmt == "mx8" else _log(rng, 33, 8192)
        rows = _log(rng, 1, min(16384, 16384 * 4096 // width))
        dt = rng.choice(("bf16", "f16", "f32"))
        c = _norm("", rows, width, dt, rng.choice((dt, "f32")), fmt, rng.random() < 0.6)
    elif op == "gemm":
        out, inner = _log(rng, 100, 129280), _log(rng, 64, 8192)
        if out * inner > 129280 * 4096:
            out = 129280 * 4096 // inner
        rows = _log(rng, 1, max(1, min(8192, 512 * 129280 // out, 512 * 129280 * 4096 // (out * inner))))
        c = _gemm("", rows, out, inner, rng.choice(("bf16", "f16", "f32")))
    else:
        vocab = _log(rng, 1000, 131072)
        rows = _log(rng, 1, 512)
        in_place = rng.random() < 0.25       # masks only: run() is repeated on the same logits
        c = _rules("", rows, vocab, rng.choice(("f32", "bf16", "f16")), 0 if in_place else _log(rng, 1, 4000),
                   0 if in_place else rng.choice((0, _log(rng, 1, 300))), not in_place, in_place or rng.random() < 0.5,
                   in_place)
    del c["name"]
    return c


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        e = _DT[case["dtype"]].itemsize
        scales = n // 32 if case["fmt"] == "mx8" else 4 * case["rows"]
        return {"bytes": n * (e * (3 if case["residual"] else 1) + 1) + case["width"] * _DT[case["weight"]].itemsize +
                scales, "flops": 8 * n}
    if case["op"] == "gemm":
        t, n, k = case["rows"], case["out"], case["inner"]
        return {"bytes": t * k + n * k + 4 * (t + n) + t * n * _DT[case["dtype"]].itemsize, "flops": 2 * t * n * k}
    s, v = case["rows"], case["vocab"]
    e = _DT[case["dtype"]].itemsize
    words = 4 * ((v + 31) // 32)
    if case["in_place"]:       # the mask, and the half of the logits that it takes away
        return {"bytes": s * (words + e * v // 2), "flops": s * v}
    b = 2 * e * v + (words if case["mask"] else 0) + 8 * case["bias"]
    if case["penalties"]:
        b += words + 4 * min(v, case["history"] // 2)
    return {"bytes": s * b, "flops": 4 * s * v}


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {"norm": _prepare_norm, "gemm": _prepare_gemm, "rules": _prepare_rules}[case["op"]](case, g)


def _prepare_norm(case, g):
    t, d, dt = case["rows"], case["width"], _DT[case["dtype"]]
    x = torch.randn(t, d, device=DEV, generator=g)
    x[:, :: max(1, d // 7)] *= 12.0                       # outlier channels, as residual streams have
    st = {"case": case, "x": x.to(dt), "residual": None, "residual_out": None,
          "weight": (1.0 + 0.1 * torch.randn(d, device=DEV, generator=g)).to(_DT[case["weight"]])}
    if case["residual"]:
        st["residual"] = (3.0 * torch.randn(t, d, device=DEV, generator=g)).to(dt)
        st["residual_out"] = torch.empty(t, d, device=DEV, dtype=dt)
    # output buffers that a program keeps; rows of int8 operands start on 16-byte boundaries
    if case["fmt"] == "mx8":
        tp = -(-t // 128) * 128
        st["q"] = torch.empty(tp, d, device=DEV, dtype=torch.uint8)
        st["scale"] = torch.empty(tp // 128, d // 128, 512, device=DEV, dtype=torch.uint8)
    else:
        q = torch.zeros(t, -(-d // 16) * 16, device=DEV, dtype=torch.int8)[:, :d]
        st["q"] = q if case["fmt"] == "i8" else q.view(torch.float8_e4m3fn)
        st["scale"] = torch.empty(t, device=DEV)
    st["y"] = torch.empty(t, d, device=DEV, dtype=torch.bfloat16)
    return st


def _prepare_gemm(case, g):
    t, n, k = case["rows"], case["out"], case["inner"]
    ld = -(-k // 16) * 16
    w = torch.zeros(n, ld, device=DEV, dtype=torch.int8)
    ws = torch.empty(n, device=DEV)
    step = max(1, (1 << 26) // k)
    for r in range(0, n, step):                           # weights quantized a channel at a time
        f = torch.randn(min(step, n - r), k, device=DEV, generator=g) * k ** -0.5
        a = f.abs().amax(1)
        ws[r:r + step] = a / 127
        w[r:r + step, :k] = (f * (127 / a)[:, None]).round().to(torch.int8)
    f = torch.randn(t, k, device=DEV, generator=g)
    f[:, :: max(1, k // 7)] *= 6.0
    a = f.abs().amax(1)
    x = torch.zeros(t, ld, device=DEV, dtype=torch.int8)
    x[:, :k] = (f * (127 / a)[:, None]).round().to(torch.int8)
    return {"case": case, "x": x[:, :k], "xs": a / 127, "w": w[:, :k], "ws": ws,
            "out": torch.empty(t, n, device=DEV, dtype=_DT[case["dtype"]])}


def _prepare_rules(case, g):
    s, v, h = case["rows"], case["vocab"], case["history"]
    dt = _DT[case["dtype"]]
    words = (v + 31) // 32
    st = {"case": case, "logits": (2.5 * torch.randn(s, v, device=DEV, generator=g)).to(dt), "history": None,
          "bias": None, "mask": None, "out": None if case["in_place"] else torch.empty(s, v, device=DEV, dtype=dt)}
    if case["penalties"]:
        # half of each history is the prompt; tokens repeat as text does (low ids often)
        u = torch.rand(s, h, device=DEV, generator=g)
        toks = (v * u ** 3).long().clamp_(max=v - 1)
        n_prompt = h - h // 2
        seen = torch.zeros(s, 32 * words, device=DEV, dtype=torch.bool)
        seen.scatter_(1, toks, True)
        counts = torch.zeros(s, v, device=DEV, dtype=torch.int32)
        gen = toks[:, n_prompt:]
        counts.scatter_add_(1, gen, torch.ones_like(gen, dtype=torch.int32))
        perm = torch.randperm(s, device=DEV, generator=g)      # batch row -> history slot
        inv = torch.empty_like(perm)
        inv[perm] = torch.arange(s, device=DEV)
        st["history"] = (_pack(seen)[inv].contiguous(), counts[inv].contiguous())
        st["slots"] = perm.int()
        st["tokens"], st["n_prompt"] = toks, n_prompt
        st["repetition"] = 1.0 + 0.3 * torch.rand(s, device=DEV, generator=g)
        st["frequency"] = 0.5 * torch.rand(s, device=DEV, generator=g)
        st["presence"] = 0.5 * torch.rand(s, device=DEV, generator=g)
    if case["bias"]:
        b = min(case["bias"], v)
        ids = torch.rand(s, v, device=DEV, generator=g).topk(b, 1).indices.sort(1).values
        st["bias"] = (torch.arange(0, s * b + 1, b, device=DEV, dtype=torch.int32), ids.reshape(-1).int().contiguous(),
                      4.0 * torch.randn(s * b, device=DEV, generator=g))
    if case["mask"]:
        allowed = torch.rand(s, 32 * words, device=DEV, generator=g) < 0.5
        st["mask"] = (torch.arange(s, device=DEV, dtype=torch.int32).flip(0).contiguous(), _pack(allowed))
    return st


def _pack(bits):
    """Truth values [S, 32 W] -> words [S, W], bit j of word i = entry 32 i + j."""
    s, n = bits.shape
    w = (bits.view(s, n // 32, 32).long() << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _unpack(words, n):
    b = (words[:, :, None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return b.view(words.shape[0], -1)[:, :n] != 0


# --------------------------------------------------------------------- one pass
def run(state):
    return {"norm": _run_norm, "gemm": _run_gemm, "rules": _run_rules}[state["case"]["op"]](state)


EPS = 1e-6


def _run_norm(st):
    fmt, t = st["case"]["fmt"], st["case"]["rows"]
    if own:
        norm = _ops()[0]
        got = norm.rms_norm_quant(st["x"], st["weight"], EPS, fmt, residual=st["residual"],
                                  residual_out=st["residual_out"], q_out=st["q"], scale_out=st["scale"])
        out = {"y": norm.dequantize_rows(got[0], got[1], t, out=st["y"])}
        if fmt != "mx8":
            out["scale"] = got[1]
        if st["residual"] is not None:
            out["residual"] = got[2]
        return out
    s = st["x"].float()
    out = {}
    if st["residual"] is not None:
        s = s + st["residual"].float()
        out["residual"] = s.to(st["x"].dtype)
    y = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS) * st["weight"].float()
    if fmt == "mx8":
        b = y.view(t, -1, 32)
        _, e = torch.frexp(b.abs().amax(-1, keepdim=True).clamp_min(1e-4) / 448.0 * (1 - 2.0 ** -24))
        sc = torch.exp2(e.float())                        # the power of two at or above amax / 448
        out["y"] = ((b / sc).clamp(-448, 448).to(torch.float8_e4m3fn).float() * sc).view(t, -1).to(torch.bfloat16)
        return out
    top = 127.0 if fmt == "i8" else 448.0
    sc = y.abs().amax(-1, keepdim=True).clamp_min(1e-30) / top
    q = (y / sc).round().clamp(-127, 127) if fmt == "i8" else (y / sc).clamp(-448, 448).to(torch.float8_e4m3fn).float()
    out["y"] = (q * sc).to(torch.bfloat16)
    out["scale"] = sc[:, 0]
    return out


def _run_gemm(st):
    if own:
        gemm = _ops()[1]
        return gemm.gemm_i8(st["x"], st["xs"], gemm.I8Weight(st["w"], st["ws"]), st["out"])
    y = st["x"].float() @ st["w"].float().t()
    return (y * st["xs"][:, None] * st["ws"][None, :]).to(_DT[st["case"]["dtype"]])


def _run_rules(st):
    z0 = st["logits"]
    if own:
        lg = _ops()[2]
        rules = lg.RowRules()
        hist = None
        if st["history"] is not None:
            hist = lg.TokenHistory(*st["history"])
            rules.penalties(st["slots"], st["repetition"], st["frequency"], st["presence"])
        if st["bias"] is not None:
            rules.biases(*st["bias"])
        if st["mask"] is not None:
            rules.masks(*st["mask"])
        return lg.apply_logits_rules(z0, rules, hist, out=st["out"])
    v = z0.shape[1]
    z = z0.float()
    if st["history"] is not None:
        slots = st["slots"].long()
        seen = _unpack(st["history"][0][slots], v)
        cnt = st["history"][1][slots].float()
        rep = st["repetition"][:, None]
        z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
        z = z - st["frequency"][:, None] * cnt - st["presence"][:, None] * (cnt > 0)
    if st["bias"] is not None:
        off, ids, vals = st["bias"]
        rows = torch.repeat_interleave(torch.arange(len(z), device=z.device), (off[1:] - off[:-1]).long(),
                                       output_size=ids.numel())
        z = z.index_put((rows, ids.long()), vals, accumulate=True)
    if st["mask"] is not None:
        z = torch.where(_unpack(st["mask"][1][st["mask"][0].long()], v), z, float("-inf"))
    z = z.to(z0.dtype)
    return z0.copy_(z) if st["case"]["in_place"] else z


# ------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "gemm": _exact_gemm, "rules": _exact_rules}[case["op"]](case, st)


def _exact_norm(case, st):
    u = st["x"].double()
    out = {}
    if case["residual"]:
        u += st["residual"].double()
        out["residual"] = u
    n = u / (u.pow(2).sum(1, keepdim=True) / case["width"] + EPS).sqrt()
    n *= st["weight"].double()[None]
    del u
    if case["fmt"] == "mx8":
        m = n.abs().unflatten(1, (-1, 32)).max(-1).values.clamp(min=1e-4)
        step = torch.pow(2.0, torch.ceil(torch.log2(m / 448)))
        out["y"] = (_e4m3(n.unflatten(1, (-1, 32)) / step[..., None]) * step[..., None]).flatten(1)
        return out
    m = n.abs().max(1).values.clamp(min=1e-30)
    if case["fmt"] == "i8":
        out["scale"] = m / 127
        out["y"] = torch.round(n / out["scale"][:, None]) * out["scale"][:, None]
    else:
        out["scale"] = m / 448
        out["y"] = _e4m3(n / out["scale"][:, None]) * out["scale"][:, None]
    return out


def _e4m3(v):
    """Nearest value with 3 fraction bits and exponents down to 2^-6 (ties to even), at most 448."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.pow(2.0, e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_gemm(case, st):
    x = st["x"].double() * st["xs"].double()[:, None]
    out = torch.empty(case["rows"], case["out"], device=DEV, dtype=torch.float64)
    step = max(1, (1 << 28) // case["inner"])
    for r in range(0, case["out"], step):
        out[:, r:r + step] = torch.mm(x, (st["w"][r:r + step].double() * st["ws"][r:r + step].double()[:, None]).t())
    return out


def _exact_rules(case, st):
    z = st["logits"].double()
    if case["penalties"]:
        for s in range(case["rows"]):                     # from the token lists, a row at a time
            toks = st["tokens"][s]
            every = torch.unique(toks)
            row = z[s]
            val = row[every]
            rep = float(st["repetition"][s])
            row[every] = torch.where(val > 0, val / rep, val * rep)
            ids, n = torch.unique(toks[st["n_prompt"]:], return_counts=True)
            row[ids] -= float(st["frequency"][s]) * n.double() + float(st["presence"][s])
    if case["bias"]:
        off, ids, vals = st["bias"]
        for s in range(case["rows"]):
            a, b = int(off[s]), int(off[s + 1])
            z[s].index_add_(0, ids[a:b].long(), vals[a:b].double())
    if case["mask"]:
        v = torch.arange(case["vocab"], device=DEV)
        rows, words = st["mask"]
        for s in range(case["rows"]):
            w = words[rows[s].long()].long()
            z[s][(torch.bitwise_right_shift(w[v // 32], v % 32) & 1) == 0] = -math.inf
    return z
