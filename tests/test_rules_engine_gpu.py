"""Penalties, biases and grammars through the engine on the GPU (CUDA-graph replay
included), and the int8 output head: each sampled row's logits are the rules'
formula over the row's raw logits, and the token is their argmax."""

import pytest
import torch

from dsv4_flash_deployment_b200.engine.engine import Engine
from dsv4_flash_deployment_b200.ops import gemm as G
from dsv4_flash_deployment_b200.ops import norm as Q

from test_model_gpu import small_v4
from test_rules_engine import _formula
from test_step_tail_ops_gpu import U, _check_gemm, _check_norm

pytestmark = pytest.mark.gpu


def _engine(cfg, **kw):
    return Engine.build(cfg, "cuda", max_seqs=3, max_batched_tokens=64, max_seq_len=128, seed=3, chunk_size=24, **kw)


def _prompts(cfg, seed=2):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (30, 17, 44)]


def _check_rows(eng, rows, kinds):
    v = eng.cfg.vocab_size
    raw = eng.model._lp_raw[: len(rows)].cpu()
    z = eng.model.logits[: len(rows), :v].cpu()
    for i, (r, t) in enumerate(rows):
        kw = kinds[r.req_id]
        want = _formula(raw[i], r.prompt, r.output[:-1], **kw)
        gone = torch.isinf(want)
        assert torch.equal(torch.isinf(z[i]), gone)
        # at most six fp32 roundings of partial results no larger than this
        size = raw[i].double().abs() * max(kw.get("rep", 1), 1 / kw.get("rep", 1)) + \
            len(r.output) * abs(kw.get("freq", 0)) + abs(kw.get("pres", 0)) + sum(abs(b) for _, b in kw.get("bias", ()))
        assert ((z[i].double() - want).abs() <= 6 * U * size)[~gone].all()
        assert t == int(z[i].argmax())


@pytest.mark.parametrize("graphs", [True, False])
def test_rules_on_the_device(graphs):
    cfg = small_v4()
    eng = _engine(cfg, use_graphs=graphs)
    allowed = list(range(100, 300))
    kinds = [(dict(repetition_penalty=1.7, frequency_penalty=0.5), dict(rep=1.7, freq=0.5)),
             (dict(presence_penalty=-0.75, logit_bias={7: 2.0, 300: -1.5}), dict(pres=-0.75, bias=((7, 2.0), (300, -1.5)))),
             (dict(allowed_token_ids=allowed, presence_penalty=9.0), dict(allowed=allowed, pres=9.0))]
    for turn in range(2):        # the second time on slots with another request's history
        by_id, reqs = {}, []
        for p, (opts, kw) in zip(_prompts(cfg, turn), kinds):
            r = eng.add_request(p, 9, ignore_eos=True, logprobs=1, **opts)
            by_id[r.req_id] = kw
            reqs.append(r)
        n = 0
        while not all(r.finished for r in reqs):
            rows = [(r, t) for r, t in eng.step() if t is not None]
            if rows:
                _check_rows(eng, rows, by_id)
                n += len(rows)
        assert n == 27 and set(reqs[2].output) <= set(allowed) and len(set(reqs[2].output)) == 9
    eng.check_errors()
    if graphs:
        assert eng.stats["graph_captures"] > 0


def test_requests_without_rules_beside_ruled_ones():
    """A batch without rules keeps its tokens, before and after one with them."""
    cfg = small_v4()
    eng = _engine(cfg)
    ps = _prompts(cfg)
    before = eng.generate(ps, 8, ignore_eos=True)
    one = eng.add_request(ps[0], 8, ignore_eos=True, presence_penalty=1e6)
    rest = [eng.add_request(p, 8, ignore_eos=True) for p in ps[1:]]
    while not all(r.finished for r in [one] + rest):
        eng.step()
    assert [r.output for r in rest] == before[1:] and len(set(one.output)) == 8
    assert eng.generate(ps, 8, ignore_eos=True) == before
    eng.check_errors()


def test_ruled_sampling_repeats_with_a_seed():
    cfg = small_v4()
    eng = _engine(cfg)
    p = _prompts(cfg)[0]
    kw = dict(temperature=2.0, top_k=40, seed=9, frequency_penalty=1.0, logit_bias={3: 4.0})
    a = eng.generate([p], 8, ignore_eos=True, **kw)
    assert eng.generate([p], 8, ignore_eos=True, **kw) == a
    eng.check_errors()


def test_int8_output_head():
    cfg = small_v4()
    eng = _engine(cfg, head_int8=True)
    m = eng.model
    reqs = [eng.add_request(p, 5, ignore_eos=True, repetition_penalty=1.3 if i else 1.0)
            for i, p in enumerate(_prompts(cfg))]
    n = 0
    while not all(r.finished for r in reqs):
        rows = [(r, t) for r, t in eng.step() if t is not None]
        s = len(rows)
        if not s:
            continue
        n += s
        x, q, sc = m.u_sample[:s], m.u_sample_q[:s], m.u_sample_s[:s]
        _check_norm((q, sc), x, m.norm_w, cfg.rms_norm_eps, "i8", None)
        raw = G.gemm_i8(q, sc, m.head_q, out_dtype=torch.float32)
        _check_gemm(raw, q, sc, m.head_q)
        for i, (r, t) in enumerate(rows):
            if r is reqs[0]:      # no rule: the step's logits are the product itself
                assert torch.equal(m.logits[i], raw[i]) and t == int(raw[i, : cfg.vocab_size].argmax())
    eng.check_errors()
    assert n == 15
    # the codes stand for the bf16 head to half a step of each channel's scale
    w = m.head.double()
    assert ((m.head_q.q.double() * m.head_q.scale.double()[:, None] - w).abs() <=
            m.head_q.scale.double()[:, None] * 0.5001).all()
    got = Q.dequantize_rows(m.head_q.q, m.head_q.scale)
    assert got.shape == m.head.shape
