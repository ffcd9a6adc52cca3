"""Penalties, biases and grammars of requests through the engine and the server (CPU
oracle step): the generated tokens are the argmax of the rules' formula over the
oracle's own logits, whatever a request is batched with or how its prompt is cut."""

import asyncio

import numpy as np
import pytest
import torch

from dsv4_flash_deployment_b200.config import toy_v4_config
from dsv4_flash_deployment_b200.engine.config import EngineConfig
from dsv4_flash_deployment_b200.models.model import SeqChunk, StepMeta
from dsv4_flash_deployment_b200.models.sampling import MAX_BIAS, AllowedTokens, TokenRules, token_words
from dsv4_flash_deployment_b200.ref import numerics as N
from dsv4_flash_deployment_b200.serving.launch import build_local_engine

P = [3 + (7 * i) % 200 for i in range(20)]


def _engine(chunk=16, **kw):
    return build_local_engine(EngineConfig(device="cpu", model="toy-v4", max_seqs=3, max_batched_tokens=48,
                                           chunk_size=chunk, max_model_len=96, **kw))


def _run(eng, reqs):
    while not all(r.finished for r in reqs):
        eng.step()
    return [r.output for r in reqs]


def _formula(raw, prompt, out, rep=1.0, freq=0.0, pres=0.0, bias=(), allowed=None):
    z = raw.double().clone()
    for t in set(prompt) | set(out):
        z[t] = z[t] / rep if z[t] > 0 else z[t] * rep
    for t in set(out):
        z[t] -= freq * out.count(t) + pres
    for t, b in bias:
        z[t] += b
    if allowed is not None:
        keep = torch.zeros(len(z), dtype=torch.bool)
        keep[list(allowed)] = True
        z[~keep] = float("-inf")
    return z


@pytest.mark.parametrize("rules,kw", [
    (dict(repetition_penalty=1.8), dict(rep=1.8)),
    (dict(frequency_penalty=0.7, presence_penalty=0.4), dict(freq=0.7, pres=0.4)),
    (dict(repetition_penalty=0.5, presence_penalty=-0.3, logit_bias={5: 3.0, 9: float("-inf")}),
     dict(rep=0.5, pres=-0.3, bias=((5, 3.0), (9, float("-inf"))))),
    (dict(frequency_penalty=2.0, allowed_token_ids=[7, 8, 9, 10, 300]), dict(freq=2.0, allowed=(7, 8, 9, 10, 300))),
])
def test_tokens_follow_the_formula(rules, kw):
    eng = _engine()
    out = _run(eng, [eng.add_request(P, 8, ignore_eos=True, **rules)])[0]
    st = eng.model.ref.new_state(1)
    raw = None
    for t in P:
        raw, _ = eng.model.ref.step(torch.tensor([t]), st)
    for i, t in enumerate(out):
        z = _formula(raw[0].float()[: eng.cfg.vocab_size], P, out[:i], **kw)
        assert float(z[t]) >= float(z.max()) - 1e-5 * max(1.0, abs(float(z.max())))
        raw, _ = eng.model.ref.step(torch.tensor([t]), st)


def test_rules_hold_whatever_the_batch_and_the_chunks():
    rules = dict(repetition_penalty=1.5, presence_penalty=2000.0, logit_bias={11: 1000.0, 12: 500.0})
    eng = _engine()
    alone = _run(eng, [eng.add_request(P, 10, ignore_eos=True, **rules)])[0]
    plain = _run(eng, [eng.add_request(P, 10, ignore_eos=True)])[0]
    assert alone != plain
    for chunk in (3, 16):
        eng = _engine(chunk)
        for _ in range(2):       # the second time on slots that other requests have used
            reqs = [eng.add_request([9, 8, 7, 6] * 3, 12, ignore_eos=True, presence_penalty=1.0),
                    eng.add_request(P, 10, ignore_eos=True, **rules), eng.add_request(P, 10, ignore_eos=True)]
            outs = _run(eng, reqs)
            assert outs[1] == alone and outs[2] == plain


def test_presence_penalty_forbids_repeats_and_seeds_still_repeat():
    eng = _engine()
    out = _run(eng, [eng.add_request(P, 20, ignore_eos=True, presence_penalty=1e6)])[0]
    assert len(set(out)) == 20
    kw = dict(temperature=2.0, seed=5, presence_penalty=1e6, top_k=50)
    a, b = _run(eng, [eng.add_request(P, 12, ignore_eos=True, **kw) for _ in range(2)])
    assert a == b and len(set(a)) == 12


def test_logprobs_stay_those_of_the_raw_logits():
    eng = _engine()
    r0 = eng.add_request(P, 1, ignore_eos=True, logprobs=5)
    _run(eng, [r0])
    r = eng.add_request(P, 1, ignore_eos=True, logprobs=5, logit_bias={r0.output[0]: float("-inf")})
    _run(eng, [r])
    assert r.output[0] != r0.output[0] and r.logprobs[0]["top"] == r0.logprobs[0]["top"]


class _Counter:
    """Allows one token more than it was at last."""

    def __init__(self, vocab, end):
        self.v, self.end = vocab, end

    def mask(self, output):
        n = 40 + len(output)
        return token_words([n], self.v) if n < self.end else np.zeros((self.v + 31) // 32, np.int32)


def test_grammar_object_and_its_end():
    eng = _engine()
    v = eng.cfg.vocab_size
    r = eng.add_request(P, 20, grammar=_Counter(v, 45))
    _run(eng, [r])
    # where the grammar allows nothing, the end of sequence remains
    assert r.output == [40, 41, 42, 43, 44, eng.eos_id] and r.finish_reason == "stop"

    class Broken:
        def mask(self, output):
            if output:
                raise KeyError("x")

    bad, other = eng.add_request(P, 6, ignore_eos=True, grammar=Broken()), eng.add_request(P, 6, ignore_eos=True)
    _run(eng, [bad, other])
    assert bad.finish_reason == "cancelled" and "KeyError" in bad.error and len(other.output) == 6


def test_rules_are_checked():
    make = lambda **k: TokenRules.make(100, **k)
    assert make() is None and make(repetition_penalty=1, frequency_penalty=0, logit_bias={}) is None
    for bad in (dict(repetition_penalty=0), dict(repetition_penalty=-1), dict(repetition_penalty=float("nan")),
                dict(repetition_penalty=1e-60), dict(repetition_penalty=1e39), dict(frequency_penalty=float("inf")),
                dict(presence_penalty=float("nan")), dict(logit_bias={100: 1}), dict(logit_bias={-1: 1}),
                dict(logit_bias={1: float("nan")}), dict(logit_bias={1: float("inf")}), dict(logit_bias={1: 1, "1": 2}),
                dict(logit_bias={i: 1 for i in range(MAX_BIAS + 1)}), dict(allowed_token_ids=[]),
                dict(allowed_token_ids=[100]), dict(grammar=3),
                dict(allowed_token_ids=[1], grammar=AllowedTokens([2], 100))):
        with pytest.raises(ValueError):
            TokenRules.make(400 if len(bad.get("logit_bias", ())) > MAX_BIAS else 100, **bad)
    eng = _engine()
    with pytest.raises(TypeError):
        eng.add_request(P, 4, penalty=2)
    with pytest.raises(ValueError):
        eng.add_request(P, 4, logit_bias={eng.cfg.vocab_size: 1.0})
    eng.model.tp = object()
    with pytest.raises(ValueError):
        eng.add_request(P, 4, repetition_penalty=2.0)
    eng.add_request(P, 4, repetition_penalty=1.0)


def test_grammar_words_are_checked():
    g = lambda w: TokenRules(grammar=type("G", (), {"mask": lambda s, o: w})())
    assert g(None).words([], 40, 1) is None
    assert g(np.array([0, 1 << 8], np.uint32)).words([], 40, 1).tolist() == [2, 0]      # only bits past the end
    assert g(np.array([0, 1 << 8], np.uint32)).words([], 41, 1).tolist() == [0, 256]
    for w in (np.zeros(1, np.int32), np.zeros(2, np.int64), np.zeros((2, 2), np.int32)):
        with pytest.raises(ValueError):
            g(w).words([], 40, 1)
    assert N.unpack_bits(torch.from_numpy(token_words([0, 31, 39], 40).copy())[None], 40)[0].nonzero()[:, 0].tolist() == \
        [0, 31, 39]


def test_step_meta_rows_of_rules():
    cfg = toy_v4_config()
    pen, bia = TokenRules.make(500, presence_penalty=1.0), TokenRules.make(500, logit_bias={3: 1.0, 2: -1.0})
    words = token_words([1], cfg.vocab_size)
    m = StepMeta(cfg, [SeqChunk(0, 4, [5, 6, 7], True, rules=pen, n_prompt=6),
                       SeqChunk(1, 0, [9, 9], False, rules=pen, n_prompt=6), SeqChunk(2, 3, [1], True),
                       SeqChunk(3, 8, [4], True, rules=bia, n_prompt=2, mask=words)])
    assert m.ruled and m.resets == [1]
    assert m.hist.tolist() == [0, 0, 1, 0, 0, -1, -1]
    assert m.r_slot.tolist() == [0, -1, -1] and m.r_pres.tolist() == [1, 0, 0] and m.mask_rows.tolist() == [-1, -1, 0]
    assert m.bias_off.tolist() == [0, 0, 0, 2] and m.bias_ids.tolist() == [2, 3] and m.bias_vals.tolist() == [-1, 1]
    p = m.padded(64, 8, 7)
    assert p.ruled and len(p.hist) == p.T == 8 and p.hist[7] == -1
    assert len(p.r_slot) == len(p.mask_rows) == len(p.sample_rows) == 4 == len(p.bias_off) - 1
    assert p.r_slot[3] == -1 and p.mask_rows[3] == -1 and p.bias_off[4] == p.bias_off[3]
    assert StepMeta(cfg, [SeqChunk(0, 4, [5], True)]).key() != StepMeta(cfg, [SeqChunk(0, 4, [5], True, rules=pen)]).key()
    with pytest.raises(ValueError):
        StepMeta(cfg, [SeqChunk(0, 4, [5], True, True, rules=pen)])


def test_server_fields():
    from dsv4_flash_deployment_b200.serving import app as A

    body = {"repetition_penalty": 1.2, "frequency_penalty": 0, "presence_penalty": None,
            "logit_bias": {"5": -100}, "allowed_token_ids": [5, 6]}
    assert A._rules_fields(body) == {"repetition_penalty": 1.2, "logit_bias": {5: -100.0}, "allowed_token_ids": [5, 6]}
    assert A._rules_fields({}) == {}
    for bad in ({"logit_bias": [1]}, {"repetition_penalty": "x"}, {"logit_bias": {"a": 1}}):
        with pytest.raises((ValueError, TypeError)):
            A._rules_fields(bad)


def test_server_answers_with_rules():
    from aiohttp.test_utils import TestClient, TestServer

    from dsv4_flash_deployment_b200.serving.app import ServerState, build_app
    from dsv4_flash_deployment_b200.serving.engine_loop import EngineLoop
    from dsv4_flash_deployment_b200.serving.tokenizer import load_tokenizer

    eng = _engine()
    loop = EngineLoop(eng).start()
    try:
        async def go():
            st = ServerState(loop, load_tokenizer(None, eng.cfg), "m", 96)
            async with TestClient(TestServer(build_app(st))) as cl:
                ask = lambda **k: cl.post("/v1/completions", json={"prompt": P, "max_tokens": 4, "ignore_eos": True, **k})
                r = await ask(allowed_token_ids=[65], n=1)
                ok = await r.json()
                r2 = await ask(logit_bias={"100000": 1})
                r3 = await ask(repetition_penalty=0)
                return r.status, ok, r2.status, r3.status
        status, ok, bad, bad2 = asyncio.run(go())
    finally:
        loop.stop()
    assert status == 200 and bad == 400 and bad2 == 400
    assert ok["usage"]["completion_tokens"] == 4


def test_multi_rank_front_carries_the_rules():
    from dsv4_flash_deployment_b200.engine.dist_engine import _local_step

    eng, ref = _engine(), _engine()
    rules = dict(repetition_penalty=1.5, allowed_token_ids=list(range(30, 200)))
    want = _run(ref, [ref.add_request(P, 6, ignore_eos=True, **rules)])[0]
    ids, got = {}, []
    msg = {"adds": [(77, 0, P, 6, True, (), 0.0, rules)], "cancels": [], "any_work": True, "stop": False}
    for _ in range(30):
        for gid, tok, fin, reason, lp in _local_step(eng, msg, 0, ids, 3):
            assert gid == 77
            if tok is not None:
                got.append(tok)
        msg = dict(msg, adds=[])
        if len(got) == 6:
            break
    assert got == want
