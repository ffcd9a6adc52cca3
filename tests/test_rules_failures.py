"""Requests whose grammar cannot say what may follow: no token is taken for them, the
request ends with its error, and everybody else goes on (CPU oracle step)."""

import asyncio

import numpy as np
import pytest

from dsv4_flash_deployment_b200.engine.config import EngineConfig
from dsv4_flash_deployment_b200.engine.dist_engine import _local_step
from dsv4_flash_deployment_b200.models.sampling import AllowedTokens, NothingAllowed, TokenRules, token_words
from dsv4_flash_deployment_b200.serving.engine_loop import EngineLoop, GenParams
from dsv4_flash_deployment_b200.serving.launch import build_local_engine

from test_rules_engine import P, _engine, _run


class FailsAfter:
    """Any token, until ``n`` of them are there."""

    def __init__(self, n):
        self.n = n

    def mask(self, output):
        if len(output) >= self.n:
            raise KeyError("no such state")
        return None


class WrongWords:
    def mask(self, output):
        return np.zeros(64, np.int64)


def _idle(eng):
    return eng.sched.idle and eng.sched.slots.n_free == eng.sched.max_seqs


@pytest.mark.parametrize("n,new", [(0, 1), (0, 6), (2, 3), (2, 6)])
def test_no_token_is_taken_where_the_grammar_fails(n, new):
    eng = _engine()
    other = eng.add_request(P, 8, ignore_eos=True, logprobs=2)
    bad = eng.add_request(P[:7], new, ignore_eos=True, grammar=FailsAfter(n), logprobs=1)
    events = []
    while not all(r.finished for r in (bad, other)):
        events += eng.step()
    assert len(bad.output) == n == len(bad.logprobs) == sum(r is bad and t is not None for r, t in events)
    assert bad.finish_reason == "cancelled" and "KeyError" in bad.error
    alone = _engine()
    want = alone.add_request(P, 8, ignore_eos=True, logprobs=2)
    _run(alone, [want])
    assert other.output == want.output and other.error is None and len(other.logprobs) == 8
    assert other.logprobs == want.logprobs and _idle(eng)


def test_nothing_else_to_run():
    """The failing request is the step's only one: no model step runs, and the request is reported."""
    eng = _engine()
    bad = eng.add_request(P, 4, grammar=WrongWords())
    events = eng.step()
    while not bad.finished:
        events += eng.step()
    assert [(r is bad, t) for r, t in events][-1] == (True, None) and not bad.output
    assert "int32 words" in bad.error and _idle(eng)


@pytest.mark.parametrize("grammar", [FailsAfter(0), FailsAfter(1), WrongWords()])
def test_generate_raises(grammar):
    eng = _engine()
    with pytest.raises(RuntimeError, match="grammar"):
        eng.generate([P, P[:5]], 1 if not isinstance(grammar, FailsAfter) else 3, grammar=grammar)
    assert _idle(eng) and len(eng.generate([P], 2, ignore_eos=True)[0]) == 2


def test_the_stream_ends_with_the_error():
    eng = _engine()
    loop = EngineLoop(eng).start()

    async def one(params):
        s = loop.submit(P, params)
        got = []
        while True:
            got.append(await asyncio.wait_for(s.q.get(), 60))
            if got[-1][0] != "token":
                return got

    async def go():
        return await asyncio.gather(one(GenParams(5, ignore_eos=True, rules={"grammar": FailsAfter(2)})),
                                    one(GenParams(5, ignore_eos=True)))
    try:
        bad, good = asyncio.run(go())
    finally:
        loop.stop()
    assert [k for k, _ in bad] == ["token", "token", "error"] and "KeyError" in bad[-1][1]
    assert [k for k, _ in good] == ["token"] * 5 + ["done"] and loop.healthy
    assert loop.stats["failed"] == 1 and loop.stats["finished"] == 1


def test_other_ranks_report_the_error():
    eng = build_local_engine(EngineConfig(device="cpu", model="toy-v4", max_seqs=3, max_batched_tokens=48, chunk_size=16,
                                          max_model_len=96), extra_slots=1)
    ids, got = {}, []
    msg = {"adds": [(7, 0, P, 6, True, (), 0.0, {"grammar": FailsAfter(1)})], "cancels": [], "any_work": True,
           "stop": False}
    for _ in range(8):
        got += _local_step(eng, msg, 0, ids, 3)
        msg = dict(msg, adds=[])
    toks = [e for e in got if e[1] is not None]
    ends = [e for e in got if e[2]]
    assert len(toks) == 1 and len(ends) == 1
    gid, tok, fin, reason, lp, error = ends[0]
    assert gid == 7 and tok is None and reason == "cancelled" and "KeyError" in error


class NotToBeSent:
    """Holds what cannot be pickled."""

    def __init__(self):
        self.f = lambda output: None

    def mask(self, output):
        return self.f(output)


class NotToBeReceived:
    """Pickles, but cannot be made again from its pickle."""

    def __reduce__(self):
        return (_refuse, ())

    def mask(self, output):
        return None


class OnlyOnRankZero:
    """A rank other than the first cannot make it from its pickle."""

    def __init__(self, rank=0):
        if rank != 0:
            raise ImportError("not here")

    def __reduce__(self):
        return (_made_where, ())

    def mask(self, output):
        return None


_RANK = [0]


def _made_where():
    return OnlyOnRankZero(_RANK[0])


def _refuse():
    raise ImportError("not to be had")


def _rank_grammars(rank, world):
    import torch.distributed as dist

    from dsv4_flash_deployment_b200.engine.dist_engine import DistributedEngine, worker_loop
    from dsv4_flash_deployment_b200.models.sampling import AllowedTokens

    _RANK[0] = rank
    eng = build_local_engine(EngineConfig(device="cpu", model="toy-v4", max_seqs=2, max_batched_tokens=32, chunk_size=16,
                                          max_model_len=96), extra_slots=1)
    if rank != 0:
        return worker_loop(eng, dist.group.WORLD)
    de = DistributedEngine(eng, dist.group.WORLD)
    refused = 0
    for g in (NotToBeSent(), NotToBeReceived()):
        try:
            de.add_request(P, 3, grammar=g)
        except ValueError:
            refused += 1
    left = (len(de.pending_adds), sum(de.load), len(de.live))
    ok = [de.add_request(P, 3, ignore_eos=True, grammar=AllowedTokens([20 + i], eng.cfg.vocab_size)) for i in range(2)]
    lost = [de.add_request(P, 3, ignore_eos=True, grammar=OnlyOnRankZero()) for _ in range(2)]
    odd = [de.add_request(P, 2, ignore_eos=True, allowed_token_ids=iter([30])),
           de.add_request(P, 2, ignore_eos=True, logit_bias=zip(np.array([31]), np.array([1e30])),
                          presence_penalty=np.float32(-1))]
    while not all(r.finished for r in ok + lost + odd):
        de.step()
    again = de.generate([P], 2, ignore_eos=True)
    de.shutdown()
    return {"odd": [r.output for r in odd], "refused": refused, "left": left, "ok": [(r.rank, r.output, r.error) for r in ok], "loads": de.load,
            "lost": {r.rank: (len(r.output), r.finish_reason, r.error) for r in lost}, "again": len(again[0])}


def test_grammars_that_do_not_travel():
    """Refused when the request is added; one that only another rank cannot make ends its
    own request there and nothing else."""
    from dsv4_flash_deployment_b200.utils.launch import spawn

    res = spawn(_rank_grammars, 2, timeout_s=300)[0]
    assert res["refused"] == 2 and res["left"] == (0, 0, 0)
    assert sorted(res["ok"]) == [(0, [20] * 3, None), (1, [21] * 3, None)]
    assert res["lost"][0] == (3, "length", None)
    n, reason, error = res["lost"][1]
    assert n == 0 and reason == "cancelled" and "not here" in error
    assert res["odd"] == [[30, 30], [31, 31]]
    assert res["again"] == 2 and res["loads"] == [0, 0]


# ------------------------------------------------------- rows where nothing is left
NINF = float("-inf")


def test_an_allowed_list_that_is_wholly_banned_is_refused():
    eng = _engine()
    v = eng.cfg.vocab_size
    for kw in (dict(allowed_token_ids=[65], logit_bias={65: NINF}), dict(allowed_token_ids=[65], logit_bias={65: -1e39}),
               dict(allowed_token_ids=[5, 6], logit_bias={6: NINF, 5: NINF, 7: 1.0})):
        with pytest.raises(ValueError, match="banned"):
            eng.add_request(P, 3, **kw)
        with pytest.raises(ValueError):
            TokenRules.make(v, **kw)
    with pytest.raises(ValueError, match="words"):       # made for a smaller vocabulary
        TokenRules.make(v, grammar=AllowedTokens([2], 40), logit_bias={v - 1: NINF})
    with pytest.raises(ValueError, match="banned"):
        TokenRules.make(40, logit_bias={t: NINF for t in range(40)})
    # one of two is left, and a large finite value does not ban
    out = _run(eng, [eng.add_request(P, 3, ignore_eos=True, allowed_token_ids=[5, 6], logit_bias={5: NINF}),
                     eng.add_request(P, 3, ignore_eos=True, allowed_token_ids=[9], logit_bias={9: -1e30})])
    assert out == [[6] * 3, [9] * 3]


def test_banned_tokens_leave_the_mask():
    g = lambda w: type("G", (), {"mask": lambda s, o: np.array(w, np.uint32)})()
    r = TokenRules.make(70, logit_bias={3: NINF, 33: NINF, 34: 1.0, 1: -4e38}, grammar=g([0b1010, 0b110, 0]))
    assert r.words([], 70, 2).tolist() == [0, 0b100, 0]
    r = TokenRules.make(70, logit_bias={3: NINF, 33: NINF, 34: NINF, 1: NINF}, grammar=g([0b1010, 0b110, 1 << 6]))
    assert r.words([], 70, 2).tolist() == [4, 0, 0]           # the end of sequence; bit 70 is past the end
    for eos in (None, 3, -1, 70):
        with pytest.raises(NothingAllowed):
            r.words([], 70, eos)


class _Ends:
    """Token 40 once, then nothing."""

    def __init__(self, vocab):
        self.v = vocab

    def mask(self, output):
        return token_words([40], self.v) if not output else np.zeros((self.v + 31) // 32, np.int32)


@pytest.mark.parametrize("how", ["banned", "none"])
def test_the_request_ends_where_nothing_may_follow(how):
    """With no end of sequence to give, the output is complete without one."""
    eng = _engine()
    bias = {eng.eos_id: NINF} if how == "banned" else None
    if how == "none":
        eng.eos_id = None
    other = eng.add_request(P, 6, ignore_eos=True)
    r = eng.add_request(P, 6, ignore_eos=True, grammar=_Ends(eng.cfg.vocab_size), logit_bias=bias)
    _run(eng, [r, other])
    assert r.output == [40] and r.finish_reason == "stop" and r.error is None and len(other.output) == 6
    assert _idle(eng) and eng.generate([P], 3, grammar=_Ends(eng.cfg.vocab_size), logit_bias=bias) == [[40]]


@pytest.mark.parametrize("extra", [{}, dict(temperature=1.0, seed=3), dict(temperature=1.0, top_k=5), dict(logprobs=2)])
def test_penalties_that_leave_nothing_end_the_request(extra):
    """The one allowed token's logit goes to -inf in the penalty: nothing is sampled in its place."""
    eng = _engine()
    kw = dict(allowed_token_ids=[P[3]], frequency_penalty=3e38, ignore_eos=True, **extra)
    r, other = eng.add_request(P, 6, **kw), eng.add_request(P, 6, ignore_eos=True)
    _run(eng, [r, other])
    # counted once it is at -3e38, counted twice at -inf
    assert r.output == [P[3]] * 2 and "nothing" in r.error and r.finish_reason == "cancelled"
    assert len(r.logprobs) == (2 if "logprobs" in extra else 0) and len(other.output) == 6 and _idle(eng)


def test_speculative_decoding_takes_rules_that_do_nothing():
    from types import SimpleNamespace

    from dsv4_flash_deployment_b200.spec.serving import SpecServingEngine

    cfg = _engine().cfg
    eng = SpecServingEngine(SimpleNamespace(cfg=cfg, max_seqs=1, blk=4, open_rows=lambda: None), 96)
    eng.add_request(P, 4, repetition_penalty=1.0, frequency_penalty=None, logit_bias={})
    for kw in (dict(repetition_penalty=1.1), dict(allowed_token_ids=[1]), dict(logit_bias={1: 0.5})):
        with pytest.raises(ValueError, match="speculative"):
            eng.add_request(P, 4, **kw)
    with pytest.raises(TypeError):
        eng.add_request(P, 4, penalty=2.0)
