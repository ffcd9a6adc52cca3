"""Requests whose grammar cannot say what may follow: no token is taken for them, the
request ends with its error, and everybody else goes on (CPU oracle step)."""

import asyncio

import numpy as np
import pytest

from dsv4_flash_deployment_b200.engine.config import EngineConfig
from dsv4_flash_deployment_b200.engine.dist_engine import _local_step
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
