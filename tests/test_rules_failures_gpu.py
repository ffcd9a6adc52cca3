"""Rules that leave a row nothing, on the device: the row's request ends, the rest go on."""

import pytest

from test_model_gpu import small_v4
from test_rules_engine_gpu import _engine, _prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("extra", [{}, dict(temperature=1.0, seed=3), dict(temperature=1.0, top_k=5, top_p=0.9),
                                   dict(logprobs=2)])
def test_penalties_that_leave_nothing_end_the_request(extra, graphs):
    cfg = small_v4()
    eng = _engine(cfg, use_graphs=graphs)
    ps = _prompts(cfg)
    alone = eng.generate([ps[1]], 6, ignore_eos=True)[0]
    r = eng.add_request(ps[0], 6, ignore_eos=True, allowed_token_ids=[ps[0][3]], frequency_penalty=3e38, **extra)
    other = eng.add_request(ps[1], 6, ignore_eos=True)
    while not (r.finished and other.finished):
        eng.step()
    # counted once the logit is near -3e38, counted twice it is -inf
    assert r.output == [ps[0][3]] * 2 and "nothing" in r.error and r.finish_reason == "cancelled"
    assert other.output == alone
    eng.check_errors()
