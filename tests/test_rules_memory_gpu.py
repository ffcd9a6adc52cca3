"""The engine's buffers for the rules on logits exist before the first request."""

import pytest

from test_rules_engine_gpu import _engine, _prompts
from test_model_gpu import small_v4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [True, False])
def test_buffers_are_there_before_the_first_rule(graphs):
    cfg = small_v4()
    eng = _engine(cfg, use_graphs=graphs)
    before = [t.data_ptr() for t in eng.model.rules.tensors()]
    reqs = [eng.add_request(p, 4, ignore_eos=True, presence_penalty=1e6, logit_bias={i: -5.0, 9: float("-inf")},
                            allowed_token_ids=range(100 + i)) for i, p in enumerate(_prompts(cfg))]
    while not all(r.finished for r in reqs):
        eng.step()
    assert [t.data_ptr() for t in eng.model.rules.tensors()] == before
    for i, r in enumerate(reqs):
        assert len(set(r.output)) == 4 and max(r.output) < 100 + i and 9 not in r.output
    eng.check_errors()
