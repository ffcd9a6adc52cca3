"""Memory of the rules on logits: made when an engine is built, all of it or none."""

import pytest
import torch

from dsv4_flash_deployment_b200.config import toy_v4_config
from dsv4_flash_deployment_b200.models import model as M
from dsv4_flash_deployment_b200.models.model import DSV4Model, RuleBuffers, SeqChunk, StepMeta
from dsv4_flash_deployment_b200.models.sampling import MAX_BIAS, TokenRules, token_words


def _put(dst, arr):
    dst[: len(arr)].copy_(torch.from_numpy(arr))


def test_every_sequence_with_every_rule_fits():
    cfg = toy_v4_config()
    v, seqs = cfg.vocab_size, 3
    b = RuleBuffers(seqs, 8, 8, v, "cpu")
    allowed = [token_words([i, v - 1 - i], v) for i in range(seqs)]
    rules = [TokenRules.make(v, presence_penalty=1.0, logit_bias={t + i: -1.0 for t in range(min(MAX_BIAS, v - seqs))})
             for i in range(seqs)]
    m = StepMeta(cfg, [SeqChunk(i, 4, [5], True, rules=rules[i], n_prompt=4, mask=allowed[i]) for i in range(seqs)])
    m = m.padded(8, 8, seqs)
    b.upload(m, _put)
    r = b.rows(len(m.sample_rows))
    assert r.mask.shape == (seqs + 1, (v + 31) // 32)
    for i in range(seqs):
        assert r.mask[int(r.mask_rows[i])].tolist() == allowed[i].tolist()
        a, e = int(r.bias_off[i]), int(r.bias_off[i + 1])
        assert r.bias_ids[a:e].tolist() == [t for t, _ in rules[i].bias]
    assert b.masks.numel() == (seqs + 1) * ((v + 31) // 32) and b.bias_ids.numel() == (seqs + 1) * MAX_BIAS


def test_a_failed_allocation_leaves_nothing_half_made(monkeypatch):
    m = DSV4Model.__new__(DSV4Model)
    m.n_slots, m.max_tokens, m.max_sample, m.vocab, m.dev = 2, 8, 8, 100, torch.device("cpu")


    def fails(*a, **kw):
        raise torch.OutOfMemoryError("no memory")

    real = M.torch.zeros
    monkeypatch.setattr(M.torch, "zeros", lambda *s, **kw: real(*s, **kw) if len(s) == 2 else fails())
    with pytest.raises(torch.OutOfMemoryError):
        m.alloc_rules()
    assert m.rules is None
    monkeypatch.undo()
    m.alloc_rules()
    first = m.rules
    m.alloc_rules()
    assert m.rules is first and first.history.counts.shape == (3, 100)


@pytest.mark.parametrize("slots,tokens", [(1, 8), (16, 64), (513, 1024)])
def test_the_planner_counts_what_is_allocated(slots, tokens):
    from dsv4_flash_deployment_b200.config import v4_flash_config
    from dsv4_flash_deployment_b200.engine import memory

    cfg = v4_flash_config() if slots < 100 else toy_v4_config()
    b = RuleBuffers(slots, tokens, tokens, cfg.vocab_size, "cpu")
    held = sum(t.numel() * t.element_size() for t in b.tensors())
    assert memory.rules_bytes(cfg, tokens, slots) == held
    plain = memory.non_expert_bytes(cfg, tokens, slots, 128, rules=False)
    assert memory.non_expert_bytes(cfg, tokens, slots, 128) == plain + held
    with_head = memory.non_expert_bytes(cfg, tokens, slots, 128, rules=False, head_int8=True)
    assert with_head - plain >= cfg.vocab_size * (cfg.dim + 4) + tokens * (cfg.dim + 4)


def test_the_pool_shrinks_by_what_the_rules_and_the_head_take():
    from dsv4_flash_deployment_b200.config import v4_flash_config
    from dsv4_flash_deployment_b200.engine import memory

    cfg = v4_flash_config()
    args = dict(max_tokens=1024, n_slots=513, max_seq=2048, kv_block=64, ep_world=8)
    size = lambda **kw: memory.kv_pool_tokens_for(cfg, 178 * 2 ** 30, 0.85, **args, **kw)
    assert size(rules=False) > size() > size(head_int8=True)
