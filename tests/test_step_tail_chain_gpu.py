"""The step-tail operators where they meet others: the MXFP8 rows of the norm in the
block-scaled product, and the int8 output head against the bf16 one."""

import pytest
import torch

from dsv4_flash_deployment_b200.ops import gemm as G
from dsv4_flash_deployment_b200.ops import norm as Q
from dsv4_flash_deployment_b200.ops.layout import chunks_to_sf

from test_gemm_gpu import _rand_fp8_weight
from test_model_gpu import small_v4
from test_rules_engine_gpu import _engine, _prompts
from test_step_tail_ops_gpu import BF, _check_norm, _done, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1, 7, 128, 300])
@pytest.mark.parametrize("k", [512, 1024])
def test_mxfp8_rows_feed_the_block_scaled_product(t, k):
    n = 384
    wq, ws = _rand_fp8_weight(n, k, 1)
    mw = G.MxWeight.from_checkpoint(wq, ws, "cuda")
    g = _gen(t + k)
    x, res = (torch.randn(t, k, device="cuda", generator=g).to(BF) for _ in range(2))
    nw = (1 + 0.2 * torch.randn(k, device="cuda", generator=g)).to(BF)
    got = Q.rms_norm_quant(x, nw, 1e-6, "mx8", residual=res)
    out = G.gemm_mx(got[0], got[1], t, mw, torch.empty(t, n, device="cuda"), G.EPI_F32)
    _done()
    _check_norm(got, x, nw, 1e-6, "mx8", res)
    sb = chunks_to_sf(got[1], t, k // 32).double()
    v = got[0][:t].view(torch.float8_e4m3fn).double() * torch.exp2(sb - 127).repeat_interleave(32, 1)
    w = wq.double().cuda() * torch.exp2(ws.double().cuda() - 127).repeat_interleave(32, 0).repeat_interleave(32, 1)
    # each product is exact in fp32; k additions, each off by a step (2^-23) of a partial sum
    assert ((out.double() - v @ w.t()).abs() <= k * 2.0 ** -23 * (v.abs() @ w.abs().t())).all()
    if t > 1:     # a row that is not finite is NaN behind the product too, and no other is
        x[t // 2, 3] = float("inf")
        got = Q.rms_norm_quant(x, nw, 1e-6, "mx8", residual=res)
        again = G.gemm_mx(got[0], got[1], t, mw, torch.empty(t, n, device="cuda"), G.EPI_F32)
        _done()
        rows = torch.arange(t, device="cuda") == t // 2
        assert torch.isnan(again[rows]).all() and torch.equal(again[~rows], out[~rows])


def _first_rows(eng, prompts):
    """The head's input and logits behind each prompt's last token, and the token."""
    m = eng.model
    reqs = [eng.add_request(p, 3, ignore_eos=True) for p in prompts]
    got = {}
    while not all(r.finished for r in reqs):
        rows = [(r, t) for r, t in eng.step() if t is not None]
        for i, (r, t) in enumerate(rows):
            if len(r.output) == 1:
                got[r.req_id] = (m.u_sample[i].double(), m.logits[i, : eng.cfg.vocab_size].double(), t)
    eng.check_errors()
    return [got[r.req_id] for r in reqs]


@pytest.mark.parametrize("graphs", [True, False])
def test_int8_head_against_the_bf16_head(graphs):
    """The same model and prompts through both heads.  The int8 engine's u_sample is the
    collapsed stream before the final norm, the bf16 engine's the norm's output: the one's
    norm is the other, and the logits differ by what the codes' half steps can add up to."""
    cfg = small_v4()
    prompts = _prompts(cfg)
    a, b = _engine(cfg, use_graphs=graphs), _engine(cfg, use_graphs=graphs, head_int8=True)
    assert torch.equal(a.model.head, b.model.head) and torch.equal(a.model.norm_w, b.model.norm_w)
    w = a.model.head[: cfg.vocab_size].double()
    ws = b.model.head_q.scale[: cfg.vocab_size].double()
    nw = a.model.norm_w.double()
    d = cfg.dim
    for (u, la, ta), (c, lb, tb) in zip(_first_rows(a, prompts), _first_rows(b, prompts)):
        y = c / (c.square().mean() + cfg.rms_norm_eps).sqrt() * nw
        # c and u round to bf16 once each (half a step, 2^-8), c's rounding also moves the root
        assert ((u - y).abs() <= y.abs() * (3 * 2.0 ** -8 + 2.0 ** -14)).all()
        ex = y.abs().amax() / 127 * 0.501 + 3 * 2.0 ** -8 * y.abs()      # int8's x against bf16's
        ew = ws * 0.501                                                  # int8's w against bf16's, a column
        tol = ex @ w.abs().t() + ew * (y.abs() + ex).sum() + d * 2.0 ** -23 * (u.abs() @ w.abs().t())
        err = (la - lb).abs()
        assert (err <= tol).all(), float((err / tol).max())
        # the bound is far from what another row's logits would differ by
        assert tol.max() < 0.7 * (la.max() - la.min())
        # the int8 head's token is one the bf16 head gives about as much to
        assert float(la[ta] - la[tb]) <= float(tol[ta] + tol[tb])
    assert len(prompts) == 3


def test_int8_head_under_speculative_decoding():
    """Drafted tokens are verified by the int8 head: the stream is that head's greedy one
    (up to near-ties between the 1-token and the 5-token path, as with the bf16 head)."""
    from dsv4_flash_deployment_b200.engine.builder import build_model
    from dsv4_flash_deployment_b200.io.checkpoint_spec import make_random_weights
    from dsv4_flash_deployment_b200.spec.dspark import SpecEngine

    from test_dspark_gpu import _greedy, spec_cfg

    cfg = spec_cfg()
    w = make_random_weights(cfg, seed=6)
    prompts = [torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (19, 26)]
    kw = dict(max_tokens=64, n_slots=4, max_seq_len=128, weights=w, head_int8=True)
    want = _greedy(build_model(cfg, "cuda", **kw), cfg, prompts[0], 20)
    eng = SpecEngine(build_model(cfg, "cuda", **kw), w, max_seqs=4)
    got = eng.generate(prompts, 20)
    _done()
    assert sum(int(a == b) for a, b in zip(got[0], want)) >= 18 and len(got[1]) == 20 and eng.stats.rounds > 0


@pytest.mark.parametrize("graphs", [True, False])
def test_histories_start_over_after_a_preemption(graphs):
    """A preempted request's context is prefilled again, its own output with it: a token of
    either is counted once, so none comes twice under a penalty that forbids it."""
    from dsv4_flash_deployment_b200.engine.engine import Engine

    cfg = small_v4()
    eng = Engine.build(cfg, "cuda", max_seqs=3, max_batched_tokens=64, max_seq_len=128, seed=3, chunk_size=24,
                       use_graphs=graphs, kv_block=4, kv_pool_tokens=160, kv_preempt=True)
    n = 40
    reqs = [eng.add_request(p, n, ignore_eos=True, presence_penalty=1e6, logit_bias={5: float("-inf")})
            for p in _prompts(cfg)]
    counted = []
    while not all(r.finished for r in reqs):
        eng.step()
        live = [r for r in reqs if r.slot >= 0 and r.output and r.prompt_done]
        counted += [(r, eng.model.rules.history.counts[r.slot].sum().item(), len(r.output)) for r in live]
    eng.check_errors()
    assert sum(r.preemptions for r in reqs) > 0
    for r in reqs:
        assert len(r.output) == n and len(set(r.output)) == n and 5 not in r.output
    # after a step the last token is not in the history yet; every other one is, once
    assert counted and all(c == k - 1 for _, c, k in counted)
