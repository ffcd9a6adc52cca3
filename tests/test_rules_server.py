"""Values of the rules' fields that no engine can take are answered with 400."""

import asyncio

from aiohttp.test_utils import TestClient, TestServer

from dsv4_flash_deployment_b200.serving.app import ServerState, build_app
from dsv4_flash_deployment_b200.serving.engine_loop import EngineLoop
from dsv4_flash_deployment_b200.serving.tokenizer import load_tokenizer

from test_rules_engine import P, _engine

BAD = ['"allowed_token_ids": [Infinity]', '"allowed_token_ids": [NaN]', '"allowed_token_ids": 5', '"allowed_token_ids": []',
       '"allowed_token_ids": [65], "logit_bias": {"65": -Infinity}', '"logit_bias": {"65": 1e999}',
       '"logit_bias": {"65": 1' + "0" * 400 + '}', '"frequency_penalty": 1' + "0" * 400, '"presence_penalty": NaN',
       '"logit_bias": {"65": [1]}', '"repetition_penalty": -Infinity']


def test_values_out_of_range_are_refused():
    eng = _engine()
    loop = EngineLoop(eng).start()

    async def go():
        st = ServerState(loop, load_tokenizer(None, eng.cfg), "m", 96)
        async with TestClient(TestServer(build_app(st))) as cl:
            async def ask(fields):
                body = f'{{"prompt": {P}, "max_tokens": 2, "ignore_eos": true, {fields}}}'
                r = await cl.post("/v1/completions", data=body, headers={"Content-Type": "application/json"})
                return r.status
            return [(f[:60], await ask(f)) for f in BAD], await ask('"logit_bias": {"65": -Infinity}')
    try:
        got, ok = asyncio.run(go())
    finally:
        loop.stop()
    assert [g for g in got if g[1] != 400] == [] and ok == 200 and loop.healthy
