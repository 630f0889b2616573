"""Requests that share the server with others: one that is refused fails alone."""
import asyncio

import pytest
import torch

from oslo_b200 import models
from oslo_b200.lightseq import generate


def _gpt2():
    torch.manual_seed(0)
    return models.GPT2LMHeadModel(models.GPT2Config(vocab_size=67, n_positions=32, n_embd=32, n_layer=1, n_head=4, resid_pdrop=0.0,
                                                    embd_pdrop=0.0, attn_pdrop=0.0)).eval()


def _batch(requests, **kw):
    """Results (or exceptions) of requests ``(ids, settings)`` that arrive together, and the batches they ran in."""
    from oslo_b200.lightseq.serving import DynamicBatcher

    m, calls = _gpt2(), []

    def run(ids, **params):
        calls.append(tuple(ids.shape))
        return generate(m, ids, **params)

    async def go():
        batcher = DynamicBatcher(run, max_batch=8, max_wait_ms=200.0, **kw)
        out = await asyncio.wait_for(asyncio.gather(*[batcher.submit(ids, max_new_tokens=3, **p) for ids, p in requests], return_exceptions=True), 60)
        await batcher.stop()
        return out

    return asyncio.run(go()), calls


def test_settings_that_are_lists_do_not_stop_the_batcher():
    forced = [[9, 1e4]]
    out, calls = _batch([([1, 2], dict(logit_bias=forced)), ([3, 4], {}), ([5, 6], dict(logit_bias=[[9, 1e4]])),
                         ([7, 8], dict(logit_bias={9: 1e4})), ([1, 2], dict(logit_bias={3, 4}))])
    assert out[0] == ([1, 2, 9, 9, 9], 2) and out[2] == ([5, 6, 9, 9, 9], 2)  # equal lists share a batch
    assert out[3] == ([7, 8, 9, 9, 9], 1)
    assert out[1][0][:2] == [3, 4] and len(out[1][0]) == 5
    assert isinstance(out[4], Exception) and sorted(calls) == [(1, 2)] * 3 + [(2, 2)]


def test_biases_over_http():
    testclient = pytest.importorskip("fastapi.testclient")
    from oslo_b200.lightseq.serving import create_app

    try:
        client = testclient.TestClient(create_app(_gpt2(), max_wait_ms=1.0))
    except RuntimeError as e:  # the test client needs a package that the server does not
        pytest.skip(str(e))
    with client:
        _ask(lambda body: (lambda r: (r.status_code, r.json()))(client.post("/generate", json=body)))


def test_biases_of_requests():
    """The same through the application's own handlers."""
    _through_the_handlers(_ask)


def _through_the_handlers(ask):
    fastapi = pytest.importorskip("fastapi")
    from oslo_b200.lightseq.serving import create_app

    app = create_app(_gpt2(), max_wait_ms=1.0)
    handler = next(r.endpoint for r in app.routes if getattr(r, "path", "") == "/generate")

    async def one(body):
        try:
            return 200, await asyncio.wait_for(handler(body), 60)
        except fastapi.HTTPException as e:
            return e.status_code, e.detail
        finally:
            await app.state.batcher.stop()
            app.state.batcher.queue = None

    ask(lambda body: asyncio.run(one(body)))


def _ask(post):
    ids = dict(input_ids=[[1, 2]], max_new_tokens=3)
    for bias in ([[9, 1e4]], {"9": 1e4}, [["9", "1e4"]], [[9, -5.0], [9, 1e4]]):
        status, body = post(dict(ids, logit_bias=bias))
        assert status == 200 and body["output_ids"] == [[1, 2, 9, 9, 9]], (bias, body)
    plain = post(ids)[1]["output_ids"]
    assert post(dict(ids, logit_bias=None))[1]["output_ids"] == post(dict(ids, logit_bias=[]))[1]["output_ids"] == plain
    for bias in (7, [1, 2], [[1, 2, 3]], {"a": 1}, {"1": "x"}, [[[1], 2]], "ab", True):
        status, body = post(dict(ids, logit_bias=bias))
        assert status == 422, (bias, status, body)
    assert post(ids)[1]["output_ids"] == plain


def test_a_refused_prompt_does_not_take_others_along():
    paged = dict(paged_cache=True)
    alone = {n: generate(_gpt2(), torch.arange(1, n + 1)[None], max_new_tokens=3)[0].tolist() for n in (2, 3)}
    # empty; longer than the model's positions; not numbers
    for bad in ([], list(range(1, 40)), ["x", "y", "z", "w"]):
        out, _ = _batch([([1, 2, 3], paged), (bad, paged), ([1, 2], paged), ([1, 2, 3], paged)], ragged=True)
        assert isinstance(out[1], Exception), bad
        assert [out[i][0] for i in (0, 2, 3)] == [alone[3], alone[2], alone[3]]
    out, calls = _batch([([1, 2, 3], paged), ([1, 2], paged)], ragged=True)  # together as ever
    assert [r for r, n in out] == [alone[3], alone[2]] and calls == [(2, 3)]


def test_numbers_for_rows_do_not_meet_in_a_batch():
    """A list of penalties belongs to the rows of its own request, whatever shares the window."""
    pen = lambda x: dict(presence_penalty=x)
    requests = [([1, 2], pen([1e4])), ([1, 2], pen([1e4])), ([1, 2], pen((1e4,))), ([1, 2], pen((1e4,))), ([1, 2], pen([1e4, 0.0]))]
    out, calls = _batch(requests)
    want = generate(_gpt2(), torch.tensor([[1, 2]]), max_new_tokens=3, presence_penalty=1e4)[0].tolist()
    assert all(r == (want, 1) for r in out[:4]) and isinstance(out[4], ValueError) and calls == [(1, 2)] * 5


def test_penalties_over_http_are_numbers():
    def ask(post):
        ids = dict(input_ids=[[1, 2], [3, 4]], max_new_tokens=2)
        assert post(dict(ids, presence_penalty=1, repetition_penalty=1.5))[0] == 200
        for bad in ([1.0, 2.0], "1", None):
            assert post(dict(ids, presence_penalty=bad))[0] == 422, bad

    _through_the_handlers(ask)
