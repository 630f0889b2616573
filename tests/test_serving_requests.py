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
