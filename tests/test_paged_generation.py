"""Generation over the paged cache, with penalties, biases and grammar masks: the operators together, as they are used."""
import asyncio
import math

import pytest
import torch

from oslo_b200 import models
from oslo_b200.lightseq import LSGpt, LSModelConfig, generate
from oslo_b200.nn import functional as OF
from oslo_b200.ops.attention import decode_cache
from oslo_b200.ops.paged import PagedDecodeCache

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def _model(kind, dev="cpu"):
    torch.manual_seed(0)
    if kind == "gpt2":
        m = models.GPT2LMHeadModel(models.GPT2Config(vocab_size=67, n_positions=96, n_embd=32, n_layer=2, n_head=4, resid_pdrop=0.0,
                                                     embd_pdrop=0.0, attn_pdrop=0.0))
    elif kind == "neox":
        m = models.GPTNeoXForCausalLM(models.GPTNeoXConfig(vocab_size=67, hidden_size=64, num_hidden_layers=2, num_attention_heads=4,
                                                           intermediate_size=64, rotary_pct=0.25, max_position_embeddings=96))
    else:
        m = models.LlamaForCausalLM(models.LlamaConfig(vocab_size=67, hidden_size=64, intermediate_size=64, num_hidden_layers=2,
                                                       num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=24))
    for p in m.parameters():  # spread the logits: picked tokens do not hang on the last bits
        p.data.mul_(4.0 if p.dim() > 1 else 1.0)
    return m.eval().to(dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["gpt2", "neox", "llama"])
def test_paged_generation_equals_dense(dev, kind):
    m = _model(kind, dev)
    prompt = torch.randint(0, 67, (3, 13), device=dev)
    want = generate(m, prompt, max_new_tokens=24)  # crosses pages of 16, and the first rotation table of the Llama model
    assert torch.equal(generate(m, prompt, max_new_tokens=24, paged_cache=True, page_size=16), want)
    assert torch.equal(generate(m, prompt, max_new_tokens=24, paged_cache=True), want)
    eos = int(want[0, 16])
    assert torch.equal(generate(m, prompt, max_new_tokens=9, paged_cache=True, page_size=32, eos_token_id=eos),
                       generate(m, prompt, max_new_tokens=9, eos_token_id=eos))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["gpt2", "neox", "llama"])
def test_prompts_of_different_lengths_equal_one_by_one(dev, kind):
    m = _model(kind, dev)
    lens = [5, 17, 1, 16]
    ids = torch.randint(0, 67, (4, 20), device=dev)
    kw = dict(max_new_tokens=12, repetition_penalty=1.3, frequency_penalty=0.2, presence_penalty=0.1)
    got = generate(m, ids, paged_cache=True, page_size=16, prompt_lengths=lens, **kw)
    assert got.shape == (4, 32)
    for r, n in enumerate(lens):
        alone = generate(m, ids[r : r + 1, :n], **kw)[0]
        assert torch.equal(got[r, : n + 12], alone), r
        assert (got[r, n + 12 :] == 0).all()
    eos = int(got[1, 20])
    stopped = generate(m, ids, paged_cache=True, prompt_lengths=lens, eos_token_id=eos, **kw)
    for r, n in enumerate(lens):
        alone = generate(m, ids[r : r + 1, :n], eos_token_id=eos, **kw)[0]
        assert torch.equal(stopped[r, : len(alone)], alone)
        assert (stopped[r, len(alone) :] == eos).all()


def test_incremental_logits_and_pages():
    m = _model("llama")
    ids = torch.randint(0, 67, (2, 40))
    cache = PagedDecodeCache(max_tokens=40, page_size=16, num_pages=6)
    at = [9, 4]
    with torch.no_grad():
        full = [m(input_ids=ids[r : r + 1]).logits[0] for r in range(2)]
        cache.begin_forward(at)
        with decode_cache(cache):
            first = m(input_ids=ids[:, :9]).logits
        cache.advance(9)
        for r in range(2):
            assert torch.allclose(first[r, at[r] - 1], full[r][at[r] - 1], atol=1e-4)
        for s in (1, 3, 1, 5, 1, 1, 7):  # several tokens at once see one another in order
            feed = torch.stack([ids[r, at[r] : at[r] + s] for r in range(2)])
            cache.begin_forward()
            with decode_cache(cache):
                got = m(input_ids=feed).logits
            cache.advance(s)
            for r in range(2):
                assert torch.allclose(got[r], full[r][at[r] : at[r] + s], atol=1e-4), (r, s)
                at[r] += s
    assert cache.lengths == at == [28, 23] and [len(p) for p in cache.pages] == [2, 2] and len(cache._free) == 2
    assert len(cache.k_pages) == 2 and cache.k_pages[0].shape == (6, 2, 16, 8)  # the key heads once, not repeated
    with pytest.raises(RuntimeError, match="different lengths"):
        cache.offset
    with pytest.raises(RuntimeError, match="beams"):
        cache.reorder(torch.tensor([1, 0]))


def test_refusals_of_the_generation():
    m = _model("gpt2")
    ids = torch.randint(0, 67, (2, 6))
    for kw in (dict(paged_cache=True, num_beams=2), dict(paged_cache=True, use_cache=False), dict(prompt_lengths=[3, 6]),
               dict(paged_cache=True, prompt_lengths=[3]), dict(paged_cache=True, prompt_lengths=[0, 6]),
               dict(paged_cache=True, prompt_lengths=[3, 7]), dict(paged_cache=True, page_size=24),
               dict(paged_cache=True, prompt_lengths=[3, 6], no_repeat_ngram_size=2), dict(repetition_penalty=0.0),
               dict(logit_bias={67: 1.0})):
        with pytest.raises(ValueError):
            generate(m, ids, max_new_tokens=2, **kw)
    ls = LSGpt(LSModelConfig(hidden_size=32, nhead=4, intermediate_size=64, num_decoder_layer=1, vocab_size=67)).eval()
    ids = torch.randint(1, 67, (2, 6))
    assert torch.equal(generate(ls, ids, max_new_tokens=5, paged_cache=True), generate(ls, ids, max_new_tokens=5))
    with pytest.raises(ValueError, match="one length"):
        generate(ls, ids, max_new_tokens=2, paged_cache=True, prompt_lengths=[3, 6])


def test_refusals_of_the_cache():
    with pytest.raises(ValueError):
        PagedDecodeCache(10, page_size=8)
    with pytest.raises(ValueError):
        PagedDecodeCache(0)
    q, k = torch.randn(2, 20, 4, 8), torch.randn(2, 20, 2, 8)
    with torch.no_grad():
        cache = PagedDecodeCache(64, page_size=16, num_pages=3)
        with pytest.raises(RuntimeError, match="exhausted"):
            cache.attend(q, k, k)
        cache = PagedDecodeCache(19, page_size=16)
        with pytest.raises(ValueError, match="max_tokens"):
            cache.attend(q, k, k)
        cache = PagedDecodeCache(64, page_size=16)
        cache.begin_forward([20, 21])
        with pytest.raises(ValueError, match="real"):
            cache.attend(q, k, k)
        cache.begin_forward([20, 7])
        cache.attend(q, k, k)
        cache.advance(20)
        cache.begin_forward()
        with pytest.raises(ValueError, match="rows"):
            cache.attend(q[:1, :1], k[:1, :1], k[:1, :1])
        cache.begin_forward([2, 1])
        with pytest.raises(ValueError, match="padded"):
            cache.attend(q[:, :2], k[:, :2], k[:, :2])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("paged", [False, True])
def test_rules_of_the_logits_in_generation(dev, paged):
    m = _model("gpt2", dev)
    ids = torch.randint(0, 67, (2, 7), device=dev)
    kw = dict(max_new_tokens=10, paged_cache=paged)
    plain = generate(m, ids, **kw)
    assert torch.equal(generate(m, ids, logit_bias={}, **kw), plain)
    forced = generate(m, ids, logit_bias={"11": 1e4}, **kw)
    assert (forced[:, 7:] == 11).all()
    assert torch.equal(generate(m, ids, logit_bias=[(11, 1e4)], **kw), forced)
    spread = generate(m, ids, logit_bias={11: 1e4}, frequency_penalty=1e6, **kw)
    assert all(len(set(row)) == 10 for row in spread[:, 7:].tolist())  # each token once: its next turn costs more than the bias gives

    seen = []

    def even(tokens, lengths):
        seen.append((tokens.shape[1], lengths))
        keep = torch.zeros(2, 67, dtype=torch.bool, device=dev)
        keep[:, 0::2] = True
        return keep if len(seen) % 2 else OF.pack_token_mask(keep)

    assert (generate(m, ids, allowed_tokens=even, **kw)[:, 7:] % 2 == 0).all()
    assert [n for n, _ in seen] == list(range(7, 17))
    assert torch.equal(generate(m, ids, allowed_tokens=lambda t, n: None, **kw), plain)

    # the penalty for repetition, spelled out over the whole prefix
    want = ids
    with torch.no_grad():
        for _ in range(10):
            x = m(input_ids=want).logits[:, -1].float()
            for r in range(2):
                for t in set(want[r].tolist()):
                    x[r, t] = x[r, t] / 1.7 if x[r, t] > 0 else x[r, t] * 1.7
                for t in set(want[r, 7:].tolist()):
                    x[r, t] -= 0.3
            want = torch.cat([want, x.argmax(-1, keepdim=True)], dim=1)
    assert torch.equal(generate(m, ids, repetition_penalty=1.7, presence_penalty=0.3, **kw), want)


def test_rules_reach_beams_and_sampling():
    m = _model("gpt2")
    ids = torch.randint(0, 67, (2, 7))
    plain = generate(m, ids, max_new_tokens=6, num_beams=3)
    assert torch.equal(generate(m, ids, max_new_tokens=6, num_beams=3, frequency_penalty=0.0), plain)
    only = [3, 8, 60]
    keep = torch.zeros(1, 67, dtype=torch.bool)
    keep[:, only] = True
    for kw in (dict(num_beams=3), dict(do_sample=True, top_k=5)):
        out = generate(m, ids, max_new_tokens=6, allowed_tokens=lambda t, n: keep, **kw)
        assert set(out[:, 7:].reshape(-1).tolist()) <= set(only)


def test_server_batches_prompts_of_different_lengths():
    from oslo_b200.lightseq.serving import DynamicBatcher

    m = _model("llama")
    calls = []

    def run(ids, **params):
        calls.append((tuple(ids.shape), params.get("prompt_lengths")))
        return generate(m, ids, **params)

    prompts = [[1, 2, 3], [4, 5, 6, 7, 8], [9]]

    async def go(ragged, **params):
        batcher = DynamicBatcher(run, max_batch=4, max_wait_ms=200.0, ragged=ragged)
        out = await asyncio.gather(*[batcher.submit(p, max_new_tokens=6, **params) for p in prompts])
        await batcher.stop()
        return out

    alone = [generate(m, torch.tensor([p]), max_new_tokens=6)[0].tolist() for p in prompts]
    assert asyncio.run(go(True, paged_cache=True)) == [(row, 3) for row in alone]
    assert calls == [((3, 5), [3, 5, 1])]
    assert asyncio.run(go(True)) == [(row, 1) for row in alone]
    assert asyncio.run(go(False, paged_cache=True)) == [(row, 1) for row in alone]


def test_server_takes_the_settings():
    testclient = pytest.importorskip("fastapi.testclient")
    from oslo_b200.lightseq.serving import create_app

    try:
        client = testclient.TestClient(create_app(_model("gpt2"), max_wait_ms=1.0))
    except RuntimeError as e:  # the test client needs a package that the server does not
        pytest.skip(str(e))
    with client:
        body = dict(input_ids=[[1, 2, 3], [4, 5]], max_new_tokens=4, paged_cache=True, logit_bias={"9": 1e4})
        r = client.post("/generate", json=body)
        assert r.status_code == 200 and r.json()["output_ids"] == [[1, 2, 3, 9, 9, 9, 9], [4, 5, 9, 9, 9, 9]]


def _parallel_worker(rank, world, kind, two_d):
    import oslo_b200
    from oslo_b200 import ParallelContext, ParallelMode
    from oslo_b200.parallel import TensorParallel

    pc = ParallelContext.from_torch(tensor_parallel_size=world, backend="gloo", seed=0,
                                    tensor_parallel_mode=ParallelMode.TENSOR_2D if two_d else ParallelMode.TENSOR_1D)
    ref, wrapped = _model(kind), TensorParallel(_model(kind), pc)
    oslo_b200.ready(wrapped, pc)
    prompt = torch.randint(1, 67, (2, 9), generator=torch.Generator().manual_seed(1))
    kw = dict(max_new_tokens=10, paged_cache=True, page_size=16, repetition_penalty=1.3)
    assert torch.equal(generate(wrapped, prompt, **kw), generate(ref, prompt, **kw))
    if two_d:
        with pytest.raises(ValueError, match="split the batch"):
            generate(wrapped, prompt, prompt_lengths=[4, 9], **kw)
    else:
        assert torch.equal(generate(wrapped, prompt, prompt_lengths=[4, 9], **kw), generate(ref, prompt, prompt_lengths=[4, 9], **kw))
    pc.destroy()


@pytest.mark.parametrize("kind,world,two_d", [("gpt2", 2, False), ("neox", 2, False), ("llama", 2, False), ("neox", 4, True),
                                              ("gpt2", 4, True)])
def test_paged_generation_through_tensor_parallel_models(kind, world, two_d):
    from dist_utils import run_dist

    run_dist(_parallel_worker, world, kind, two_d)


# ------------------------------------------------------------------------------------------------ the operators on the GPU
def _step(q, k, v, kp, vp, table, held, rope, logits, tokens, lens):
    """One decoding step's calls."""
    turned = OF.paged_kv_append(k, v, kp, vp, table, held, q=q, rope=rope)
    out = OF.paged_attention(turned, kp, vp, table, held + 1)
    return out, OF.process_logits(logits, tokens, lens, repetition_penalty=1.2, frequency_penalty=0.1)


def _state(seed, b=3, hq=8, hkv=2, d=64, page=16, width=40, most=600, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
    table = torch.randperm(b * width, device="cuda", generator=g).int().view(b, width)
    held = torch.randint(1, most, (b,), device="cuda", generator=g, dtype=torch.int32)
    rope = (*OF.rope_tables(width * page, d, device="cuda"), d, True)
    return [r(b, 1, hq, d), r(b, 1, hkv, d), r(b, 1, hkv, d), r(b * width, hkv, page, d), r(b * width, hkv, page, d), table, held, rope,
            torch.randn(b, 5000, device="cuda", generator=g), torch.randint(0, 5000, (b, 70), device="cuda", generator=g),
            torch.randint(1, 70, (b,), device="cuda", generator=g, dtype=torch.int32)]


@gpu
@pytest.mark.parametrize("width,most", [(40, 600), (400, 6000)])  # one launch with clusters; two launches
def test_step_in_cuda_graphs(width, most):
    """Two graphs of the same step on different states, replayed by turns and with new inputs, give what eager calls give."""
    states = [_state(i, width=width, most=most) for i in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for st in states:
            _step(*st)
        side.synchronize()
        for st in states:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(_step(*st))
            graphs.append(g)
    torch.cuda.synchronize()
    for round_ in range(3):
        fresh = [_state(10 * round_ + i, width=width, most=most) for i in (3, 4)]
        for st, new in zip(states, fresh):
            for a, b in zip(st, new):
                if isinstance(a, torch.Tensor):
                    a.copy_(b)
        want = [_step(*st) for st in fresh]
        graphs[round_ % 2].replay()
        graphs[1 - round_ % 2].replay()
        torch.cuda.synchronize()
        for got, exp, st, new in zip(outs, want, states, fresh):
            assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])
            assert torch.equal(st[3], new[3]) and torch.equal(st[4], new[4])


@gpu
@pytest.mark.parametrize("width,most", [(40, 600), (400, 6000)])
def test_steps_on_two_streams(width, most):
    states = [_state(20 + i, width=width, most=most) for i in range(6)]
    want = [_step(*[t.clone() if isinstance(t, torch.Tensor) else t for t in st]) for st in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, st in enumerate(states):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_step(*st))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@gpu
def test_results_do_not_change_from_run_to_run():
    for width, most in ((40, 600), (400, 6000)):
        st = _state(30, b=5, width=width, most=most)
        first = _step(*st)
        for _ in range(10):
            again = _step(*st)
            assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_generation_in_16_bits_follows_the_dense_cache(dtype):
    """Teacher-forced logits of both caches.  They round the attention's output once each, to the model's type: per layer the
    residual stream may differ by two half steps of the layer's output, which the norms keep at the size of the stream."""
    from oslo_b200.ops.attention import DecodeCache

    m = _model("llama", "cuda").to(dtype)
    ids = torch.randint(0, 67, (3, 60), device="cuda")
    got, want = [], []
    with torch.no_grad():
        for cache, out in ((PagedDecodeCache(60, 16), got), (DecodeCache(), want)):
            for a, e in [(0, 30)] + [(i, i + 1) for i in range(30, 60)]:
                cache.begin_forward()
                with decode_cache(cache):
                    out.append(m(input_ids=ids[:, a:e]).logits.float())
                cache.advance(e - a)
    got, want = torch.cat(got, 1), torch.cat(want, 1)
    eps = torch.finfo(dtype).eps
    rel = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
    # 2 layers x 2 residual additions and projections, each rounding both runs: 16 half steps, and their spread over later layers
    assert rel <= 16 * eps, rel
    assert math.isfinite(rel)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_calls_with_and_without_the_step_module_agree(dtype, monkeypatch):
    from oslo_b200.ops import _lib, logits as logits_ops, paged as paged_ops

    module = _lib.step_calls()
    assert module is not None
    taken = []

    def through(f):
        def call(*args):
            out = f(*args)
            taken.append(out is not NotImplemented)
            return out

        return call

    def run(width, most):
        torch.manual_seed(0)  # both sides get the same inputs
        q, k, v, kp, vp, table, held, rope, x, tokens, lens = _state(40, width=width, most=most, dtype=dtype)
        b = q.shape[0]
        mask = torch.randn(b, 1, 1, width * 16, device="cuda")
        kp, vp = kp.clone(), vp.clone()
        none = torch.zeros_like(held)
        out = [OF.paged_kv_append(k, v, kp, vp, table, held, count=none + 1, q=q, rope=rope),
               OF.paged_kv_append(k, v, kp, vp, table, held)]
        out += [OF.paged_attention(q, kp, vp, table, held + 1, **kw)
                for kw in (dict(), dict(scale=0.2), dict(mask=mask), dict(mask=mask[:1]), dict(mask=mask.double()))]
        rates = torch.rand(b, device="cuda") + 0.5
        allowed = OF.pack_token_mask(torch.rand(b, 5000, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) < 0.5)
        for kw in (dict(), dict(tokens=tokens, repetition_penalty=1.5), dict(tokens=tokens.int(), presence_penalty=rates * 0 + 0.3),
                   dict(tokens=tokens, token_lengths=lens, prompt_lengths=lens // 2, frequency_penalty=1),
                   dict(bias=x[0]), dict(bias=x * 2, allowed=allowed), dict(allowed=allowed[:1]), dict(bias=x[0].half())):
            out.append(OF.process_logits(x.to(dtype), **kw))
        return out + [kp, vp]

    for width, most in ((40, 600), (400, 6000)):
        run(width, most)
        monkeypatch.setattr(paged_ops, "_direct", tuple(through(f) for f in (module.paged_kv_append, module.paged_attention)))
        monkeypatch.setattr(logits_ops, "_direct", through(module.process_logits))
        before = _lib.native_calls
        a = run(width, most)
        assert _lib.native_calls - before >= 15 and sum(taken) >= 11 and not all(taken)
        monkeypatch.setattr(paged_ops, "_direct", (paged_ops._not_built,) * 2)
        monkeypatch.setattr(logits_ops, "_direct", lambda *args: NotImplemented)
        b = run(width, most)
        for i, (x, y) in enumerate(zip(a, b)):
            assert (x is None and y is None) or torch.equal(x.nan_to_num(), y.nan_to_num()), i
        taken.clear()


def test_step_module_leaves_what_is_not_ordinary():
    from oslo_b200.csrc.build import build_step
    from oslo_b200.ops import _lib

    build_step()
    module = _lib.step_calls()
    t = torch.zeros(2, 1, 4, 64)
    for args in ((), (t,) * 7, (t, t, t, t, t, None, None), (None,) * 9, (t,) * 9, (1,) * 9, ("q",) * 7):
        for f in (module.paged_kv_append, module.paged_attention, module.process_logits):
            assert f(*args) is NotImplemented
