"""Penalties that differ from row to row of a generation."""
import pytest
import torch

from oslo_b200 import models
from oslo_b200.lightseq import generate

gpu = pytest.mark.gpu


def _gpt2(dev):
    torch.manual_seed(0)
    m = models.GPT2LMHeadModel(models.GPT2Config(vocab_size=67, n_positions=64, n_embd=32, n_layer=2, n_head=4, resid_pdrop=0.0,
                                                 embd_pdrop=0.0, attn_pdrop=0.0))
    for p in m.parameters():  # spread the logits: picked tokens do not hang on the last bits
        p.data.mul_(4.0 if p.dim() > 1 else 1.0)
    return m.eval().to(dev)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("kw", [dict(), dict(paged_cache=True, page_size=16), dict(num_beams=3), dict(use_cache=False)])
def test_each_row_has_its_own_penalties(dev, kw):
    m = _gpt2(dev)
    ids = torch.randint(0, 67, (3, 7), generator=torch.Generator().manual_seed(1)).to(dev)
    settings = dict(repetition_penalty=[1.0, 1.9, 1.3], presence_penalty=[0.0, 0.5, 3.0], frequency_penalty=[0.0, 2.0, 0.1])
    want = torch.cat([generate(m, ids[r : r + 1], max_new_tokens=9, **{k: v[r] for k, v in settings.items()}, **kw) for r in range(3)])
    assert torch.equal(generate(m, ids, max_new_tokens=9, **settings, **kw), want)
    as_tensors = {k: torch.tensor(v, device=dev) for k, v in settings.items()}
    assert torch.equal(generate(m, ids, max_new_tokens=9, **as_tensors, **kw), want)
    assert torch.equal(generate(m, ids, max_new_tokens=9, **{**settings, "presence_penalty": torch.tensor([0.0, 0.5, 3.0])}, **kw), want)
    assert as_tensors["repetition_penalty"].shape == (3,)
    for bad in (dict(repetition_penalty=[1.0, 2.0]), dict(presence_penalty=torch.ones(1)), dict(frequency_penalty=torch.ones(9)),
                dict(repetition_penalty=[1.0, 0.0, 1.0]), dict(repetition_penalty=float("nan")), dict(repetition_penalty=torch.ones(3, 1))):
        with pytest.raises(ValueError):
            generate(m, ids, max_new_tokens=2, **bad, **kw)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_rows_of_different_lengths_have_their_own_penalties(dev):
    m = _gpt2(dev)
    ids, lens, rep = torch.randint(0, 67, (3, 9), generator=torch.Generator().manual_seed(2)).to(dev), [9, 2, 5], [1.7, 1.0, 1.2]
    got = generate(m, ids, max_new_tokens=6, paged_cache=True, prompt_lengths=lens, repetition_penalty=rep)
    for r in range(3):
        alone = generate(m, ids[r : r + 1, : lens[r]], max_new_tokens=6, repetition_penalty=rep[r])[0]
        assert torch.equal(got[r, : lens[r] + 6], alone)
