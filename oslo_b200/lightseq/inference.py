"""Text generation for the in-tree causal language models: greedy, top-k / top-p sampling and beam search, with
n-gram blocking on the fused kernel and a key / value cache: the prompt is run once, after which every step feeds only
the newest token and attends over the cached keys and values (``oslo_b200.ops.attention.DecodeCache``, or in pages that
never move and for prompts of different lengths: ``oslo_b200.ops.paged.PagedDecodeCache``).  Penalties for repeated tokens,
biases and grammar masks on the logits are one kernel (``oslo_b200.ops.logits.process_logits``).

A compact counterpart of LightSeq's inference engine entry points (oslo/lightseq2/inference/pywrapper/*, sampling and
beam-search kernels in inference/kernels/transformerKernels.cc.cu): the model forward runs on this repository's
training kernels; the decoding bookkeeping is vectorised torch code on the device (no host loop over hypotheses).
"""
from __future__ import annotations

from typing import Callable, Mapping, Optional, Sequence, Union

import torch
import torch.nn.functional as F

from oslo_b200.nn.ngram_repeat_block import NGramRepeatBlock
from oslo_b200.ops.attention import DecodeCache, decode_cache
from oslo_b200.ops.logits import pack_token_mask, process_logits
from oslo_b200.ops.paged import PagedDecodeCache


def _logits(model, ids, cache: Optional[DecodeCache] = None):
    """Next-token logits.  With a cache only the tokens it has not seen yet are run through the model."""
    if cache is None:
        out = model(input_ids=ids)
    else:
        new = ids[:, cache.offset :]
        cache.begin_forward()
        with decode_cache(cache):
            out = model(input_ids=new)
        cache.advance(new.shape[1])
    logits = out.logits if hasattr(out, "logits") else out[0]
    return _whole_logits(model, logits[:, -1, :]).float()


def _whole_logits(model, last: torch.Tensor) -> torch.Tensor:
    """Tensor-parallel models whose head keeps the vocabulary sharded (for the vocab-parallel loss) return a slice of the
    logits; picking the next token needs all of them.  ``last``: ``[batch, vocab or a shard of it]``."""
    pc = getattr(model, "parallel_context", None)
    if pc is None or getattr(pc, "tensor_parallel_size", 1) == 1:
        return last
    base = getattr(model, "module", model)
    vocab = getattr(base, "orig_vocab_size", None) or base.config.vocab_size
    if last.shape[-1] >= vocab:
        return last[..., :vocab]
    from oslo_b200.distributed import ParallelMode, comm

    mode = pc.tensor_parallel_mode
    if mode == ParallelMode.TENSOR_1D:
        full = comm.all_gather(last.contiguous(), dim=-1, parallel_context=pc, parallel_mode=ParallelMode.TENSOR_1D)
    elif mode == ParallelMode.TENSOR_2D:
        from oslo_b200.parallel.tensor_parallel._ops_2d import gather_output_2d

        full = gather_output_2d(last.contiguous(), pc)
    elif mode == ParallelMode.TENSOR_2P5D:
        from oslo_b200.parallel.tensor_parallel._ops_2p5d import gather_output_2p5d

        full = gather_output_2p5d(last.contiguous(), pc)
    else:
        from oslo_b200.parallel.tensor_parallel._ops_3d import gather_output_3d

        full = gather_output_3d(last.contiguous(), pc)
    return full[..., :vocab]


def _filter(logits, top_k: int, top_p: float):
    if top_k and top_k > 0:
        kth = logits.topk(min(top_k, logits.shape[-1]), dim=-1).values[:, -1:]
        logits = logits.masked_fill(logits < kth, float("-inf"))
    if top_p and top_p < 1.0:
        sorted_logits, idx = logits.sort(dim=-1, descending=True)
        cum = sorted_logits.softmax(-1).cumsum(-1)
        drop = cum - sorted_logits.softmax(-1) > top_p
        sorted_logits = sorted_logits.masked_fill(drop, float("-inf"))
        logits = torch.full_like(logits, float("-inf")).scatter(1, idx, sorted_logits)
    return logits


class _LogitsRules:
    """The penalties, biases and grammar of one generation, applied to the next-token logits of a step."""

    def __init__(self, repetition_penalty, presence_penalty, frequency_penalty, logit_bias, allowed_tokens, beams=1):
        self.beams, self.spread = beams, False
        self.penalties = dict(repetition_penalty=repetition_penalty, presence_penalty=presence_penalty,
                              frequency_penalty=frequency_penalty)
        for name, p in self.penalties.items():  # one number a row
            if isinstance(p, (list, tuple)):
                self.penalties[name] = torch.tensor(p, dtype=torch.float32)
        self.counts = any(isinstance(p, torch.Tensor) or p != none for p, none in zip(self.penalties.values(), (1.0, 0.0, 0.0)))
        repetition = self.penalties["repetition_penalty"]
        if not (bool((repetition > 0).all()) if isinstance(repetition, torch.Tensor) else repetition > 0):
            raise ValueError(f"repetition_penalty is positive: got {repetition_penalty}")
        self.bias, self.allowed_tokens = logit_bias, allowed_tokens
        self.active = self.counts or logit_bias is not None or allowed_tokens is not None

    def __call__(self, logits, ids, lengths, prompts):
        """``ids [rows, >= lengths]``, of which ``lengths`` (int32 ``[rows]``; ``None``: all) count and ``prompts`` are the prompt."""
        if not self.active:
            return logits
        rows, vocab = logits.shape
        if self.bias is not None and not isinstance(self.bias, torch.Tensor):
            pairs = list(self.bias.items() if isinstance(self.bias, Mapping) else self.bias)
            bias = torch.zeros(vocab)
            for token, value in pairs:
                if not 0 <= int(token) < vocab:
                    raise ValueError(f"logit_bias names token {token}, the vocabulary has {vocab}")
                bias[int(token)] = float(value)
            self.bias = bias
        if self.bias is not None:
            self.bias = self.bias.to(logits.device)
        allowed = None
        if self.allowed_tokens is not None:
            allowed = self.allowed_tokens(ids, lengths)
            if allowed is not None and allowed.dtype == torch.bool:
                allowed = pack_token_mask(allowed)
        history = {}
        if self.counts:
            for name, p in self.penalties.items():
                if isinstance(p, torch.Tensor) and not self.spread:
                    if p.shape != (rows // self.beams,):
                        raise ValueError(f"{name} is a number or one number for each of {rows // self.beams} rows: got {tuple(p.shape)}")
                    self.penalties[name] = p.to(logits.device).repeat_interleave(self.beams)  # a row's beams share its number
            self.spread = True
            history = dict(tokens=ids, token_lengths=lengths, prompt_lengths=prompts, **self.penalties)
        return process_logits(logits, bias=self.bias, allowed=allowed, **history)


@torch.no_grad()
def generate(model, input_ids: torch.Tensor, max_new_tokens: int = 32, do_sample: bool = False, top_k: int = 0,
             top_p: float = 1.0, temperature: float = 1.0, num_beams: int = 1, no_repeat_ngram_size: int = 0,
             eos_token_id: Optional[int] = None, length_penalty: float = 1.0, pad_multiple: int = 1,
             use_cache: bool = True, paged_cache: bool = False, page_size: int = 64,
             prompt_lengths: Optional[Sequence[int]] = None, repetition_penalty: Union[float, torch.Tensor, Sequence] = 1.0,
             presence_penalty: Union[float, torch.Tensor, Sequence] = 0.0, frequency_penalty: Union[float, torch.Tensor, Sequence] = 0.0,
             logit_bias: Union[None, torch.Tensor, Mapping, Sequence] = None, allowed_tokens: Optional[Callable] = None):
    """Returns ``[batch, prompt + new]`` token ids (best beam when ``num_beams > 1``).  ``use_cache=False`` re-runs the
    whole prefix every step (the reference behaviour for models whose attention does not go through ``oslo_b200.ops``).

    ``paged_cache``: keep keys and values in pages of ``page_size`` tokens and attend with the paged kernel (no beams).  With it,
    ``prompt_lengths`` gives the number of tokens of each right-padded prompt; row ``i`` of the result is then its prompt,
    what was generated, and padding (``eos_token_id`` or 0).
    ``repetition_penalty`` (of prompt and generated tokens), ``presence_penalty``, ``frequency_penalty`` (of generated tokens;
    each is a number or one number a row), ``logit_bias`` (a tensor ``[vocab]``, a mapping or pairs token -> value) and
    ``allowed_tokens`` change the logits before temperature and sampling (of beams: their log-probabilities), see
    :func:`oslo_b200.ops.logits.process_logits`.
    ``allowed_tokens(ids, lengths)`` is called every step with the tokens so far (``lengths``: int32 ``[rows]`` of those that
    count, ``None``: all) and returns ``[rows, vocab]`` booleans, packed words, or ``None`` for no restriction."""
    if paged_cache and not use_cache:
        raise ValueError("paged_cache is a kind of cache: it needs use_cache")
    if paged_cache and num_beams > 1:
        raise ValueError("the paged cache does not follow beams: use the dense cache for num_beams > 1")
    if prompt_lengths is not None and not paged_cache:
        raise ValueError("prompts of different lengths need paged_cache=True")
    rules = _LogitsRules(repetition_penalty, presence_penalty, frequency_penalty, logit_bias, allowed_tokens, num_beams)
    model.eval()
    pc = getattr(model, "parallel_context", None)
    if num_beams > 1 and use_cache and pc is not None and getattr(pc, "tensor_parallel_size", 1) > 1:
        from oslo_b200.distributed import ParallelMode as _PM

        if pc.tensor_parallel_mode != _PM.TENSOR_1D:
            # the N-D layouts split the batch over ranks, so a beam's parent may be cached on another rank: beams re-run
            # their prefix instead of reordering caches
            use_cache = False
    if num_beams > 1:
        return _beam_search(model, input_ids, max_new_tokens, num_beams, no_repeat_ngram_size, eos_token_id, length_penalty,
                            use_cache, rules)
    pick = _picker(do_sample, top_k, top_p)
    if prompt_lengths is not None:
        if no_repeat_ngram_size > 0:
            raise ValueError("n-gram blocking takes prompts of one length")
        return _generate_ragged(model, input_ids, [int(n) for n in prompt_lengths], max_new_tokens, pick, temperature, eos_token_id,
                                page_size, rules)
    ids = input_ids
    blocker = NGramRepeatBlock()
    done = torch.zeros(ids.shape[0], dtype=torch.bool, device=ids.device)
    cache = None
    if use_cache:
        cache = PagedDecodeCache(ids.shape[1] + max_new_tokens, page_size) if paged_cache else DecodeCache()
    prompts = torch.full((ids.shape[0],), ids.shape[1], dtype=torch.int32, device=ids.device) if rules.counts else None
    for _ in range(max_new_tokens):
        logits = rules(_logits(model, ids, cache), ids, None, prompts) / max(temperature, 1e-6)
        if no_repeat_ngram_size > 0:
            logits = blocker(ids, logits.contiguous(), ids.shape[0], ids.shape[1] - 1, 1, no_repeat_ngram_size)
        nxt = pick(logits)
        if eos_token_id is not None:
            nxt = torch.where(done.unsqueeze(1), torch.full_like(nxt, eos_token_id), nxt)
            done |= nxt.squeeze(1) == eos_token_id
        ids = torch.cat([ids, nxt], dim=1)
        if eos_token_id is not None and bool(done.all()):
            break
    return ids


def _picker(do_sample, top_k, top_p):
    """Next tokens ``[rows, 1]`` from logits ``[rows, vocab]``."""
    if not do_sample:
        return lambda logits: logits.argmax(-1, keepdim=True)
    from .kernels import sample_tokens

    return lambda logits: sample_tokens(logits, top_k, top_p)  # the device kernel on CUDA (no vocabulary sort)


def _generate_ragged(model, input_ids, lengths, max_new_tokens, pick, temperature, eos, page_size, rules):
    """Generation from right-padded prompts of different lengths over the paged cache."""
    if not getattr(getattr(model, "module", model), "ragged_prompts", False):
        raise ValueError(f"{type(model).__name__} takes prompts of one length")
    pc = getattr(model, "parallel_context", None)
    if pc is not None and getattr(pc, "tensor_parallel_size", 1) > 1:
        from oslo_b200.distributed import ParallelMode

        if pc.tensor_parallel_mode != ParallelMode.TENSOR_1D:
            raise ValueError("layouts that split the batch over ranks take prompts of one length")
    b, width = input_ids.shape
    if len(lengths) != b or min(lengths) < 1 or max(lengths) > width:
        raise ValueError(f"prompt_lengths has a number from 1 to {width} for each of the {b} prompts: got {lengths}")
    dev = input_ids.device
    pad = 0 if eos is None else eos
    length = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out = input_ids.new_full((b, width + max_new_tokens), pad)
    out[:, :width] = torch.where(torch.arange(width, device=dev) < length[:, None], input_ids, out[:, :width])
    cache = PagedDecodeCache(max(lengths) + max_new_tokens, page_size)
    prompts = length if rules.counts else None
    done = torch.zeros(b, dtype=torch.bool, device=dev)
    rows = torch.arange(b, device=dev)
    feed, counts, last = out[:, : max(lengths)], lengths, (length - 1).long()
    new = 0
    for new in range(1, max_new_tokens + 1):
        cache.begin_forward(counts)
        with decode_cache(cache):
            logits = model(input_ids=feed)
        cache.advance(feed.shape[1])
        logits = logits.logits if hasattr(logits, "logits") else logits[0]
        logits = _whole_logits(model, logits[rows, last]).float()
        logits = rules(logits, out, length, prompts) / max(temperature, 1e-6)
        nxt = pick(logits).squeeze(1)
        if eos is not None:
            nxt = torch.where(done, torch.full_like(nxt, eos), nxt)
            done |= nxt == eos
        out[rows, length.long()] = nxt
        length = length + 1
        feed, counts, last = nxt[:, None], None, torch.zeros_like(last)
        if eos is not None and bool(done.all()):
            break
    return out[:, : width + new]


def _beam_search(model, input_ids, max_new_tokens, beams, ngram, eos, length_penalty, use_cache=True, rules=None):
    b, prompt = input_ids.shape
    dev = input_ids.device
    ids = input_ids.repeat_interleave(beams, dim=0)  # [b * beams, t]
    scores = torch.zeros(b, beams, device=dev)
    scores[:, 1:] = float("-inf")  # all beams start identical: keep one alive
    finished = torch.zeros(b * beams, dtype=torch.bool, device=dev)
    blocker = NGramRepeatBlock()
    cache = DecodeCache() if use_cache else None
    prompts = torch.full((b * beams,), prompt, dtype=torch.int32, device=dev) if rules is not None and rules.counts else None
    for _ in range(max_new_tokens):
        lp = F.log_softmax(_logits(model, ids, cache), dim=-1)
        if rules is not None:
            lp = rules(lp, ids, None, prompts)
        if ngram > 0:
            lp = blocker(ids, lp.contiguous(), b, ids.shape[1] - 1, beams, ngram)
        vocab = lp.shape[-1]
        if eos is not None:
            # finished hypotheses may only extend with EOS at no cost
            frozen = torch.full_like(lp, float("-inf"))
            frozen[:, eos] = 0.0
            lp = torch.where(finished.unsqueeze(1), frozen, lp)
        cand = (scores.view(-1, 1) + lp).view(b, beams * vocab)
        top, idx = cand.topk(beams, dim=-1)
        src = idx // vocab + (torch.arange(b, device=dev) * beams).unsqueeze(1)
        tok = idx % vocab
        ids = torch.cat([ids[src.view(-1)], tok.view(-1, 1)], dim=1)
        if cache is not None:
            cache.reorder(src.view(-1))  # the surviving hypotheses keep the keys / values of the beams they extend
        scores = top
        if eos is not None:
            finished = finished[src.view(-1)] | (tok.view(-1) == eos)
            if bool(finished.all()):
                break
    new_len = ids.shape[1] - prompt
    final = scores / (max(new_len, 1) ** length_penalty)
    best = final.argmax(dim=-1) + torch.arange(b, device=dev) * beams
    return ids[best]
