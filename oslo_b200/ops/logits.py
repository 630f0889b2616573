"""Penalties for repeated tokens, biases and grammar masks on next-token logits (``csrc/logits_sm100a.cu``).

``process_logits(logits, tokens, ...)`` changes the logits of one decoding step before a token is picked from them;
``pack_token_mask(mask)`` packs a boolean mask of allowed tokens into the 32-bit words that it takes.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Union

import torch

from . import _lib

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_REPETITION = 2.0 ** 126  # its reciprocal still is a normal 32-bit number, and the other way round
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # of a device's current stream
_device = getattr(torch._C, "_cuda_getDevice", None)


def pack_token_mask(mask: torch.Tensor) -> torch.Tensor:
    """Boolean ``[rows, vocab]`` (true = allowed) -> int32 ``[rows, ceil(vocab / 32)]``; token ``j`` is bit ``j % 32`` of word
    ``j // 32``."""
    if mask.dim() != 2 or mask.dtype != torch.bool:
        raise ValueError(f"mask is boolean [rows, vocab]: got {mask.dtype} {tuple(mask.shape)}")
    rows, v = mask.shape
    bits = torch.nn.functional.pad(mask, (0, -v % 32)).view(rows, -1, 32).long()
    words = (bits << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _per_row(name, p, rows: int, device):
    """(tensor or None, scalar) of a penalty given as a number or as one number a row."""
    if isinstance(p, torch.Tensor):
        if p.shape != (rows,) or p.device != device or not p.is_floating_point():
            raise ValueError(f"{name} is a number or a floating tensor [{rows}] on {device}: got {p.dtype} {tuple(p.shape)} on {p.device}")
        return (p if p.dtype == torch.float32 and p.is_contiguous() else p.float().contiguous()), 0.0
    return None, float(p)


def _partly_over(out, x) -> bool:
    """Whether rows of ``out`` lie over rows of ``x`` without being the same rows (``x`` whose rows are not contiguous is copied)."""
    rows, v = x.shape
    a, b = out.data_ptr(), x.data_ptr()
    if rows * v == 0 or (v > 1 and x.stride(1) != 1) or (a == b and (rows == 1 or out.stride(0) == x.stride(0))):
        return False
    size = x.element_size()
    row, so, sx = v * size, out.stride(0) * size, x.stride(0) * size
    if a + (rows - 1) * so + row <= b or b + (rows - 1) * sx + row <= a:
        return False
    mine, theirs = a + torch.arange(rows, device="cpu") * so, b + torch.arange(rows, device="cpu") * sx
    near = torch.searchsorted(theirs, mine - row, right=True).clamp(max=rows - 1)  # the first that ends behind the row's beginning
    return bool(((theirs[near] > mine - row) & (theirs[near] < mine + row)).any())


def process_logits(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, token_lengths: Optional[torch.Tensor] = None,
                   prompt_lengths: Optional[torch.Tensor] = None, repetition_penalty: Union[float, torch.Tensor] = 1.0,
                   presence_penalty: Union[float, torch.Tensor] = 0.0, frequency_penalty: Union[float, torch.Tensor] = 0.0,
                   bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Next-token ``logits [rows, vocab]`` after penalties, biases and a grammar mask, in this order:

    1. a token that occurs in the row's history has its logit ``x`` divided by ``repetition_penalty`` (multiplied where ``x`` is
       not positive);
    2. a token that was generated ``c > 0`` times loses ``presence_penalty + frequency_penalty * c``;
    3. ``bias`` is added;
    4. tokens that are not ``allowed`` become ``-inf``.

    ``tokens``: int64 or int32 ``[rows, length]``, the history; ids outside the vocabulary are ignored.  ``token_lengths``: int32
    ``[rows]``, how many of them count (``None``: all).  ``prompt_lengths``: int32 ``[rows]``, how many of those are the prompt, not
    generated (``None``: none).  The penalties are numbers or floating tensors ``[rows]``, ``repetition_penalty`` from ``2**-126`` to
    ``2**126``.  ``bias``: ``[vocab]`` or ``[rows, vocab]``.
    ``allowed``: int32 ``[rows or 1, ceil(vocab / 32)]`` from :func:`pack_token_mask`; a row that allows nothing is all ``-inf``.
    The result is a new tensor, or ``out`` (which may be ``logits``).  For inference: tensors that require a gradient or carry a
    forward derivative are refused.
    """
    if logits.is_cuda and out is None:
        y = _step(logits, tokens, token_lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty, bias, allowed)
        if y is not NotImplemented:
            return y
    dtype, dev = logits.dtype, logits.device
    if logits.dim() != 2 or dtype not in _DT:
        raise ValueError(f"logits are float32, float16 or bfloat16 [rows, vocab]: got {dtype} {tuple(logits.shape)}")
    if _lib.carries_gradient(*(t for t in (logits, bias, repetition_penalty, presence_penalty, frequency_penalty, out)
                               if isinstance(t, torch.Tensor))):
        raise RuntimeError("process_logits is for inference: call it under torch.no_grad() or detach its inputs")
    rows, v = logits.shape
    rep, rep_s = _per_row("repetition_penalty", repetition_penalty, rows, dev)
    pres, pres_s = _per_row("presence_penalty", presence_penalty, rows, dev)
    freq, freq_s = _per_row("frequency_penalty", frequency_penalty, rows, dev)
    if rep is None and not 1 / MAX_REPETITION <= rep_s <= MAX_REPETITION:
        raise ValueError(f"repetition_penalty is positive, from 1 / {MAX_REPETITION:g} to {MAX_REPETITION:g}: got {rep_s}")
    if tokens is None:
        if token_lengths is not None or prompt_lengths is not None:
            raise ValueError("token_lengths and prompt_lengths describe tokens, which are missing")
        if rep is not None or pres is not None or freq is not None or rep_s != 1.0 or pres_s or freq_s:
            raise ValueError("the penalties need the tokens of each row's history")
    else:
        if tokens.dim() != 2 or tokens.shape[0] != rows or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != dev:
            raise ValueError(f"tokens are int64 or int32 [{rows}, length] on {dev}: got {tokens.dtype} {tuple(tokens.shape)} on "
                             f"{tokens.device}")
        for name, t in (("token_lengths", token_lengths), ("prompt_lengths", prompt_lengths)):
            if t is not None and (t.dtype != torch.int32 or t.shape != (rows,) or t.device != dev or not t.is_contiguous()):
                raise ValueError(f"{name} is a contiguous int32 tensor [{rows}] on {dev}: got {t.dtype} {tuple(t.shape)} on {t.device}")
    if bias is not None:
        if bias.shape not in ((v,), (rows, v)) or not bias.is_floating_point() or bias.device != dev:
            raise ValueError(f"bias is a floating tensor [{v}] or [{rows}, {v}] on {dev}: got {bias.dtype} {tuple(bias.shape)} on "
                             f"{bias.device}")
        bias = bias if bias.dtype == torch.float32 else bias.float()
    if allowed is not None and (allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.shape[0] not in (1, rows)
                                or allowed.shape[1] != (v + 31) // 32 or allowed.device != dev):
        raise ValueError(f"allowed is int32 [{rows} or 1, {(v + 31) // 32}] on {dev}: got {allowed.dtype} {tuple(allowed.shape)} on "
                         f"{allowed.device}")
    if out is not None and (out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev or out.stride(1) != 1):
        raise ValueError(f"out is like the logits, with contiguous rows: got {out.dtype} {tuple(out.shape)} on {out.device}")
    if out is not None and ((rows > 1 and out.stride(0) < v) or _partly_over(out, logits)):
        raise ValueError("out has rows of its own, and is the logits or apart from them")
    if not logits.is_cuda:
        y = _reference(logits, tokens, token_lengths, prompt_lengths, *(t if t is not None else s for t, s in
                       ((rep, rep_s), (pres, pres_s), (freq, freq_s))), bias, allowed)
        return y if out is None else out.copy_(y)
    if dev.index != _device():
        with torch.cuda.device(dev):
            return process_logits(logits, tokens, token_lengths, prompt_lengths, repetition_penalty, presence_penalty,
                                  frequency_penalty, bias, allowed, out)
    xs = logits.stride()
    if xs[1] != 1:
        logits = logits.contiguous()
        xs = logits.stride()
    y = torch.empty((rows, v), dtype=dtype, device=dev) if out is None else out
    length = tok_stride = 0
    if tokens is not None and tokens.shape[1]:
        length, ts = tokens.shape[1], tokens.stride()
        if ts[1] != 1:
            tokens = tokens.contiguous()
            ts = tokens.stride()
        tok_stride = ts[0]
    bias_stride = allowed_stride = 0
    if bias is not None:
        bias = bias if bias.stride(-1) == 1 else bias.contiguous()
        bias_stride = bias.stride(0) if bias.dim() == 2 else 0
    if allowed is not None:
        allowed = allowed if allowed.stride(1) == 1 else allowed.contiguous()
        allowed_stride = allowed.stride(0) if allowed.shape[0] > 1 else 0
    rc = _fn()(_ARGS.pack(
        logits.data_ptr(), y.data_ptr(), tokens.data_ptr() if length else 0, 0 if token_lengths is None else token_lengths.data_ptr(),
        0 if prompt_lengths is None else prompt_lengths.data_ptr(), 0 if rep is None else rep.data_ptr(),
        0 if pres is None else pres.data_ptr(), 0 if freq is None else freq.data_ptr(), 0 if bias is None else bias.data_ptr(),
        0 if allowed is None else allowed.data_ptr(), _raw_stream(dev.index), xs[0], v if out is None else out.stride(0), tok_stride,
        bias_stride, allowed_stride, rows, v, length, 1 if length and tokens.dtype == torch.int64 else 0, _DT[dtype], rep_s, pres_s,
        freq_s))
    if rc:
        raise RuntimeError(f"oslo_process_logits failed ({rc})")
    return y


_direct = None


def _step(*args):
    """The call through the step module, where its arguments are ordinary; else ``NotImplemented``."""
    global _direct
    if _direct is None:
        module = _lib.step_calls()
        _direct = module.process_logits if module is not None else lambda *args: NotImplemented
    y = _direct(*args)
    if y is not NotImplemented:
        _lib.native_calls += 1
    return y


_ARGS = struct.Struct("=21q3d")  # arguments travel as one struct of eight-byte fields
_native = None


def _fn():
    global _native
    if _native is None:
        _lib._load_cuda_lib().oslo_process_logits.argtypes = [ctypes.c_char_p]
        _native = _lib.cuda_lib().oslo_process_logits
    return _native


def _reference(logits, tokens, token_lengths, prompt_lengths, rep, pres, freq, bias, allowed):
    x = logits.float()
    rows, v = x.shape
    col = lambda p: p[:, None] if isinstance(p, torch.Tensor) else p
    if tokens is not None and tokens.shape[1] and v:
        t = torch.arange(tokens.shape[1], device=x.device)
        known = (tokens >= 0) & (tokens < v)
        if token_lengths is not None:
            known &= t < token_lengths[:, None]
        made = known if prompt_lengths is None else known & (t >= prompt_lengths[:, None])
        ids = tokens.long().clamp(0, v - 1)
        seen = torch.zeros_like(x).scatter_add_(1, ids, known.float()) > 0
        c = torch.zeros_like(x).scatter_add_(1, ids, made.float())
        x = torch.where(seen, torch.where(x > 0, x / col(rep), x * col(rep)), x)
        x = torch.where(c > 0, x - col(pres) - col(freq) * c, x)
    if bias is not None:
        x = x + bias
    if allowed is not None:
        j = torch.arange(v, device=x.device)
        x = x.masked_fill(((allowed[:, j // 32] >> (j % 32).to(torch.int32)) & 1) == 0, float("-inf"))
    return x.to(logits.dtype)
