"""Paged key / value cache for serving (``csrc/paged_cache_sm100a.cu``, ``csrc/paged_attention_sm100a.cu``).

Keys and values live in pools ``[pages, kv_heads, page_size, head_dim]``; ``block_table[b, j]`` is the page that holds tokens
``j * page_size ..`` of sequence ``b``, so sequences of any lengths share one pool and grow without being copied.

``paged_kv_append``   rotates new queries and keys by their positions and stores keys and values in their pages, one pass
``paged_attention``   softmax attention of the newest tokens over the pages
``PagedDecodeCache``  the paged counterpart of :class:`oslo_b200.ops.attention.DecodeCache`: pages are taken from a free list as
                      sequences grow, and the sequences of a batch may have different lengths

The functions are for inference: inputs that require a gradient or carry a forward derivative are refused.  On the GPU a page,
position or length outside its pool or table is skipped by the kernel and reported by ``oslo_b200.ops._lib.check_status()``; on the
CPU it raises.
"""
from __future__ import annotations

import ctypes
import math
import struct
from functools import lru_cache
from typing import List, Optional, Sequence

import torch

from . import _lib

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # of a device's current stream
_device = getattr(torch._C, "_cuda_getDevice", None)
MAX_HEAD_DIM = 256
MAX_SCALE = 2.0 ** 127  # times log2(e) it still is a 32-bit number
_INFERENCE = "the paged cache is for inference: call it under torch.no_grad() or detach its inputs"


def _check_pages(k_pages, v_pages, block_table, b: int, hd: int, dtype, device: int):
    """Raises unless pools and table fit ``b`` sequences of this type; returns what the kernels need of their layout."""
    shape, ks, vs, table = k_pages.shape, k_pages.stride(), v_pages.stride(), block_table.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError(f"k_pages and v_pages are [pages, kv_heads, page_size, head_dim], both alike: got {tuple(shape)} "
                         f"and {tuple(v_pages.shape)}")
    pages, hkv, page, d = shape
    if dtype not in _DT or k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise ValueError(f"queries, keys, values and pages share one of float32, float16, bfloat16: got {dtype}, {k_pages.dtype}, "
                         f"{v_pages.dtype}")
    if d != hd:
        raise ValueError(f"head_dim of the pages is {d}, of the tokens {hd}")
    if page == 0 or page % 16 or d == 0 or d % 8 or d > MAX_HEAD_DIM or hkv == 0:
        raise ValueError(f"page_size is a multiple of 16 and head_dim a multiple of 8 up to {MAX_HEAD_DIM}: got {page}, {d} "
                         f"({hkv} key heads)")
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    if ks[3] != 1 or vs[3] != 1 or ks[2] != d or vs[2] != d or (ks[0] | ks[1] | vs[0] | vs[1]) % 8 or (kp | vp) % 16:
        raise ValueError("the tokens of a head inside a page are contiguous, and pages and heads start on 16-byte boundaries: got "
                         f"strides {ks} and {vs}")
    if len(table) != 2 or table[0] != b or block_table.dtype != torch.int32:
        raise ValueError(f"block_table is int32 [{b}, pages per sequence]: got {block_table.dtype} {tuple(table)}")
    row, col = block_table.stride()
    width = table[1]
    if col != 1 and width > 1:
        raise ValueError(f"the rows of block_table are contiguous: got strides {(row, col)}")
    if k_pages.get_device() != device or v_pages.get_device() != device or block_table.get_device() != device:
        raise ValueError(f"tensors are on devices {device}, {k_pages.device}, {v_pages.device} and {block_table.device}")
    if width * page > 0x3FFFFFFF:
        raise ValueError("block_table spans more than 2**30 tokens")
    return pages, hkv, page, width, row, ks, vs, kp, vp


def _check_ints(name, t, b: int, device: int):
    if t.dtype != torch.int32 or t.shape != (b,) or not t.is_contiguous() or t.get_device() != device:
        raise ValueError(f"{name} is a contiguous int32 tensor [{b}] beside the other ones: got {t.dtype} {tuple(t.shape)} on {t.device}")


def _check_rope(rope, hd: int, device: int):
    cos, sin, rot, neox = rope
    if rot < 0 or rot % 2 or rot > hd:
        raise ValueError(f"rot_dim is even and at most {hd}: got {rot}")
    shape = cos.shape
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or len(shape) != 2 or shape[1] != rot // 2 or sin.shape != shape \
            or not cos.is_contiguous() or not sin.is_contiguous() or cos.get_device() != device or sin.get_device() != device:
        raise ValueError(f"the rotation's tables are contiguous float32 [positions, {rot // 2}] beside the other tensors: got "
                         f"{cos.dtype} {tuple(shape)} and {sin.dtype} {tuple(sin.shape)} on {cos.device} and {sin.device}")
    return cos, sin, rot, 1 if neox else 0, shape[0]


def _mask32(mask):
    """``mask`` in 32 bits; finite numbers stay finite: the lowest one of 64 bits hides nothing, as that of 32 bits does not."""
    if mask.dtype == torch.float64:
        most = torch.finfo(torch.float32).max
        mask = torch.where(mask.isfinite(), mask.clamp(-most, most), mask)
    return mask.float()


def _aligned(t):
    """``t`` with unit inner stride and 16-byte aligned heads (a copy where it has not), its strides and its address."""
    st, at = t.stride(), t.data_ptr()
    if st[3] == 1 and not ((st[0] | st[1] | st[2]) % (16 // t.element_size()) or at % 16):
        return t, st, at
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride(), t.data_ptr()


def paged_kv_append(k, v, k_pages, v_pages, block_table, start, count=None, q=None, rope=None):
    """Store new tokens in the paged cache, rotated by their positions.

    ``k``, ``v``: ``[b, s, kv_heads, head_dim]`` (any strides), token ``i`` of sequence ``b`` has position ``start[b] + i``.
    ``start``: int32 ``[b]``, the tokens that each sequence holds already.  ``count``: int32 ``[b]``, how many of the ``s`` tokens
    are real (the rest is padding and is not stored; ``None``: all).  ``rope = (cos, sin, rot_dim, neox)`` as for
    :func:`oslo_b200.ops.attention.qkv_attention` rotates keys and queries; the tables need a row for every position.
    Pages are written in place, everything else in them stays; two tokens with the same page and row are a mistake of the
    caller (either may be stored).

    Returns the rotated ``q`` ``[b, s, heads, head_dim]`` as a new tensor (rows of padding are zeros), or ``None`` without ``q``.
    """
    if k.is_cuda:
        out = _step(0, k, v, k_pages, v_pages, block_table, start, count, q, rope)
        if out is not NotImplemented:
            return out
    shape, dtype, dev = k.shape, k.dtype, k.get_device()
    if len(shape) != 4 or v.shape != shape or v.dtype != dtype or v.get_device() != dev:
        raise ValueError(f"k and v are [b, s, kv_heads, head_dim], both alike: got {tuple(shape)} {dtype} and {tuple(v.shape)} "
                         f"{v.dtype}")
    b, s, hkv, hd = shape
    pages, heads, page, width, row, kps, vps, kp, vp = _check_pages(k_pages, v_pages, block_table, b, hd, dtype, dev)
    if heads != hkv:
        raise ValueError(f"the pages hold {heads} key heads, the tokens {hkv}")
    _check_ints("start", start, b, dev)
    if count is not None:
        _check_ints("count", count, b, dev)
    hq = 0
    if q is not None:
        qshape = q.shape
        if len(qshape) != 4 or qshape[0] != b or qshape[1] != s or qshape[3] != hd or q.dtype != dtype or q.get_device() != dev:
            raise ValueError(f"q is [{b}, {s}, heads, {hd}] {dtype} beside k: got {tuple(qshape)} {q.dtype} on {q.device}")
        hq = qshape[2]
    cos, sin, rot, neox, positions = _check_rope(rope, hd, dev) if rope is not None else (None, None, 0, 1, 0)
    if _lib.carries_gradient(k, v, q, k_pages, v_pages, cos, sin):
        raise RuntimeError(_INFERENCE)
    if not k.is_cuda:
        return _append_reference(k, v, k_pages, v_pages, block_table, start, count, q, rope if rot else None)
    if dev != _device():
        with torch.cuda.device(dev):
            return paged_kv_append(k, v, k_pages, v_pages, block_table, start, count, q, rope)
    out, qs, qp, op = None, (0, 0, 0), 0, 0
    if q is not None:
        out = q.new_empty(qshape)
        if hq:
            q, qs, qp = _aligned(q)
            op = out.data_ptr()
    k, ks, kx = _aligned(k)
    v, vs, vx = _aligned(v)
    rc = _load()[0](_APPEND_ARGS.pack(
        qp, kx, vx, op, kp, vp, block_table.data_ptr(), start.data_ptr(), 0 if count is None else count.data_ptr(),
        cos.data_ptr() if rot else 0, sin.data_ptr() if rot else 0, _status_ptr(dev), _raw_stream(dev),
        qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], kps[0], kps[1], vps[0], vps[1], row,
        b, s, hq, hkv, hd, rot, neox, positions, page, width, pages, _DT[dtype]))
    if rc:
        raise RuntimeError(f"oslo_paged_kv_append failed ({rc})")
    return out


def paged_attention(q, k_pages, v_pages, block_table, lengths, scale: Optional[float] = None, mask=None):
    """Attention of the newest tokens over a paged cache.

    ``q``: ``[b, s, heads, head_dim]`` (any strides), the newest ``s`` tokens of each sequence; their keys and values are in the
    pages already.  ``lengths``: int32 ``[b]``, the tokens in each sequence, the new ones included: query ``i`` sees the first
    ``lengths[b] - s + 1 + i``.  ``heads`` is a multiple of the pages' ``kv_heads``; consecutive heads share one.
    ``mask``: additive, ``[b or 1, 1, s or 1, tokens]``, any floating type; tokens at ``-inf`` take no part, whatever they hold,
    nor does what lies behind a sequence's last token.  It covers the longest sequence.  A query that sees nothing gives zeros.
    ``scale``: up to ``2**127`` (default ``head_dim ** -0.5``).

    Returns ``[b, s, heads * head_dim]``, like :func:`oslo_b200.ops.attention.attention`.
    """
    if q.is_cuda:
        out = _step(1, q, k_pages, v_pages, block_table, lengths, scale, mask)
        if out is not NotImplemented:
            return out
    shape, dtype, dev = q.shape, q.dtype, q.get_device()
    if len(shape) != 4:
        raise ValueError(f"q is [b, s, heads, head_dim]: got {tuple(shape)}")
    b, s, hq, hd = shape
    if _lib.carries_gradient(q, k_pages, v_pages, mask):
        raise RuntimeError(_INFERENCE)
    pages, hkv, page, width, row, ks, vs, kp, vp = _check_pages(k_pages, v_pages, block_table, b, hd, dtype, dev)
    _check_ints("lengths", lengths, b, dev)
    group = hq // hkv
    if hq == 0 or group * hkv != hq:
        raise ValueError(f"{hq} query heads do not share {hkv} key heads evenly")
    scale = hd ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= MAX_SCALE:
        raise ValueError(f"scale is a number up to {MAX_SCALE:g}: got {scale}")
    if mask is not None:
        if mask.dim() != 4 or mask.shape[0] not in (1, b) or mask.shape[1] != 1 or mask.shape[2] not in (1, s) \
                or mask.get_device() != dev or not mask.is_floating_point():
            raise ValueError(f"mask is an additive floating tensor [{b} or 1, 1, {s} or 1, tokens] beside q: got {mask.dtype} "
                             f"{tuple(mask.shape)} on {mask.device}")
        mask = _mask32(mask)
    if not q.is_cuda:
        return _attention_reference(q, k_pages, v_pages, block_table, lengths, scale, mask)
    if dev != _device():
        with torch.cuda.device(dev):
            return paged_attention(q, k_pages, v_pages, block_table, lengths, scale, mask)
    q, qs, qp = _aligned(q)
    out = q.new_empty((b, s, hq * hd))
    mptr = mb = mt = 0
    mlen = -1
    if mask is not None:
        mlen = mask.shape[3]
        mask = mask.expand(b, 1, s, mlen)
        if mask.stride(3) != 1:
            mask = mask.contiguous()
        mptr, mb, mt = mask.data_ptr(), mask.stride(0), mask.stride(2)
    args = [qp, kp, vp, block_table.data_ptr(), lengths.data_ptr(), mptr, out.data_ptr(), 0, _status_ptr(dev), _raw_stream(dev),
            qs[0], qs[1], qs[2], ks[0], ks[1], vs[0], vs[1], row, mb, mt,
            b, s, hkv, group, hd, page, width, pages, mlen, _DT[dtype], scale]
    _, attend, workspace = _load()
    room = workspace(_ATTEND_ARGS.pack(*args))
    if room > 0:
        ws = torch.empty(room, dtype=torch.uint8, device=q.device)
        args[7] = ws.data_ptr()
    rc = attend(_ATTEND_ARGS.pack(*args)) if room >= 0 else room
    if rc:
        raise RuntimeError(f"oslo_paged_attention failed ({rc})")
    return out


_direct = None


def _step(which, *args):
    """The call through the step module, where its arguments are ordinary; else ``NotImplemented``."""
    global _direct
    if _direct is None:
        module = _lib.step_calls()
        _direct = (module.paged_kv_append, module.paged_attention) if module is not None else (_not_built, _not_built)
    out = _direct[which](*args)
    if out is not NotImplemented:
        _lib.native_calls += 1
    return out


def _not_built(*args):
    return NotImplemented


# arguments travel as one struct of eight-byte fields: ctypes converts one value instead of forty
_APPEND_ARGS = struct.Struct("=39q")
_ATTEND_ARGS = struct.Struct("=30qd")
@lru_cache(maxsize=None)
def _load():
    dll, lib = _lib._load_cuda_lib(), _lib.cuda_lib()
    for name in ("oslo_paged_kv_append", "oslo_paged_attention", "oslo_paged_attention_workspace_bytes"):
        getattr(dll, name).argtypes = [ctypes.c_char_p]
    dll.oslo_paged_attention_workspace_bytes.restype = ctypes.c_longlong
    return lib.oslo_paged_kv_append, lib.oslo_paged_attention, lib.oslo_paged_attention_workspace_bytes


@lru_cache(maxsize=None)
def _status_ptr(device: int) -> int:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("call the paged cache's functions once on a device before capturing them: their status word is made then")
    ptr = _lib.status_word(torch.device("cuda", device)).data_ptr()
    module = _lib.step_calls()
    if module is not None:
        module.status(device, ptr)  # from now on the step module takes this device's calls
    return ptr


# ------------------------------------------------------------------------------------------------ the cache of a generation
class PagedDecodeCache:
    """Keys and values of the tokens a model has already seen, in pages (``with decode_cache(cache): model(ids)``).

    A drop-in for :class:`oslo_b200.ops.attention.DecodeCache` except for beam search: pages of ``page_size`` tokens are taken
    from a pool as sequences grow, nothing is copied when they do, and the sequences of the batch may have different lengths.
    The first forward takes the prompts, padded on the right; ``begin_forward(counts)`` says how many tokens of each row are real.
    Its attention runs over the prompts themselves; every later forward stores its tokens and attends over the pages.  The
    pools ``[pages, kv_heads, page_size, head_dim]`` of a layer are made when its first keys come.

    ``max_tokens``: tokens a sequence may reach; ``num_pages``: pages of a layer's pool (default: enough for every sequence).
    """

    def __init__(self, max_tokens: int, page_size: int = 64, num_pages: Optional[int] = None):
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"page_size is a positive multiple of 16: got {page_size}")
        if max_tokens <= 0:
            raise ValueError(f"max_tokens is positive: got {max_tokens}")
        self.max_tokens, self.page_size, self.num_pages = max_tokens, page_size, num_pages
        self.k_pages: List[torch.Tensor] = []
        self.v_pages: List[torch.Tensor] = []
        self.lengths: List[int] = []  # tokens of each sequence
        self.pages: List[List[int]] = []  # pages of each sequence, in order
        self.block_table: Optional[torch.Tensor] = None  # int32 [batch, pages of max_tokens], on the device
        self._free: List[int] = []
        self._held = self._after = None  # int32 [batch] on the device: tokens before and after this forward
        self._counts: Optional[List[int]] = None
        self._layer = self._new = 0

    @property
    def offset(self) -> int:
        """Tokens of every sequence, where all have as many."""
        if len(set(self.lengths)) > 1:
            raise RuntimeError("the sequences of this cache have different lengths: this model takes one position for all of them")
        return self.lengths[0] if self.lengths else 0

    @property
    def longest(self) -> int:
        return max(self.lengths, default=0)

    def positions(self, s: int, device) -> torch.Tensor:
        """Positions of the next ``s`` tokens: ``[1, s]`` where all sequences have as many, else ``[batch, s]``."""
        new = torch.arange(s, device=device)
        return (new + self.offset).unsqueeze(0) if len(set(self.lengths)) <= 1 else self._held.unsqueeze(1) + new

    def begin_forward(self, counts: Optional[Sequence[int]] = None):
        self._layer, self._counts = 0, None if counts is None else [int(c) for c in counts]

    def advance(self, n: int):
        """After a forward over ``n`` tokens a row."""
        self.lengths = [have + new for have, new in zip(self.lengths, self._counts or [n] * len(self.lengths))]
        self._held, self._counts = self._after, None

    def reorder(self, index: torch.Tensor):
        raise RuntimeError("the paged cache does not follow beams: search beams over the dense cache")

    def _grow(self, b: int, s: int, device):
        """Pages for the tokens of this forward (once per forward, before its first layer stores any)."""
        if self.block_table is None:
            width = -(-self.max_tokens // self.page_size)
            if self.num_pages is None:
                self.num_pages = b * width
            self.lengths, self.pages = [0] * b, [[] for _ in range(b)]
            self._free = list(range(self.num_pages - 1, -1, -1))
            self._rows = torch.zeros(b, width, dtype=torch.int32)
            self.block_table = self._rows.to(device)
            self._held = torch.zeros(b, dtype=torch.int32, device=device)
        counts = self._counts if self._counts is not None else [s] * b
        if len(self.lengths) != b or len(counts) != b or min(counts) < 0 or max(counts) > s:
            raise ValueError(f"the cache holds {len(self.lengths)} sequences; this forward has {b} rows of {s} tokens, of which {counts} "
                             "are real")
        need = [-(-(have + new) // self.page_size) - len(own) for have, new, own in zip(self.lengths, counts, self.pages)]
        if max(have + new for have, new in zip(self.lengths, counts)) > self.max_tokens:
            raise ValueError(f"a sequence would pass max_tokens = {self.max_tokens}")
        if sum(n for n in need if n > 0) > len(self._free):
            raise RuntimeError(f"the page pool is exhausted: {sum(n for n in need if n > 0)} pages are needed, {len(self._free)} of "
                               f"{self.num_pages} are free")
        for row, n in enumerate(need):
            for _ in range(n):
                self._rows[row, len(self.pages[row])] = self._free[-1]
                self.pages[row].append(self._free.pop())
        if any(n > 0 for n in need):
            self.block_table = self._rows.to(device)
        self._new = s
        if self._counts is None:
            self._count, self._after = None, self._held + s
        else:
            self._count = torch.tensor(counts, dtype=torch.int32, device=device)
            self._after = self._held + self._count

    def attend(self, q, k, v, scale: Optional[float] = None, rope=None, mask=None):
        """What a layer's causal attention calls: ``q [b, s, heads, head_dim]``, ``k``, ``v`` ``[b, s, kv_heads, head_dim]`` of the
        new tokens -> ``[b, s, heads * head_dim]``.  ``rope = (cos, sin, rot_dim, neox)`` rotates queries and keys first; ``mask`` is
        additive over all tokens so far.  Layers are told apart by the order of their calls."""
        from .attention import dense_attention
        from .softmax import apply_rope

        b, s, hq, hd = q.shape
        if self._layer == 0:
            self._grow(b, s, q.device)
        i = self._layer
        self._layer += 1
        if i == len(self.k_pages):
            for pools in (self.k_pages, self.v_pages):
                pools.append(torch.zeros(self.num_pages, k.shape[2], self.page_size, hd, dtype=k.dtype, device=k.device))
        pools = self.k_pages[i], self.v_pages[i]
        if self.longest == 0:  # the prompts attend to themselves
            if rope is not None:
                cos, sin, rot, neox = rope
                pos = torch.arange(s, device=q.device).repeat(b)
                q = apply_rope(q.contiguous(), cos, sin, rot, neox, positions=pos)
                k = apply_rope(k.contiguous(), cos, sin, rot, neox, positions=pos)
            paged_kv_append(k, v, *pools, self.block_table, self._held, count=self._count)
            if k.shape[2] != hq:
                k, v = (t.repeat_interleave(hq // t.shape[2], dim=2) for t in (k, v))
            return dense_attention(q, k, v, True, scale, mask)
        if self._count is not None and min(self._counts) < s:
            raise ValueError("only prompts may be padded: a later forward takes as many tokens of every row")
        turned = paged_kv_append(k, v, *pools, self.block_table, self._held, q=q, rope=rope)
        if mask is not None:
            mask = mask[..., -s:, :]
        return paged_attention(turned, *pools, self.block_table, self._after, scale, mask)


# ------------------------------------------------------------------------------------------------ plain forms
def _rows_of(block_table, page: int, pages: int, row: int, n: int):
    """Page and row in it of tokens ``0 .. n`` of one sequence."""
    if n > block_table.shape[1] * page:
        raise ValueError(f"sequence {row} has {n} tokens, its row of the block table holds {block_table.shape[1] * page}")
    t = torch.arange(n, device=block_table.device)
    where = block_table[row].long()[t // page]
    if n and (int(where.min()) < 0 or int(where.max()) >= pages):
        raise ValueError(f"block_table names a page outside the pool of {pages}")
    return where, t % page


def _append_reference(k, v, k_pages, v_pages, block_table, start, count, q, rope):
    from .softmax import rope_reference

    b, s = k.shape[:2]
    pages, _, page, _ = k_pages.shape
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device) if q is not None else None
    for r in range(b):
        first, n = int(start[r]), s if count is None else max(0, min(s, int(count[r])))
        if first < 0 or (n and rope is not None and first + n > rope[0].shape[0]):
            raise ValueError(f"sequence {r} has positions {first} to {first + n}, the rotation's tables do not")
        where, at = (t[first:] for t in _rows_of(block_table, page, pages, r, first + n)) if n else (None, None)
        if not n:
            continue
        turn = lambda x: x
        if rope is not None:
            cos, sin, rot, neox = rope
            pos = torch.arange(first, first + n, device=k.device)
            turn = lambda x: rope_reference(x, cos, sin, rot, neox, positions=pos)
        k_pages[where, :, at] = turn(k[r, :n])
        v_pages[where, :, at] = v[r, :n]
        if out is not None:
            out[r, :n] = turn(q[r, :n])
    return out


def _attention_reference(q, k_pages, v_pages, block_table, lengths, scale, mask):
    b, s, hq, hd = q.shape
    pages, hkv, page, _ = k_pages.shape
    out = torch.zeros(b, s, hq, hd, dtype=torch.float32, device=q.device)
    for r in range(b):
        n = max(0, int(lengths[r]))
        if mask is not None and n > mask.shape[3]:
            raise ValueError(f"the mask covers {mask.shape[3]} tokens, sequence {r} has {n}")
        where, at = _rows_of(block_table, page, pages, r, n)
        k, v = (t[where, :, at].float().repeat_interleave(hq // hkv, dim=1) for t in (k_pages, v_pages))  # [n, hq, hd]
        for i in range(s):
            end = n - s + 1 + i
            if end <= 0:
                continue
            x = torch.einsum("hd,nhd->hn", q[r, i].float(), k[:end]) * scale
            vv = v[:end]
            if mask is not None:
                add = mask[r % mask.shape[0], 0, i % mask.shape[2], :end]
                keep = add != float("-inf")
                x, vv = (x + add)[:, keep], vv[keep]
            if x.shape[1]:
                out[r, i] = torch.einsum("hn,nhd->hd", torch.softmax(x, dim=-1), vv)
    return out.to(q.dtype).view(b, s, hq * hd)
