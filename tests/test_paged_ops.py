"""The paged key / value cache operators and the logits operator against plain statements of their formulas in 64 bits.

Tolerances count roundings.  A result rounded to type t is off by at most ``eps(t) / 2`` of its value; what happens before that
rounding is bounded per formula (see ``_attend_bound`` and ``_turn_bound``), with u = 2**-24 the unit rounding of 32 bits.
"""
import itertools
import math

import pytest
import torch

from oslo_b200.nn import functional as OF

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _half_step(t):
    return torch.finfo(t).eps / 2


def _sync_status(dev):
    if dev == "cuda":
        from oslo_b200.ops import _lib

        torch.cuda.synchronize()
        _lib.check_status()


def _pool(lens, page, hkv, d, dtype, dev, spare=3, fill=None):
    """Pools and a table with scattered pages for sequences of these capacities (tokens)."""
    need = [max(1, -(-n // page)) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages).tolist()
    width = max(need)
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    for r, n in enumerate(need):
        table[r, :n] = torch.tensor([order.pop() for _ in range(n)])
    k, v = (torch.randn(pages, hkv, page, d).to(dtype).to(dev) for _ in range(2))
    if fill is not None:
        k.fill_(fill)
        v.fill_(fill)
    return k, v, table.to(dev)


def _seq(pages, table, r, n):
    page = pages.shape[2]
    t = torch.arange(n, device=pages.device)
    return pages[table[r].long()[t // page], :, t % page]  # [n, hkv, d]


# ------------------------------------------------------------------------------------------------ append
def _turn(x, pos, rope):
    """Rotation in 64 bits and the sum of the magnitudes of its two products."""
    y, mag = x.double().clone(), x.double().abs()
    if rope is None:
        return y, torch.zeros_like(y)
    cos, sin, rot, neox = rope
    mag = torch.zeros_like(y)
    for j in range(rot // 2):
        i0, i1 = (j, j + rot // 2) if neox else (2 * j, 2 * j + 1)
        c, s = cos[pos, j].double()[:, None], sin[pos, j].double()[:, None]
        a, b = x[..., i0].double(), x[..., i1].double()
        y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
        mag[..., i0] = (a * c).abs() + (b * s).abs()
        mag[..., i1] = (b * c).abs() + (a * s).abs()
    return y, mag


def _turn_bound(y, mag, dtype):
    # two products and a sum in 32 bits: at most 3 u of the magnitudes; then one rounding (fp16 below 2**-14: steps of 2**-24)
    pre = 3 * U * mag
    return _half_step(dtype) * (y.abs() + pre) + pre + (2.0 ** -25 if dtype == torch.float16 else 1e-37)


def _append_case(dev, dtype, b, s, hq, hkv, d, rot, neox, page, starts, counts, fused):
    torch.manual_seed(b * 100 + s * 10 + d + rot)
    width = hq + 2 * hkv
    if fused:  # views into one projection output, heads interleaved
        x = torch.randn(b, s, width, d).to(dtype).to(dev)
        q, k, v = x[:, :, :hq], x[:, :, hq : hq + hkv], x[:, :, hq + hkv :]
    else:  # head-major storage that starts off the 16-byte grid, other strides
        x = torch.randn(b * s * width * d + 1).to(dtype).to(dev)[1:].view(b, width, s, d).transpose(1, 2)
        q, k, v = x[:, :, :hq], x[:, :, hq : hq + hkv], x[:, :, hq + hkv :]
    start = torch.tensor(starts, dtype=torch.int32, device=dev)
    count = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev)
    n = [s] * b if counts is None else counts
    kp, vp, table = _pool([a + s for a in starts], page, hkv, d, dtype, dev)
    rope = None
    if rot:
        cos, sin = OF.rope_tables(max(starts) + s, rot, device=dev)
        rope = (cos, sin, rot, neox)
    want_k, want_v = kp.double().clone(), vp.double().clone()
    tol_k = torch.zeros_like(want_k)
    want_q = torch.zeros(b, s, hq, d, dtype=torch.float64, device=dev)
    tol_q = torch.zeros_like(want_q)
    for r in range(b):
        if not n[r]:
            continue
        pos = torch.arange(starts[r], starts[r] + n[r], device=dev)
        y, mag = _turn(k[r, : n[r]], pos, rope)
        where, at = table[r].long()[pos // page], pos % page
        want_k[where, :, at], want_v[where, :, at] = y, v[r, : n[r]].double()
        tol_k[where, :, at] = _turn_bound(y, mag, dtype) if rope else 0.0
        y, mag = _turn(q[r, : n[r]], pos, rope)
        want_q[r, : n[r]] = y
        tol_q[r, : n[r]] = _turn_bound(y, mag, dtype) if rope else 0.0
    before = x.clone()
    got = OF.paged_kv_append(k, v, kp, vp, table, start, count=count, q=q if hq else None, rope=rope)
    _sync_status(dev)
    assert torch.equal(x, before)
    assert ((kp.double() - want_k).abs() <= tol_k).all()
    assert torch.equal(vp.double(), want_v)
    if hq:
        assert ((got.double() - want_q).abs() <= tol_q).all()
    else:
        assert got is None


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,s,hq,hkv,d,rot,neox,page,starts,counts,fused", [
    (1, 1, 4, 4, 64, 16, True, 16, [0], None, True),
    (3, 1, 8, 2, 128, 128, True, 16, [0, 15, 16], None, True),
    (2, 37, 3, 1, 96, 24, True, 32, [5, 0], [37, 11], True),      # rot / 2 = 12: partners off the 16-byte grid
    (2, 5, 4, 2, 80, 20, False, 16, [31, 2], [0, 5], False),      # a sequence without new tokens
    (2, 3, 2, 2, 256, 256, False, 64, [62, 7], None, False),
    (2, 4, 0, 3, 40, 40, True, 48, [45, 1], None, True),          # no queries
    (4, 1, 6, 6, 8, 0, True, 16, [0, 1, 2, 300], None, True),     # no rotation
    (2, 2, 2, 1, 72, 2, True, 16, [3, 4], None, False),
])
def test_append_stores_rotated_tokens_and_leaves_the_rest(dev, dtype, b, s, hq, hkv, d, rot, neox, page, starts, counts, fused):
    _append_case(dev, dtype, b, s, hq, hkv, d, rot, neox, page, starts, counts, fused)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("s,hkv", [(1000, 8), (1, 32)])
def test_append_many_tokens(dtype, s, hkv):
    _append_case("cuda", dtype, 7, s, 2 * hkv, hkv, 128, 128, True, 64, [0, 63, 64, 1, 500, 9, 128], [s, s, 0, 1, s, s // 2, s], True)


# ------------------------------------------------------------------------------------------------ attention
def _attend_bound(q, k, x, p, v, o, scale, dtype):
    """What the result may be off by.  x: scores, p: weights, both in 64 bits.

    Scores: d products summed in 32 bits, 2 d u of the sum of their magnitudes (fp32 inputs: 2**-21 more for the split into
    tf32 parts), plus scaling and mask, 4 u of the score.  A score off by e changes a weight by a factor of at most exp(2 e)
    (its own and the sum's).  exp itself: 2**-22; weights enter the product in two 16-bit parts: 2**-16; n of them summed
    in 32 bits: n u (blockwise sums and joins included)."""
    d, n = q.shape[-1], x.shape[-1]
    mags = q.abs() @ k.abs().T * abs(scale)
    split = 2.0 ** -21 if dtype == torch.float32 else 0.0
    e = ((2 * d * U + split) * mags + 4 * U * torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))).amax(-1, keepdim=True)
    part = 2.0 ** -20 if dtype == torch.float32 else 2.0 ** -16
    pre = (torch.expm1(2 * e) + 2.0 ** -21 + part + 2 * (n + 16) * U) * (p @ v.abs())
    # fp16 weights below 2**-14 have steps of 2**-24 (both parts): at most 2**-25 each, unnormalised, so of a sum of at least 1
    tiny = 2.0 ** -24 * v.abs().sum(0) if dtype == torch.float16 else 0.0
    return _half_step(dtype) * (o.abs() + pre) + pre + tiny + 1e-30


def _attend_exact(q, kp, vp, table, lens, scale, mask):
    b, s, hq, d = q.shape
    hkv = kp.shape[1]
    out = torch.zeros(b, s, hq, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for r, n in enumerate(lens):
        k, v = _seq(kp, table, r, max(n, 0)).double(), _seq(vp, table, r, max(n, 0)).double()
        for i, h in itertools.product(range(s), range(hkv)):
            end = n - s + 1 + i
            if end <= 0:
                continue
            g = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            keep = torch.ones(end, dtype=torch.bool, device=q.device)
            add = torch.zeros(end, dtype=torch.float64, device=q.device)
            if mask is not None:
                add = mask[r % mask.shape[0], 0, i % mask.shape[2], :end].double()
                keep = add != -math.inf
            if not keep.any():
                continue
            kk, vv = k[:end, h][keep], v[:end, h][keep]
            qq = q[r, i, g].double()
            x = qq @ kk.T * scale + add[keep]
            p = torch.softmax(x, -1)
            out[r, i, g] = p @ vv
            tol[r, i, g] = _attend_bound(qq, kk, x, p, vv, out[r, i, g], scale, q.dtype)
    return out.view(b, s, -1), tol.view(b, s, -1)


def _attend_case(dev, dtype, s, hq, hkv, d, page, lens, mask=None, scale=None, fill=None, qscale=1.0):
    torch.manual_seed(sum(lens) + d + hq)
    b = len(lens)
    kp, vp, table = _pool(lens, page, hkv, d, dtype, dev)
    if fill is not None:  # whatever lies outside the sequences
        used = torch.zeros(kp.shape[0], page, dtype=torch.bool, device=dev)
        for r, n in enumerate(lens):
            t = torch.arange(n, device=dev)
            used[table[r].long()[t // page], t % page] = True
        kp.masked_fill_(~used[:, None, :, None], fill)
        vp.masked_fill_(~used[:, None, :, None], fill)
    q = (torch.randn(b, s, hq + 1, d) * qscale).to(dtype).to(dev)[:, :, 1:]
    if mask is not None:
        mask = mask.to(dev)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = OF.paged_attention(q, kp, vp, table, lengths, scale=scale, mask=mask)
    _sync_status(dev)
    want, tol = _attend_exact(q, kp, vp, table, lens, 1 / math.sqrt(d) if scale is None else scale, mask)
    assert got.shape == (b, s, hq * d) and got.dtype == dtype
    off = (got.double() - want).abs()
    assert (off <= tol).all(), (off / tol.clamp(min=1e-30)).nan_to_num(nan=math.inf).max().item()
    return got


SHAPES = [  # s, hq, hkv, d, page, lens
    (1, 1, 1, 64, 16, [1]),
    (1, 4, 4, 128, 16, [1, 15, 16, 17, 0]),
    (1, 8, 1, 64, 32, [100, 33, 64]),
    (1, 18, 2, 128, 64, [65, 200]),        # 9 heads share one
    (1, 16, 1, 96, 16, [129]),
    (1, 40, 1, 80, 48, [47, 49]),          # more heads than one block takes
    (1, 6, 2, 256, 16, [70, 3]),
    (1, 20, 1, 256, 32, [90]),
    (1, 2, 1, 8, 16, [40]),
    (1, 3, 3, 136, 16, [50]),
    (4, 6, 2, 64, 16, [4, 90, 3, 1, 0]),   # new tokens that lie before the sequence's first one see nothing
    (3, 12, 1, 128, 32, [130, 31]),
    (1, 48, 1, 64, 16, [77, 0, 5]),        # 33 to 64 rows of a key head
    (5, 20, 2, 128, 16, [90, 4, 65]),
    (7, 11, 1, 256, 16, [33, 200]),        # more than 64
    (4, 34, 2, 40, 32, [3, 61]),
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("s,hq,hkv,d,page,lens", SHAPES)
def test_attention(dev, dtype, s, hq, hkv, d, page, lens):
    _attend_case(dev, dtype, s, hq, hkv, d, page, lens)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("s,hq,hkv,d,page,lens", [
    (1, 8, 8, 128, 64, [5000, 1, 0, 777, 63, 64, 65]),
    (1, 32, 8, 128, 16, [3001] + [10] * 40),
    (1, 1, 1, 64, 16, [40001]),
    (1, 16, 1, 128, 128, [20000, 129]),
    (2, 28, 4, 128, 32, [4100, 1, 2, 900]),
    (5, 71, 1, 64, 32, [1500, 33]),
    (1, 4, 2, 256, 16, [2500, 17]),
    (1, 12, 12, 64, 16, [10, 200] * 100),
    (6, 96, 6, 128, 32, [900, 33, 5000, 6, 0]),
    (4, 24, 1, 64, 32, [6001, 700, 4]),
    (150, 4, 2, 128, 64, [151, 1000]),
    (5, 40, 2, 128, 16, [300, 5, 0, 17, 1200] * 8),    # many groups of more than 32 rows
    (3, 96, 4, 64, 32, [65, 3, 700] * 6),
    (1, 70, 2, 256, 16, [40, 41] * 16),
])
def test_attention_long_and_ragged(dtype, s, hq, hkv, d, page, lens):
    _attend_case("cuda", dtype, s, hq, hkv, d, page, lens)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf])
def test_attention_does_not_look_behind_the_last_token(dev, dtype, fill):
    _attend_case(dev, dtype, 1, 6, 2, 64, 16, [1, 15, 40, 0], fill=fill)
    _attend_case(dev, dtype, 3, 6, 2, 128, 32, [3, 65, 40], fill=fill)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_new_tokens_do_not_see_later_ones(dev, dtype):
    """The later of two new tokens holds NaN and infinities; the earlier one's result does not change."""
    torch.manual_seed(3)
    kp, vp, table = _pool([40], 16, 2, 64, dtype, dev)
    q = torch.randn(1, 2, 12, 64).to(dtype).to(dev)
    lens = torch.tensor([40], dtype=torch.int32, device=dev)
    want = OF.paged_attention(q, kp, vp, table, lens)[:, 0]
    page, row = int(table[0, 39 // 16]), 39 % 16
    kp[page, :, row], vp[page, :, row] = math.nan, math.inf
    got = OF.paged_attention(q, kp, vp, table, lens)
    assert torch.equal(got[:, 0], want)
    assert got[:, 1].isnan().all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["left", "lowest", "empty", "all-lowest", "each", "bias", "16 bits"])
def test_attention_mask(dev, dtype, kind):
    torch.manual_seed(4)
    lens, s = [70, 33, 9], 2
    n = max(lens) + 3
    low = torch.finfo(torch.float32).min
    m = torch.zeros(3, 1, 1, n)
    if kind == "left":
        m[0, ..., :20], m[1, ..., :32], m[2, ..., :1] = -math.inf, -math.inf, -math.inf
    elif kind == "lowest":
        m[0, ..., :20], m[1, ..., 5:30] = low, low
    elif kind == "empty":
        m[1] = -math.inf
        m[0, ..., ::2] = -math.inf
    elif kind == "all-lowest":  # adding it leaves nothing of the scores: every token weighs the same
        m[1] = low
    elif kind == "each":
        m = torch.where(torch.rand(1, 1, s, n) < 0.5, -math.inf, 0.0)
    elif kind == "bias":
        m = torch.randn(3, 1, s, n)
    else:
        m = torch.where(torch.rand(3, 1, 1, n) < 0.5, torch.finfo(torch.bfloat16).min, 0.0).bfloat16()
    _attend_case(dev, dtype, s, 6, 2, 64, 16, lens, mask=m)


@pytest.mark.parametrize("dev", DEVICES)
def test_attention_masked_tokens_may_hold_anything(dev):
    torch.manual_seed(5)
    for dtype in TYPES:
        kp, vp, table = _pool([50], 16, 1, 64, dtype, dev)
        q = torch.randn(1, 1, 3, 64).to(dtype).to(dev)
        lens = torch.tensor([50], dtype=torch.int32, device=dev)
        m = torch.zeros(1, 1, 1, 50, device=dev)
        m[..., [0, 7, 20, 49]] = -math.inf
        want = OF.paged_attention(q, kp, vp, table, lens, mask=m)
        for t, x in ((0, math.nan), (7, math.inf), (20, -math.inf), (49, math.nan)):
            kp[int(table[0, t // 16]), :, t % 16] = x
            vp[int(table[0, t // 16]), :, t % 16] = x
        assert torch.equal(OF.paged_attention(q, kp, vp, table, lens, mask=m), want)


@pytest.mark.parametrize("dev", DEVICES)
def test_attention_scales_and_peaks(dev):
    for dtype in TYPES:
        _attend_case(dev, dtype, 1, 4, 2, 64, 16, [100, 7], scale=-0.3)
        _attend_case(dev, dtype, 1, 4, 2, 64, 16, [100, 7], scale=0.0)
        _attend_case(dev, dtype, 1, 4, 2, 64, 16, [100, 7], qscale=16.0)


@pytest.mark.parametrize("dev", DEVICES)
def test_pools_inside_a_larger_tensor(dev):
    """Keys and values of several layers in one allocation: pages and heads have strides of their own."""
    torch.manual_seed(6)
    pool = torch.randn(5, 2, 3, 2, 16, 64, device=dev).bfloat16()  # pages, k / v, layers, heads, tokens, dim
    kp, vp = pool[:, 0, 1], pool[:, 1, 1]
    table = torch.tensor([[4, 0, 2], [1, 3, 0]], dtype=torch.int32, device=dev)
    wide = torch.zeros(2, 7, dtype=torch.int32, device=dev)
    wide[:, 2:5] = table
    table = wide[:, 2:5]
    q, k, v = (torch.randn(2, 1, n, 64, device=dev).bfloat16() for n in (4, 2, 2))
    held = torch.tensor([40, 17], dtype=torch.int32, device=dev)
    before = pool.clone()
    OF.paged_kv_append(k, v, kp, vp, table, held)
    for r, t in ((0, 40), (1, 17)):
        page = int(table[r, t // 16])
        assert torch.equal(kp[page, :, t % 16], k[r, 0]) and torch.equal(vp[page, :, t % 16], v[r, 0])
        before[page, 0, 1, :, t % 16], before[page, 1, 1, :, t % 16] = k[r, 0], v[r, 0]
    assert torch.equal(pool, before)
    got = OF.paged_attention(q, kp, vp, table, held + 1)
    want, tol = _attend_exact(q, kp, vp, table, [41, 18], 1 / 8, None)
    assert ((got.double() - want).abs() <= tol).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pools_of_more_than_two_billion_elements(dtype):
    torch.manual_seed(8)
    pages, hkv, page, d = 140_000, 2, 64, 128  # 2.3e9 elements
    kp, vp = (torch.empty(pages, hkv, page, d, dtype=dtype, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 131_072, 0], [139_000, 5, pages - 2]], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(2, 150, hkv, d, device="cuda").to(dtype) for _ in range(2))
    OF.paged_kv_append(k, v, kp, vp, table, torch.zeros(2, dtype=torch.int32, device="cuda"))
    for r in range(2):
        assert torch.equal(_seq(kp, table, r, 150), k[r]) and torch.equal(_seq(vp, table, r, 150), v[r])
    q = torch.randn(2, 1, 8, d, device="cuda").to(dtype)
    got = OF.paged_attention(q, kp, vp, table, torch.tensor([150, 131], dtype=torch.int32, device="cuda"))
    _sync_status("cuda")
    want, tol = _attend_exact(q, kp, vp, table, [150, 131], d ** -0.5, None)
    assert ((got.double() - want).abs() <= tol).all()


def test_refusals_of_the_cache():
    kp, vp, table = _pool([20, 20], 16, 2, 64, torch.float32, "cpu")
    q, k, v = (torch.randn(2, 1, n, 64) for n in (4, 2, 2))
    lens = torch.tensor([3, 4], dtype=torch.int32)
    cos, sin = OF.rope_tables(64, 64)
    good = dict(k=k, v=v, k_pages=kp, v_pages=vp, block_table=table, start=lens, q=q, rope=(cos, sin, 64, True))
    OF.paged_kv_append(**good)
    for change in (dict(k=k[:, :, :1]), dict(k=k.half()), dict(k=k.half(), v=v.half()), dict(v=v.double(), k=k.double()), dict(k=k[0]),
                   dict(k_pages=kp[:, :, :8], v_pages=vp[:, :, :8]), dict(k_pages=kp[:-1]), dict(k_pages=kp.transpose(0, 1)),
                   dict(k_pages=kp.transpose(2, 3).contiguous().transpose(2, 3)), dict(block_table=table.long()),
                   dict(block_table=table[:1]), dict(block_table=table[0]), dict(start=lens.long()), dict(start=lens[:1]),
                   dict(count=lens.long()), dict(count=lens[:1]), dict(q=q[:1]), dict(q=q.half()), dict(q=q[..., :32]),
                   dict(rope=(cos.double(), sin.double(), 64, True)), dict(rope=(cos, sin, 66, True)), dict(rope=(cos, sin, 32, True)),
                   dict(rope=(cos, sin, 3, True))):
        with pytest.raises(ValueError):
            OF.paged_kv_append(**{**good, **change})
    with pytest.raises(RuntimeError, match="inference"):
        OF.paged_kv_append(**{**good, "k": k.clone().requires_grad_()})
    good = dict(q=q, k_pages=kp, v_pages=vp, block_table=table, lengths=lens)
    OF.paged_attention(**good)
    for change in (dict(q=q[0]), dict(q=q[:, :, :3]), dict(q=q.half()), dict(q=q[..., :32]), dict(lengths=lens.long()),
                   dict(lengths=lens[:1]), dict(scale=math.nan), dict(scale=math.inf), dict(mask=torch.zeros(2, 4, 1, 20)),
                   dict(mask=torch.zeros(2, 1, 2, 20)), dict(mask=torch.zeros(2, 20)), dict(mask=torch.zeros(2, 1, 1, 20).bool()),
                   dict(q=torch.randn(2, 1, 0, 64)), dict(block_table=table.float())):
        with pytest.raises(ValueError):
            OF.paged_attention(**{**good, **change})
    with pytest.raises(RuntimeError, match="inference"):
        OF.paged_attention(**{**good, "q": q.clone().requires_grad_()})
    big = torch.zeros(1, 1, 16, 264)
    with pytest.raises(ValueError, match="head_dim"):
        OF.paged_attention(torch.zeros(1, 1, 1, 264), big, big, table[:1], lens[:1])


def _bad_calls(dev):
    """(name, call, what must not change) of calls whose pages, positions or lengths leave their pool or table."""
    torch.manual_seed(7)
    kp, vp, table = _pool([32, 32], 16, 2, 64, torch.bfloat16, dev, spare=0)
    q, k, v = (torch.randn(2, 1, n, 64).bfloat16().to(dev) for n in (4, 2, 2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    rope = (*OF.rope_tables(8, 64, device=dev), 64, True)
    bad = table.clone()
    bad[0, 0], bad[1, 0] = -1, kp.shape[0]
    m = torch.zeros(2, 1, 1, 5, device=dev)
    return [
        ("page", lambda: OF.paged_kv_append(k, v, kp, vp, bad, i32(0, 0), q=q), (kp, vp)),
        ("behind the table", lambda: OF.paged_kv_append(k, v, kp, vp, table, i32(32, 2000000000), q=q), (kp, vp)),
        ("before the first", lambda: OF.paged_kv_append(k, v, kp, vp, table, i32(-1, -2147483648), q=q), (kp, vp)),
        ("rotation table", lambda: OF.paged_kv_append(k, v, kp, vp, table, i32(8, 9), q=q, rope=rope), (kp, vp)),
        ("read page", lambda: OF.paged_attention(q, kp, vp, bad, i32(9, 30)), ()),
        ("length", lambda: OF.paged_attention(q, kp, vp, table, i32(33, 2147483647)), ()),
        ("short mask", lambda: OF.paged_attention(q, kp, vp, table, i32(6, 7), mask=m), ()),
    ]


@pytest.mark.parametrize("which", range(7))
def test_pages_out_of_range_raise_on_the_cpu(which):
    name, call, same = _bad_calls("cpu")[which]
    before = [t.clone() for t in same]
    with pytest.raises(ValueError):
        call()
    assert all(torch.equal(a, b) for a, b in zip(before, same)), name


@gpu
@pytest.mark.parametrize("which", range(7))
def test_pages_out_of_range_are_skipped_and_reported(which):
    from oslo_b200.ops import _lib

    name, call, same = _bad_calls("cuda")[which]
    before = [t.clone() for t in same]
    out = call()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="paged cache"):
        _lib.check_status()
    assert all(torch.equal(a, b) for a, b in zip(before, same)), name
    assert torch.isfinite(out).all()
    _lib.check_status()  # reported once


# ------------------------------------------------------------------------------------------------ logits
def _logits_exact(x, tokens, lens, prompts, rep, pres, freq, bias, allowed):
    y = x.double().clone()
    rows, v = y.shape
    at = lambda p, r: float(p[r]) if isinstance(p, torch.Tensor) else p
    for r in range(rows):
        n = tokens.shape[1] if lens is None else int(lens[r])
        held = [t for t in tokens[r, :n].tolist()]
        made = held[0 if prompts is None else int(prompts[r]) :]
        for t in {t for t in held if 0 <= t < v}:
            y[r, t] = y[r, t] / at(rep, r) if y[r, t] > 0 else y[r, t] * at(rep, r)
            c = made.count(t)
            if c:
                y[r, t] -= at(pres, r) + at(freq, r) * c
    if bias is not None:
        y += bias.double()
    if allowed is not None:
        y[~allowed.expand(rows, v)] = -math.inf
    return y


def _logits_case(dev, dtype, rows, v, t, bias=None, allowed=None, per_row=True, lens=True, prompts=True, ids=torch.int64, spread=None,
                 strided=False, inplace=False):
    torch.manual_seed(rows + v + t)
    x = (3 * torch.randn(rows, 2, v)).to(dtype).to(dev)
    x = x[:, 1] if strided else x[:, 1].contiguous()
    x[:, 0] = 0.0
    tokens = torch.randint(-2, (spread or v) + 2, (rows, t), device=dev).to(ids)
    n = torch.randint(0, t + 1, (rows,), dtype=torch.int32, device=dev) if lens else None
    if lens:
        n[0] = t
    m = torch.randint(0, t + 1, (rows,), dtype=torch.int32, device=dev) if prompts else None
    rep, pres, freq = 1.3, 0.7, 0.2
    if per_row:
        rep, pres, freq = (a + 0.1 * torch.rand(rows, device=dev) for a in (rep, pres, freq))
    bias = {None: None, "shared": torch.randn(v, device=dev), "rows": torch.randn(rows, v, device=dev).to(dtype)}[bias]
    keep = {None: None, "shared": torch.rand(1, v, device=dev) < 0.3, "rows": torch.rand(rows, v, device=dev) < 0.5}[allowed]
    if keep is not None and rows > 1 and keep.shape[0] > 1:
        keep[1] = False
    want = _logits_exact(x, tokens, n, m, rep, pres, freq, bias, keep)
    # division or product, presence, frequency (product and difference), bias: 5 roundings of values up to the largest one
    big = (x.double().abs() * 1.5 + 1.0 + 0.5 * t + (bias.double().abs() if bias is not None else 0.0))
    tol = 5 * U * big + _half_step(dtype) * want.abs().nan_to_num(posinf=0.0) + 2.0 ** -25
    got = OF.process_logits(x, tokens, n, m, rep, pres, freq, bias, OF.pack_token_mask(keep) if keep is not None else None,
                            out=x if inplace else None)
    assert got.dtype == dtype and got.shape == (rows, v) and (got.data_ptr() == x.data_ptr()) == inplace
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)) and (got[~fine] == -math.inf).all()
    assert ((got.double() - want).abs()[fine] <= tol[fine]).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v,t,kw", [
    (1, 50, 9, dict()),
    (3, 33, 1, dict(bias="shared", allowed="rows")),
    (2, 1000, 400, dict(spread=7, bias="rows", allowed="shared", per_row=False)),
    (2, 257, 30, dict(strided=True, lens=False, prompts=False, ids=torch.int32)),
    (3, 999, 50, dict(inplace=True, allowed="rows", prompts=False)),
    (2, 31, 0, dict(bias="shared", allowed="shared", lens=False, prompts=False)),
    (1, 1, 5, dict(allowed="shared")),
])
def test_logits(dev, dtype, rows, v, t, kw):
    _logits_case(dev, dtype, rows, v, t, **kw)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v,t,kw", [
    (1, 50257, 2000, dict(bias="shared", allowed="rows")),
    (17, 32001, 4097, dict(spread=300, bias="rows", strided=True)),
    (5, 250112, 700, dict(allowed="shared", inplace=True, ids=torch.int32)),
    (200, 8193, 33, dict(allowed="rows", bias="shared")),
    (2, 300001, 100, dict(bias="shared", prompts=False)),
    (3, 8191, 32767, dict(spread=40, bias="shared")),             # the longest history of 16-bit counters
    (7, 8191, 32768, dict(spread=40, allowed="rows", strided=True)),  # 32-bit counters, rows off the 16-byte grid
    (3, 70001, 40000, dict(spread=2, prompts=False, lens=False)),
])
def test_logits_large(dtype, rows, v, t, kw):
    _logits_case("cuda", dtype, rows, v, t, **kw)


@gpu
def test_logits_of_more_than_two_billion_elements():
    rows, v = 8700, 250_112
    x = torch.empty(rows, v, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 1, 4000, 8586, 8587, 8699], device="cuda")
    x[some] = torch.randn(6, v, device="cuda").bfloat16()
    tokens = torch.randint(0, v, (rows, 20), device="cuda")
    got = OF.process_logits(x, tokens, repetition_penalty=1.2, frequency_penalty=0.1)
    assert torch.equal(got[some], OF.process_logits(x[some], tokens[some], repetition_penalty=1.2, frequency_penalty=0.1))


@pytest.mark.parametrize("dev", DEVICES)
def test_logits_keeps_infinities_and_nan(dev):
    x = torch.tensor([[math.inf, -math.inf, math.nan, 1.0, -1.0]], device=dev)
    tok = torch.arange(5, device=dev)[None]
    got = OF.process_logits(x, tok, repetition_penalty=2.0, frequency_penalty=0.5)
    want = torch.tensor([[math.inf, -math.inf, math.nan, 0.0, -2.5]], device=dev)
    assert torch.equal(got.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))
    only = OF.pack_token_mask(torch.tensor([[True, True, False, True, True]], device=dev))
    assert OF.process_logits(x, allowed=only)[0, 2] == -math.inf
    assert torch.equal(OF.process_logits(x[:, 3:]), x[:, 3:])


def test_packed_mask_bits():
    m = torch.rand(3, 77) < 0.5
    w = OF.pack_token_mask(m)
    assert w.dtype == torch.int32 and w.shape == (3, 3)
    for r, j in itertools.product(range(3), range(96)):
        assert bool((int(w[r, j // 32]) >> (j % 32)) & 1) == (j < 77 and bool(m[r, j]))


def test_refusals_of_the_logits():
    x, tok = torch.randn(2, 50), torch.zeros(2, 4, dtype=torch.int64)
    i32 = torch.tensor([1, 2], dtype=torch.int32)
    good = dict(logits=x, tokens=tok, repetition_penalty=1.1)
    OF.process_logits(**good)
    for change in (dict(logits=x[0]), dict(logits=x.double()), dict(tokens=tok[:1]), dict(tokens=tok.float()), dict(tokens=None),
                   dict(token_lengths=i32.long()), dict(token_lengths=i32[:1]), dict(prompt_lengths=i32.float()),
                   dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=math.nan),
                   dict(repetition_penalty=torch.ones(3)), dict(frequency_penalty=torch.ones(2, 1)), dict(bias=torch.zeros(49)),
                   dict(bias=torch.zeros(1, 50)), dict(bias=torch.zeros(50, dtype=torch.int64)), dict(allowed=torch.ones(2, 50).bool()),
                   dict(allowed=torch.zeros(2, 3, dtype=torch.int32)), dict(allowed=torch.zeros(3, 2, dtype=torch.int32)),
                   dict(out=torch.zeros(2, 51)), dict(out=torch.zeros(2, 50).half()), dict(tokens=None, token_lengths=i32)):
        with pytest.raises(ValueError):
            OF.process_logits(**{**good, **change})
    with pytest.raises(RuntimeError, match="inference"):
        OF.process_logits(x.clone().requires_grad_(), tok)
    with pytest.raises(ValueError):
        OF.pack_token_mask(torch.ones(2, 3))
