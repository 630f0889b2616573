"""Edges of the paged cache's and the logits' operators: values, layouts and arguments at which they could go wrong.

Tolerances count roundings, as in test_paged_ops.py: u = 2**-24 is the unit rounding of 32 bits, a result rounded to type t is off by
``eps(t) / 2`` of its value.
"""
import math

import pytest
import torch

from oslo_b200.nn import functional as OF
from test_paged_ops import DEVICES, TYPES, U, _attend_exact, _half_step, _pool, _seq, _sync_status

gpu = pytest.mark.gpu
I32 = dict(dtype=torch.int32)

# s, query heads, key heads, head dim, page, lengths, width of the table in tokens: calls that the kernels' forms take
FORMS = [
    (1, 6, 2, 64, 16, [70, 33], 0),                     # 8 rows, one launch
    (1, 4, 2, 128, 32, [500, 70], 9000),                # 8 rows, two launches
    (1, 12, 1, 256, 16, [70, 41], 0),                   # 16 rows, one launch
    (1, 24, 2, 128, 16, [300, 77], 9000),               # 16 rows, two launches
    (3, 6, 2, 64, 16, [70, 33], 0),                     # several new tokens
    (5, 40, 2, 128, 16, [90, 65] + [40] * 38, 0),       # 64 rows, one launch
    (5, 40, 2, 64, 16, [90, 65] + [200] * 38, 9000),    # 64 rows, two launches
    (3, 70, 1, 256, 16, [60, 41] + [30] * 30, 9000),
]


def _wide(table, tokens, page):
    """The same table with room for sequences of ``tokens`` tokens."""
    wide = torch.zeros(table.shape[0], max(table.shape[1], tokens // page), **I32)
    wide[:, : table.shape[1]] = table.cpu()
    return wide.to(table.device)


def _form(dev, dtype, form, seed=0):
    torch.manual_seed(seed)
    s, hq, hkv, d, page, lens, width = form
    kp, vp, table = _pool(lens, page, hkv, d, dtype, dev)
    q = torch.randn(len(lens), s, hq, d).to(dtype).to(dev)
    return q, kp, vp, _wide(table, width, page), torch.tensor(lens, **I32).to(dev)


# ------------------------------------------------------------------------------------------------ attention: values
LATER = [  # the query tokens of a sequence fill several blocks, or several warps of one
    (4, 24, 1, 64, 32, [61, 40], 0), (4, 24, 1, 64, 32, [601, 40], 9000),      # 16 rows a block, of one or two tokens
    (3, 16, 1, 256, 16, [33, 20], 0),                                         # 8 or 16 rows a block
    (2, 40, 1, 128, 16, [33, 50], 0), (9, 8, 2, 80, 16, [70, 9], 0),
    (5, 40, 2, 64, 16, [40, 5, 0, 17, 3, 90, 64, 65] * 5, 0),                 # 64 rows a block, 16 a warp
    (5, 40, 2, 128, 16, [40, 5, 0, 17, 3, 90, 64, 65] * 5, 9000),
    (7, 12, 1, 96, 16, [70, 8, 0, 33] * 20, 0),
]


@pytest.mark.parametrize("dev,form", [("cpu", LATER[4])] + [pytest.param("cuda", f, marks=gpu) for f in LATER])
@pytest.mark.parametrize("dtype", TYPES)
def test_later_tokens_do_not_show_in_any_block(dev, dtype, form):
    """The newest token's key is NaN and its value infinite; the results of the tokens before it do not change."""
    q, kp, vp, table, lens = _form(dev, dtype, form)
    s, _, _, _, page, n, _ = form
    want = OF.paged_attention(q, kp, vp, table, lens)
    rows = [r for r in range(len(n)) if n[r]]
    for r in rows:
        t = n[r] - 1
        kp[int(table[r, t // page]), :, t % page], vp[int(table[r, t // page]), :, t % page] = math.nan, math.inf
    got = OF.paged_attention(q, kp, vp, table, lens)
    assert torch.equal(got[:, : s - 1], want[:, : s - 1])
    assert got[rows, s - 1].isnan().all()


@pytest.mark.parametrize("dev,form", [("cpu", FORMS[0]), ("cpu", FORMS[4])] + [pytest.param("cuda", f, marks=gpu) for f in FORMS])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("masked", [False, True])
def test_a_seen_infinite_value_stays_infinite(dev, dtype, masked, form):
    """Keys are finite, so every weight is positive: a column with one infinity among the seen values is that infinity, one with both
    signs or a NaN is NaN, and every other column is what it is without them."""
    q, kp, vp, table, lens = _form(dev, dtype, form)
    s, _, hkv, d, page, n, _ = form
    b = len(n)
    mask = torch.randn(b, 1, 1, max(n)).to(dev) if masked else None
    column = torch.zeros(b, s, hkv, d, device=dev)  # what the infinities leave of a column
    clean = vp.clone()
    for r in range(b):
        for t, j, x in ((0, 0, math.inf), (n[r] // 2, 1, -math.inf), (n[r] - 1, 2, math.inf), (2, 3, math.inf), (n[r] - s, 3, -math.inf),
                        (5, 4, math.nan), (n[r] - 1, 5, -math.inf)):
            at = int(table[r, t // page]), slice(None), t % page, j
            vp[at], clean[at] = x, 0.0
            for i in range(s):
                if t < n[r] - s + 1 + i:
                    column[r, i, :, j] += x
    want = OF.paged_attention(q, kp, clean, table, lens, mask=mask).view(b, s, hkv, -1, d)
    got = OF.paged_attention(q, kp, vp, table, lens, mask=mask).view(b, s, hkv, -1, d)
    _sync_status(dev)
    column = column.unsqueeze(3).expand_as(got)
    wild = column != 0
    assert torch.equal(got[wild].float().nan_to_num(nan=7.0, posinf=8.0, neginf=9.0), column[wild].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))
    # the same sums in 32 bits, rounded once on either side
    tol = 2 * (max(n) + 16) * U * vp[vp.isfinite()].abs().max() + 2 * _half_step(dtype) * want.abs().float()
    assert ((got.float() - want.float()).abs() <= tol)[~wild].all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_one_token_of_infinities(dev, dtype):
    q, kp, vp, table, lens = _form(dev, dtype, (1, 4, 2, 64, 16, [1, 1], 0))
    vp[int(table[0, 0]), :, 0] = math.inf
    vp[int(table[1, 0]), :, 0, ::2] = -math.inf
    got = OF.paged_attention(q, kp, vp, table, lens).view(2, 4, 64)
    assert (got[0] == math.inf).all() and (got[1, :, ::2] == -math.inf).all()
    assert torch.equal(got[1, :2, 1::2], vp[int(table[1, 0]), 0, 0, 1::2].expand(2, -1))


def _tail_bound(q, k, x, p, v, o, scale, dtype):
    """As in test_paged_ops.py: sums of d products (2 d u of their magnitudes) and 4 u of a score change a weight by exp(2 e); the
    exponential 2**-21; two 16-bit parts of a weight 2**-16 (32-bit inputs: none); n weights summed in 32 bits.  Parts of 16-bit
    floats have steps of 2**-24 of a weight that was scaled by 2**15: a token's weight is off by at most 2**-40, whatever it is."""
    d, n = q.shape[-1], x.shape[-1]
    e = (2 * d * U * (q.abs() @ k.abs().T * abs(scale)) + 4 * U * x.abs()).amax(-1, keepdim=True)
    part = 0.0 if dtype == torch.float32 else 2.0 ** -16
    pre = (torch.expm1(2 * e) + 2.0 ** -21 + part + 2 * (n + 16) * U) * (p @ v.abs())
    small = 2.0 ** -39 * v.abs().sum(0) if dtype == torch.float16 else 0.0
    return _half_step(dtype) * (o.abs() + pre) + pre + small + 2.0 ** -25


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,n,batch", [(1, 4001, 1), (4, 131071, 1), (12, 4001, 1), (12, 60000, 1), (40, 4001, 64), (5, 300, 1)])
@pytest.mark.parametrize("gap", [12.0, 17.0, 20.0])
@pytest.mark.parametrize("masked", [False, True])
def test_many_light_tokens_behind_a_heavy_one(dtype, hq, n, batch, gap, masked):
    """One token's score is `gap` above the others', and its value is zero: the result is what the light tokens give, each of them
    exp(-gap) of the heavy one."""
    torch.manual_seed(hq + n)
    d, page = 64, 64
    kp, vp, table = _pool([n], page, 1, d, dtype, "cuda")
    q = torch.randn(1, 1, 1, d).sign().expand(batch, 1, hq, d).to(dtype).cuda()
    kp.mul_(0.0)
    vp.abs_().mul_(1000.0 if n < 10000 else 100.0)
    heavy = int(table[0, 0]), 0, 3
    kp[heavy], vp[heavy] = (q[0, 0, 0].float() * gap / 8).to(dtype), 0.0  # q k = 64 gap / 8, scaled by 1 / 8
    mask = torch.zeros(1, 1, 1, n, device="cuda") if masked else None
    got = OF.paged_attention(q, kp, vp, table.expand(batch, -1).contiguous(), torch.full((batch,), n, device="cuda", **I32), mask=mask)
    _sync_status("cuda")
    k, v = _seq(kp, table, 0, n)[:, 0].double(), _seq(vp, table, 0, n)[:, 0].double()
    x = q[0, 0].double() @ k.T / 8
    p = torch.softmax(x, -1)
    want = p @ v
    off = (got.view(batch, hq, d).double() - want).abs()
    tol = _tail_bound(q[0, 0].double(), k, x, p, v, want, 1 / 8, dtype)
    assert (off <= tol).all(), (off / tol).max().item()


# ------------------------------------------------------------------------------------------------ attention: blocks of 64 rows
SPLIT = [  # more than 32 rows of a key head, and many key heads
    (5, 40, 2, 64, 16, [40, 5, 0, 17, 3, 90, 64, 65] * 5, 0),
    (5, 40, 2, 128, 16, [40, 5, 0, 17, 3, 90, 64, 65] * 5, 9000),
    (1, 70, 2, 256, 32, [40, 0, 1, 17, 63, 90, 64, 65] * 4, 9000),
    (7, 12, 1, 96, 16, [70, 8, 0, 33] * 20, 0),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["none", "left", "lowest", "empty", "all-lowest", "bias"])
@pytest.mark.parametrize("form", SPLIT)
def test_blocks_of_64_rows_under_a_mask(dtype, kind, form):
    q, kp, vp, table, lens = _form("cuda", dtype, form)
    s, _, _, d, page, n, _ = form
    b, low = len(n), torch.finfo(torch.float32).min
    m = torch.zeros(b, 1, 1, max(n) + 3)
    if kind == "left":
        for r in range(b):
            m[r, ..., : n[r] * (r % 4) // 4] = -math.inf
    elif kind == "lowest":
        m[::2, ..., 5:30] = low
    elif kind == "empty":
        m[1::3] = -math.inf
        m[::3, ..., ::2] = -math.inf
    elif kind == "all-lowest":
        m[::2] = low
    elif kind == "bias":
        m = torch.randn(1, 1, 1, max(n) + 3)
    m = None if kind == "none" else m.cuda()
    got = OF.paged_attention(q, kp, vp, table, lens, mask=m)
    _sync_status("cuda")
    want, tol = _attend_exact(q, kp, vp, table, n, d ** -0.5, m)
    assert ((got.double() - want).abs() <= tol).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fill", [math.nan, math.inf])
@pytest.mark.parametrize("form", SPLIT)
def test_blocks_of_64_rows_do_not_look_behind_the_last_token(dtype, fill, form):
    q, kp, vp, table, lens = _form("cuda", dtype, form)
    s, _, _, d, page, n, _ = form
    used = torch.zeros(kp.shape[0], page, dtype=torch.bool, device="cuda")
    for r in range(len(n)):
        t = torch.arange(n[r], device="cuda")
        used[table[r].long()[t // page], t % page] = True
    for pool in (kp, vp):
        pool.masked_fill_(~used[:, None, :, None], fill)
    got = OF.paged_attention(q, kp, vp, table, lens)
    want, tol = _attend_exact(q, kp, vp, table, n, d ** -0.5, None)
    assert ((got.double() - want).abs() <= tol).all()
    # masked tokens may hold anything either
    m = torch.zeros(len(n), 1, 1, max(n), device="cuda")
    hidden = [0, 2, 30, max(n) - 1]
    m[..., hidden] = -math.inf
    want = OF.paged_attention(q, kp, vp, table, lens, mask=m)
    for r in range(len(n)):
        for t in hidden:
            if t < n[r]:
                kp[int(table[r, t // page]), :, t % page] = fill
                vp[int(table[r, t // page]), :, t % page] = fill
    assert torch.equal(OF.paged_attention(q, kp, vp, table, lens, mask=m), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", SPLIT)
def test_blocks_of_64_rows_skip_and_report_bad_pages_and_lengths(dtype, form):
    from oslo_b200.ops import _lib

    q, kp, vp, table, lens = _form("cuda", dtype, form)
    want = OF.paged_attention(q, kp, vp, table, lens)
    _sync_status("cuda")
    bad = table.clone()
    bad[0, 1], bad[5, 0] = -1, kp.shape[0]
    got = OF.paged_attention(q, kp, vp, bad, lens)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="paged cache"):
        _lib.check_status()
    same = [r for r in range(len(form[5])) if r not in (0, 5)]
    assert torch.equal(got[same], want[same]) and torch.isfinite(got).all()
    far = lens.clone()
    far[0], far[7] = 2147483647, table.shape[1] * form[4] + 1
    got = OF.paged_attention(q, kp, vp, table, far)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="paged cache"):
        _lib.check_status()
    same = [r for r in range(len(form[5])) if r not in (0, 7)]  # the blocks' shares follow the lengths: other sums of the same tokens
    want, tol = _attend_exact(q[same], kp, vp, table[same], [form[5][r] for r in same], form[3] ** -0.5, None)
    assert ((got[same].double() - want).abs() <= tol).all() and torch.isfinite(got).all()
    _lib.check_status()


@gpu
@pytest.mark.parametrize("s,hq,hkv,d,page,lens", [
    (1, 4, 4, 128, 16, [1, 15, 16, 17, 0]), (1, 18, 2, 128, 64, [65, 200]), (1, 20, 1, 256, 32, [90]), (4, 6, 2, 64, 16, [4, 90, 3, 1, 0]),
    (1, 3, 3, 136, 16, [50]), (1, 8, 8, 128, 64, [5000, 1, 0, 777, 63, 64, 65]), (1, 1, 1, 64, 16, [20001]), (6, 96, 6, 128, 32, [900, 33, 5, 6, 0]),
])
@pytest.mark.parametrize("masked", [False, True])
def test_attention_in_32_bits_loses_no_bits(s, hq, hkv, d, page, lens, masked):
    """32-bit inputs are multiplied and summed in 32 bits: d products, 2 d u of their magnitudes; scaling and mask 4 u of a score;
    the exponential 2**-21; n weights and values, 2 (n + 16) u."""
    torch.manual_seed(d + sum(lens))
    kp, vp, table = _pool(lens, page, hkv, d, torch.float32, "cuda")
    q = torch.randn(len(lens), s, hq, d, device="cuda")
    m = torch.randn(len(lens), 1, 1, max(lens), device="cuda") if masked else None
    got = OF.paged_attention(q, kp, vp, table, torch.tensor(lens, device="cuda", **I32), mask=m).view(len(lens), s, hkv, -1, d)
    for r, n in enumerate(lens):
        k, v = _seq(kp, table, r, n).double(), _seq(vp, table, r, n).double()
        for i in range(s):
            end = n - s + 1 + i
            if end <= 0:
                assert (got[r, i] == 0).all()
                continue
            for h in range(hkv):
                qq, kk, vv = q[r, i].view(hkv, -1, d)[h].double(), k[:end, h], v[:end, h]
                x = qq @ kk.T / math.sqrt(d)
                e = 2 * d * U * (qq.abs() @ kk.abs().T / math.sqrt(d)) + 4 * U * x.abs()
                if masked:
                    x = x + m[r, 0, 0, :end].double()
                    e = e + 4 * U * m[r, 0, 0, :end].abs()
                p = torch.softmax(x, -1)
                want = p @ vv
                pre = (torch.expm1(2 * e.amax(-1, keepdim=True)) + 2.0 ** -21 + 2 * (end + 16) * U) * (p @ vv.abs())
                assert ((got[r, i, h].double() - want).abs() <= pre + U * (want.abs() + pre)).all(), (r, i, h)


# ------------------------------------------------------------------------------------------------ arguments without elements
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_a_mask_without_tokens_is_a_short_mask(dev, dtype):
    q, kp, vp, table, lens = _form(dev, dtype, (1, 6, 2, 64, 16, [20, 3], 0))
    for rows in (1, 2):
        m = torch.zeros(rows, 1, 1, 0, device=dev)
        if dev == "cpu":
            with pytest.raises(ValueError, match="mask"):
                OF.paged_attention(q, kp, vp, table, lens, mask=m)
        else:
            from oslo_b200.ops import _lib

            got = OF.paged_attention(q, kp, vp, table, lens, mask=m)
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="paged cache"):
                _lib.check_status()
            assert (got == 0).all()
        assert (OF.paged_attention(q, kp, vp, table, torch.zeros_like(lens), mask=m) == 0).all()  # nothing to cover
        _sync_status(dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("neox", [False, True])
def test_rotation_tables_without_positions_are_short_tables(dev, neox):
    q, kp, vp, table, lens = _form(dev, torch.bfloat16, (1, 6, 2, 64, 16, [20, 3], 0))
    k, v = (torch.randn(2, 1, 2, 64).bfloat16().to(dev) for _ in range(2))
    none = torch.zeros(0, 32, device=dev)
    before = kp.clone(), vp.clone()
    call = lambda: OF.paged_kv_append(k, v, kp, vp, table, torch.zeros_like(lens), q=q, rope=(none, none, 64, neox))
    if dev == "cpu":
        with pytest.raises(ValueError, match="rotation"):
            call()
    else:
        from oslo_b200.ops import _lib

        out = call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="paged cache"):
            _lib.check_status()
        assert (out == 0).all()
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])


@pytest.mark.parametrize("dev", DEVICES)
def test_a_scale_that_32_bits_do_not_hold_is_refused(dev):
    q, kp, vp, table, lens = _form(dev, torch.float32, (1, 6, 2, 64, 16, [20, 3], 0))
    OF.paged_attention(q, kp, vp, table, lens)
    for scale in (1e39, -1e300, 3e38, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            OF.paged_attention(q, kp, vp, table, lens, scale=scale)


@pytest.mark.parametrize("dev", DEVICES)
def test_the_lowest_value_of_64_bits_is_not_minus_infinity(dev):
    """A mask of 64 bits at its type's lowest value: every token is there and weighs the same.  At -inf none is."""
    q, kp, vp, table, lens = _form(dev, torch.float32, (1, 6, 2, 64, 16, [20, 3], 0))
    for low in (torch.finfo(torch.float64).min, -1e39):
        m = torch.full((2, 1, 1, 20), low, dtype=torch.float64, device=dev)
        m[1, ..., 1] = -math.inf
        got = OF.paged_attention(q, kp, vp, table, lens, mask=m).view(2, 2, 3, 64)
        a, b = _seq(vp, table, 0, 20), _seq(vp, table, 1, 3)[[0, 2]]
        for r, v in ((0, a), (1, b)):  # a mean of n values: n sums and a division, n + 2 roundings
            tol = (v.shape[0] + 2) * U * v.abs().mean(0)[:, None] + 2.0 ** -21 * v.abs().mean(0)[:, None]
            assert ((got[r] - v.mean(0)[:, None]).abs() <= tol).all()
        m[:] = -math.inf
        assert (OF.paged_attention(q, kp, vp, table, lens, mask=m) == 0).all()


# ------------------------------------------------------------------------------------------------ no gradient is lost silently
@pytest.mark.parametrize("dev", DEVICES)
def test_inputs_that_carry_a_gradient_are_refused(dev):
    from torch.autograd import forward_ad as fwd

    q, kp, vp, table, lens = _form(dev, torch.float32, (1, 6, 2, 64, 16, [20, 3], 0))
    k, v = (torch.randn(2, 1, 2, 64, device=dev) for _ in range(2))
    cos, sin = OF.rope_tables(64, 64, device=dev)
    m = torch.zeros(2, 1, 1, 20, device=dev)
    x, tokens = torch.randn(2, 50, device=dev), torch.zeros(2, 4, dtype=torch.int64, device=dev)
    one = torch.ones(2, device=dev)
    append = dict(k=k, v=v, k_pages=kp, v_pages=vp, block_table=table, start=lens - 1, q=q)
    attend = dict(q=q, k_pages=kp, v_pages=vp, block_table=table, lengths=lens, mask=m)
    logits = dict(logits=x, tokens=tokens, repetition_penalty=one, presence_penalty=one, frequency_penalty=one, bias=torch.zeros(50, device=dev))
    OF.paged_kv_append(**append, rope=(cos, sin, 64, True))
    OF.paged_attention(**attend)
    OF.process_logits(**logits)
    calls = [(OF.paged_kv_append, append, n) for n in ("k", "v", "q", "k_pages", "v_pages")]
    calls += [(OF.paged_attention, attend, n) for n in ("q", "k_pages", "v_pages", "mask")]
    calls += [(OF.process_logits, logits, n) for n in ("logits", "bias", "repetition_penalty", "presence_penalty", "frequency_penalty")]
    for f, good, name in calls:
        with pytest.raises(RuntimeError, match="inference"):
            f(**{**good, name: good[name].clone().requires_grad_()})
        with torch.no_grad():  # nothing is recorded
            f(**{**good, name: good[name].clone().requires_grad_()})
        with fwd.dual_level():
            dual = fwd.make_dual(good[name].clone(), torch.ones_like(good[name]))
            for grad in (True, False):  # forward derivatives do not hang on the recording of backward ones
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="inference"):
                    f(**{**good, name: dual})
    for i in range(2):
        tables = [cos, sin]
        tables[i] = tables[i].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="inference"):
            OF.paged_kv_append(**append, rope=(*tables, 64, True))
        with fwd.dual_level():
            tables[i] = fwd.make_dual(tables[i].detach(), torch.ones_like(cos))
            with pytest.raises(RuntimeError, match="inference"):
                OF.paged_kv_append(**append, rope=(*tables, 64, True))
    out = torch.empty_like(x).requires_grad_()
    with pytest.raises(RuntimeError, match="inference"):
        OF.process_logits(x, out=out)
    _sync_status(dev)


# ------------------------------------------------------------------------------------------------ logits
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,t", [(1000, 3000), (1000, 40000), (70001, 9000)])
def test_the_repetition_penalty_divides(dev, dtype, v, t):
    """A quotient (a reciprocal and a product: two roundings to 32 bits) or a product (one), then one rounding to the logits' type."""
    torch.manual_seed(v)
    rep = torch.tensor([1.3, 1.1, 0.7, 3.0, 2.0 ** 126], device=dev)
    x = (3 * torch.randn(5, v, device=dev)).to(dtype)
    x[4] = (x[4].float() * (1e37 if dtype != torch.float16 else 1.0)).to(dtype)
    tokens = torch.randint(0, v, (5, t), device=dev)
    got = OF.process_logits(x, tokens, repetition_penalty=rep)
    seen = torch.zeros(5, v, dtype=torch.bool, device=dev).scatter_(1, tokens, True)
    x64, r64 = x.double(), rep.double()[:, None]
    want = torch.where(x64 > 0, x64 / r64, x64 * r64)
    normal = (want.abs() >= torch.finfo(dtype).tiny) & (want.abs() < torch.finfo(dtype).max)
    pre = 2 * U * (1 + U) * want.abs()
    tol = pre + _half_step(dtype) * (want.abs() + pre)
    assert ((got.double() - want).abs() <= tol)[seen & normal].all()
    assert torch.equal(got[~seen], x[~seen])


@pytest.mark.parametrize("dev", DEVICES)
def test_repetition_penalties_without_a_reciprocal_are_refused(dev):
    x, tokens = torch.full((1, 8), 1e38, device=dev), torch.arange(8, device=dev)[None]
    for rep in (2e38, 1e39, math.inf, 1e-38, 1e-45, 0.0):
        with pytest.raises(ValueError, match="repetition_penalty"):
            OF.process_logits(x, tokens, repetition_penalty=rep)
    got = OF.process_logits(x, tokens, repetition_penalty=2.0 ** 126)  # a power of two: exact
    assert torch.equal(got, (x.double() / 2.0 ** 126).float())


@pytest.mark.parametrize("dev", DEVICES)
def test_logits_refuse_an_output_that_overlaps_them_or_itself(dev):
    torch.manual_seed(2)
    buf = torch.randn(4, 200, device=dev)
    x = buf[:, :100]
    for out in (buf[:, 1:101], buf[:, 99:199], buf.view(-1)[300:700].view(4, 100),
                torch.empty(1, 100, device=dev).expand(4, 100), torch.empty(4 * 50 + 50, device=dev).as_strided((4, 100), (50, 1))):
        with pytest.raises(ValueError, match="out"):
            OF.process_logits(x, out=out)
    want = x.clone() + 1.0
    bias = torch.ones(100, device=dev)
    assert torch.equal(OF.process_logits(x, bias=bias, out=buf[:, 100:]), want)  # side by side in one buffer
    got = OF.process_logits(x, bias=bias, out=x)
    assert got.data_ptr() == x.data_ptr() and torch.equal(x, want)
    one = torch.randn(1, 100, device=dev)
    want = one + 1.0
    assert torch.equal(OF.process_logits(one, bias=bias, out=one), want)
    rows = torch.randn(6, 40, device=dev)  # every second row, and the rows between
    want = rows[::2] + 1.0
    assert torch.equal(OF.process_logits(rows[::2], bias=bias[:40], out=rows[1::2]), want)
    square = torch.randn(30, 30, device=dev)
    want = square.t() + 1.0
    assert torch.equal(OF.process_logits(square.t(), bias=bias[:30], out=square), want)  # columns are copied first
    same = torch.randn(1, 40, device=dev).expand(3, 40)
    assert torch.equal(OF.process_logits(same, bias=bias[:40], out=torch.empty(3, 40, device=dev)), same + 1.0)
    with pytest.raises(ValueError, match="out"):
        OF.process_logits(rows[:3], out=rows[1:4])


@pytest.mark.parametrize("dev", DEVICES)
def test_logits_of_nothing(dev):
    tokens = torch.tensor([[3, 5], [0, -1]], device=dev)
    assert OF.process_logits(torch.empty(2, 0, device=dev), tokens, repetition_penalty=1.5).shape == (2, 0)
    assert OF.process_logits(torch.empty(0, 9, device=dev), tokens[:0], repetition_penalty=1.5).shape == (0, 9)


# ------------------------------------------------------------------------------------------------ refusals, wherever the tensors are
@pytest.mark.parametrize("dev", DEVICES)
def test_refusals_of_the_cache_on_every_device(dev):
    kp, vp, table = _pool([20, 20], 16, 2, 64, torch.float32, dev)
    q, k, v = (torch.randn(2, 1, n, 64, device=dev) for n in (4, 2, 2))
    lens = torch.tensor([3, 4], device=dev, **I32)
    cos, sin = OF.rope_tables(64, 64, device=dev)
    good = dict(k=k, v=v, k_pages=kp, v_pages=vp, block_table=table, start=lens, q=q, rope=(cos, sin, 64, True))
    before = kp.clone(), vp.clone()
    elsewhere = [dict(v=v.cpu()), dict(q=q.cpu()), dict(start=lens.cpu()), dict(count=lens.cpu()), dict(block_table=table.cpu()),
                 dict(v_pages=vp.cpu()), dict(k_pages=kp.cpu()), dict(rope=(cos.cpu(), sin, 64, True)), dict(rope=(cos, sin.cpu(), 64, True))]
    for change in (dict(k=k[:, :, :1]), dict(k=k.half()), dict(k=k.half(), v=v.half()), dict(v=v.double(), k=k.double()), dict(k=k[0]),
                   dict(k_pages=kp[:, :, :8], v_pages=vp[:, :, :8]), dict(k_pages=kp[:-1]), dict(k_pages=kp.transpose(0, 1)),
                   dict(k_pages=kp.transpose(2, 3).contiguous().transpose(2, 3)), dict(block_table=table.long()),
                   dict(block_table=table[:1]), dict(block_table=table[0]), dict(start=lens.long()), dict(start=lens[:1]),
                   dict(count=lens.long()), dict(count=lens[:1]), dict(q=q[:1]), dict(q=q.half()), dict(q=q[..., :32]),
                   dict(rope=(cos.double(), sin.double(), 64, True)), dict(rope=(cos, sin, 66, True)), dict(rope=(cos, sin, 32, True)),
                   dict(rope=(cos, sin, 3, True)), dict(rope=(cos, sin[:5], 64, True)), dict(rope=(cos, sin, -2, True)),
                   dict(start=torch.stack([lens, lens], 1)[:, 0]),
                   dict(block_table=torch.stack([table, table], 2)[..., 0]),
                   *(elsewhere if dev == "cuda" else ())):
        with pytest.raises(ValueError):
            OF.paged_kv_append(**{**good, **change})
    _sync_status(dev)
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])
    OF.paged_kv_append(**good)
    good = dict(q=q, k_pages=kp, v_pages=vp, block_table=table, lengths=lens)
    OF.paged_attention(**good)
    m = torch.zeros(2, 1, 1, 20, device=dev)
    for change in (dict(q=q[0]), dict(q=q[:, :, :3]), dict(q=q.half()), dict(q=q[..., :32]), dict(lengths=lens.long()),
                   dict(lengths=lens[:1]), dict(scale=math.nan), dict(scale=math.inf), dict(mask=m.expand(2, 4, 1, 20)),
                   dict(mask=m.expand(2, 1, 2, 20)), dict(mask=m[0, 0]), dict(mask=m.bool()), dict(q=q[:, :, :0]), dict(block_table=table.float()),
                   dict(lengths=torch.stack([lens, lens], 1)[:, 0]),
                   *((dict(mask=m.cpu()), dict(lengths=lens.cpu()), dict(k_pages=kp.cpu()), dict(v_pages=vp.cpu())) if dev == "cuda" else ())):
        with pytest.raises(ValueError):
            OF.paged_attention(**{**good, **change})
    big = torch.zeros(1, 1, 16, 264, device=dev)
    with pytest.raises(ValueError, match="head_dim"):
        OF.paged_attention(torch.zeros(1, 1, 1, 264, device=dev), big, big, table[:1], lens[:1])
    _sync_status(dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals_of_the_logits_on_every_device(dev):
    x, tok = torch.randn(2, 50, device=dev), torch.zeros(2, 4, dtype=torch.int64, device=dev)
    i32 = torch.tensor([1, 2], device=dev, **I32)
    good = dict(logits=x, tokens=tok, repetition_penalty=1.1)
    OF.process_logits(**good)
    elsewhere = [dict(presence_penalty=torch.ones(2)), dict(bias=torch.zeros(50)), dict(allowed=torch.zeros(2, 2, **I32)),
                 dict(out=torch.zeros(2, 50)), dict(tokens=tok.cpu()), dict(token_lengths=i32.cpu()), dict(prompt_lengths=i32.cpu())]
    for change in (dict(logits=x[0]), dict(logits=x.double()), dict(tokens=tok[:1]), dict(tokens=tok.float()), dict(tokens=None),
                   dict(token_lengths=i32.long()), dict(token_lengths=i32[:1]), dict(prompt_lengths=i32.float()),
                   dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=math.nan),
                   dict(repetition_penalty=torch.ones(3, device=dev)), dict(frequency_penalty=torch.ones(2, 1, device=dev)),
                   dict(presence_penalty=torch.ones(2, device=dev, dtype=torch.int64)),
                   dict(bias=torch.zeros(49, device=dev)), dict(bias=torch.zeros(1, 50, device=dev)),
                   dict(bias=torch.zeros(50, dtype=torch.int64, device=dev)),
                   dict(allowed=torch.ones(2, 50, device=dev).bool()), dict(allowed=torch.zeros(2, 3, device=dev, **I32)),
                   dict(allowed=torch.zeros(3, 2, device=dev, **I32)),
                   dict(out=torch.zeros(2, 51, device=dev)), dict(out=torch.zeros(2, 50, device=dev).half()),
                   dict(out=torch.zeros(50, 2, device=dev).t()), dict(tokens=None, token_lengths=i32), *(elsewhere if dev == "cuda" else ())):
        with pytest.raises(ValueError):
            OF.process_logits(**{**good, **change})
