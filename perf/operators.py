"""Cases and plain forms of the operators of one token-generation step over a paged key / value cache.

``paged_kv_append``  rotates the new queries and keys by their positions and stores keys and values in the pages of their
                     sequences;
``paged_attention``  attends from the newest tokens over the pages;
``process_logits``   applies penalties for repeated tokens, biases and a grammar mask to the next-token logits.

``own`` selects between the plain forms below (elementary torch operations in 32 bits) and the framework's entry points.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one conversation on a 1.3B decoder (16 heads of 128, a quarter of each rotated): latency counts
        dict(name="append-one", op="append", dtype="bf16", b=1, s=1, hq=16, hkv=16, d=128, rot=32, neox=True, page=16, most=200),
        # a serving batch at different positions, grouped heads
        dict(name="append-batch", op="append", dtype="bf16", b=256, s=1, hq=32, hkv=8, d=128, rot=128, neox=True, page=64, most=512),
        # prompts of different lengths padded to the longest, full heads
        dict(name="append-prompts", op="append", dtype="bf16", b=8, s=1999, hq=32, hkv=32, d=128, rot=128, neox=True, page=64, most=0),
        # one conversation, short context: latency counts
        dict(name="attend-one-short", op="attend", dtype="bf16", b=1, s=1, hq=16, hkv=16, d=128, page=16, most=200, mask=False),
        # one conversation over a long document: the length is what can be split
        dict(name="attend-one-long", op="attend", dtype="bf16", b=1, s=1, hq=32, hkv=8, d=128, page=64, most=131071, mask=False),
        # a serving batch of requests of very different lengths, some slots idle, grouped heads
        dict(name="attend-ragged", op="attend", dtype="bf16", b=32, s=1, hq=32, hkv=8, d=128, page=64, most=4096, mask=False),
        # a large batch with as many key heads as query heads: the cache's bytes are all there is
        dict(name="attend-large", op="attend", dtype="bf16", b=64, s=1, hq=32, hkv=32, d=128, page=32, most=6000, mask=False),
        # four proposed tokens at once over one shared key head
        dict(name="attend-proposed", op="attend", dtype="fp16", b=16, s=4, hq=24, hkv=1, d=64, page=32, most=6001, mask=False),
        # 32-bit inference of a 12-head decoder with left-padded prompts
        dict(name="attend-masked-fp32", op="attend", dtype="fp32", b=8, s=1, hq=12, hkv=12, d=64, page=16, most=1000, mask=True),
        # one conversation's logits: latency counts
        dict(name="logits-one", op="logits", dtype="fp32", rows=1, v=50304, t=700, bias="none", allowed=False, per_row=False),
        # a batch under one shared bias
        dict(name="logits-batch", op="logits", dtype="fp32", rows=32, v=32000, t=2048, bias="shared", allowed=True, per_row=True),
        # a large multilingual vocabulary, every option per request
        dict(name="logits-large", op="logits", dtype="bf16", rows=192, v=250112, t=4095, bias="shared", allowed=True, per_row=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "logits", "logits"])
    if op == "logits":
        v = _log(rng, 1000, 250112)
        return dict(op=op, dtype=rng.choice(["fp32", "bf16", "fp16"]), rows=_log(rng, 1, max(1, min(256, 40_000_000 // v))), v=v,
                    t=_log(rng, 1, 8000), bias=rng.choice(["none", "shared", "rows"]), allowed=rng.random() < 0.6,
                    per_row=rng.random() < 0.6)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    d = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 5, 8, 12, 16, 32])
    group = rng.choice([1, 1, 2, 3, 4, 7, 8, 12, 16])
    page = rng.choice([16, 32, 64, 128])
    token = 2 * hkv * d * SIZES[dtype]  # bytes of one token's keys and values
    if op == "append":
        prompt = rng.random() < 0.4
        s = _log(rng, 2, 2000) if prompt else rng.choice([1, 1, 1, 2, 5])
        b = _log(rng, 1, max(1, min(512, 300_000_000 // (s * (token + hkv * group * d * SIZES[dtype])))))
        most = rng.choice([0, 0, 33, 150]) if prompt else min(_log(rng, 1, 600), 200_000_000 // (b * token))
        rot = rng.choice([r for r in (0, d // 4, d // 2, d, d) if r % 2 == 0])
        return dict(op=op, dtype=dtype, b=b, s=s, hq=hkv * group, hkv=hkv, d=d, rot=rot, neox=rng.random() < 0.7, page=page, most=most)
    most = _log(rng, 1, 100_000)
    s = rng.choice([1, 1, 1, 1, 2, 3, 6])
    # the plain form holds the scores of every head: its size is bounded beside the cache's
    b = _log(rng, 1, max(1, min(256, int(min(1_500_000_000 / (most * token), 500_000_000 / (most * hkv * group * s))))))
    return dict(op=op, dtype=dtype, b=b, s=s, hq=hkv * group, hkv=hkv, d=d, page=page, most=max(most, s), mask=rng.random() < 0.3)


# ------------------------------------------------------------------------------------------------ sizes of a case's rows
def _lengths(case):
    """Tokens in each sequence (attend: the new ones included; append: those held before).  The first has the most; the
    others spread over their logarithm, one slot of a larger batch is idle."""
    b, most, s = case["b"], case["most"], case["s"]
    rng = random.Random(b * 1000003 + most * 101 + s)
    out = [most] + [_log(rng, max(1, most // 40), most) if most > 1 else most for _ in range(b - 1)]
    if case["op"] == "attend":
        if b >= 64:  # a large batch under load: all of them long
            out = [most] + [rng.randint(most * 3 // 4, most) for _ in range(b - 1)]
        out = [max(n, s) for n in out]
        if b >= 8:
            out[b // 2] = 0
    return out


def _counts(case):
    """Real tokens among the ``s`` new ones of each sequence (append)."""
    b, s = case["b"], case["s"]
    rng = random.Random(b * 7919 + s * 31 + 5)
    out = [s] + [rng.randint(max(1, s // 2), s) for _ in range(b - 1)]
    if b >= 8 and s > 1:
        out[b // 2] = 0
    return out


def _history(case):
    """(tokens in the history, prompt tokens among them) of each row (logits)."""
    rng = random.Random(case["rows"] * 31337 + case["t"])
    lens = [case["t"]] + [rng.randint(0, case["t"]) for _ in range(case["rows"] - 1)]
    return lens, [rng.randint(0, n) for n in lens]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=gen)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["op"] == "logits":
        rows, v, t = case["rows"], case["v"], case["t"]
        logits = (3 * normal(rows, v)).to(DTYPES[case["dtype"]])
        # texts repeat themselves: token ids follow a power law
        u = torch.rand(rows, t, device="cuda", generator=gen, dtype=torch.float64)
        perm = torch.randperm(v, device="cuda", generator=gen)
        tokens = perm[(v ** u - 1).long().clamp(0, v - 1)]
        lens, prompts = _history(case)
        st = dict(case=dict(case), logits=logits, tokens=tokens, lens=ints(lens), prompts=ints(prompts), bias=None, allowed=None)
        if case["per_row"]:
            st["rep"] = 1.0 + 0.5 * torch.rand(rows, device="cuda", generator=gen)
            st["pres"] = torch.rand(rows, device="cuda", generator=gen)
            st["freq"] = 0.3 * torch.rand(rows, device="cuda", generator=gen)
        else:
            st["rep"], st["pres"], st["freq"] = 1.1 + 0.001 * (seed % 100), 0.5, 0.1
        if case["bias"] != "none":
            st["bias"] = normal(*((v,) if case["bias"] == "shared" else (rows, v)))
        if case["allowed"]:
            words = (v + 31) // 32
            bits = torch.randint(0, 1 << 32, (rows, words), device="cuda", generator=gen, dtype=torch.int64)
            bits &= torch.randint(0, 1 << 32, (rows, words), device="cuda", generator=gen, dtype=torch.int64)
            bits[::3] = (1 << 32) - 1  # requests without a grammar
            st["allowed"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        return st

    dtype, b, s, hq, hkv, d, page = DTYPES[case["dtype"]], case["b"], case["s"], case["hq"], case["hkv"], case["d"], case["page"]
    lens = _lengths(case)
    final = [n + s for n in lens] if case["op"] == "append" else lens
    need = [max(1, -(-n // page)) for n in final]
    pages = sum(need) + 3  # a few of the pool's pages belong to nobody
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at : at + n] + [0] * (max(need) - n))
        at += n
    spread = torch.exp(0.3 * normal(hkv, 1, d))  # some channels of the keys are larger than others
    k_pages = torch.empty(pages, hkv, page, d, dtype=dtype, device="cuda")
    v_pages = torch.empty(pages, hkv, page, d, dtype=dtype, device="cuda")
    step = max(1, 50_000_000 // (hkv * page * d))
    for i in range(0, pages, step):
        k_pages[i : i + step] = normal(*k_pages[i : i + step].shape) * spread
        v_pages[i : i + step] = normal(*v_pages[i : i + step].shape)
    st = dict(case=dict(case), k_pages=k_pages, v_pages=v_pages, table=ints(table), lens=ints(lens), longest=max(final))
    # the new tokens come out of one fused projection, as strided views
    qkv = normal(b, s, (hq + 2 * hkv), d).to(dtype)
    st["q"] = qkv[:, :, :hq]
    if case["op"] == "append":
        st["k"], st["v"] = qkv[:, :, hq : hq + hkv], qkv[:, :, hq + hkv :]
        st["count"] = ints(_counts(case)) if s > 1 else None
        st["rope"] = None
        if case["rot"]:
            inv = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
            angle = torch.arange(max(final) + 1, dtype=torch.float64, device="cuda")[:, None] * inv
            st["rope"] = (angle.cos().float(), angle.sin().float(), case["rot"], case["neox"])
        return st
    st["mask"] = None
    if case["mask"]:  # left-padded prompts: the first tokens of each sequence are padding
        pad = torch.rand(b, 1, device="cuda", generator=gen) * 0.5 * st["lens"][:, None]
        keep = torch.arange(max(lens), device="cuda")[None] >= pad
        st["mask"] = torch.zeros(b, 1, 1, max(lens), device="cuda").masked_fill(~keep[:, None, None], -math.inf)
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"append": _append, "attend": _attend, "logits": _logits}[state["case"]["op"]](state)


def _append(st):
    if own:
        from oslo_b200.nn import functional as OF

        q = OF.paged_kv_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["lens"], count=st["count"], q=st["q"],
                               rope=st["rope"])
        return q, st["k_pages"], st["v_pages"]
    b, s, page = st["case"]["b"], st["case"]["s"], st["case"]["page"]
    i = torch.arange(s, device="cuda")
    pos = st["lens"][:, None].long() + i
    real = (i < st["count"][:, None]) if st["count"] is not None else torch.ones_like(pos, dtype=torch.bool)
    q, k = _rotate(st["q"], pos, st["rope"]), _rotate(st["k"], pos, st["rope"])
    q = torch.where(real[..., None, None], q, torch.zeros((), dtype=q.dtype, device="cuda"))  # padding has no rotated query
    row, col = real.nonzero(as_tuple=True)
    at = pos[row, col]
    where = st["table"][row, at // page].long()
    st["k_pages"][where, :, at % page] = k[row, col]
    st["v_pages"][where, :, at % page] = st["v"][row, col]
    return q, st["k_pages"], st["v_pages"]


def _rotate(x, pos, rope):
    if rope is None:
        return x.clone()
    cos, sin, rot, neox = rope
    c, s = cos[pos][:, :, None], sin[pos][:, :, None]
    x32 = x.float()
    a, b = (x32[..., : rot // 2], x32[..., rot // 2 : rot]) if neox else (x32[..., 0:rot:2], x32[..., 1:rot:2])
    pair = a * c - b * s, b * c + a * s
    turned = torch.cat(pair, dim=-1) if neox else torch.stack(pair, dim=-1).flatten(-2)
    return torch.cat([turned, x32[..., rot:]], dim=-1).to(x.dtype)


def _attend(st):
    if own:
        from oslo_b200.nn import functional as OF

        return OF.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"], mask=st["mask"])
    q = st["q"]
    b, s, hq, d = q.shape
    hkv = st["k_pages"].shape[1]
    n = st["longest"]

    def gathered(pages):  # [b, hkv, n, d]
        return pages[st["table"].long()].transpose(1, 2).reshape(b, hkv, -1, d)[:, :, :n].float()

    rows = q.float().reshape(b, s, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)  # [b, hkv, s * group, d]
    scores = (rows @ gathered(st["k_pages"]).transpose(-1, -2)).view(b, hkv, s, -1, n) * (1.0 / math.sqrt(d))
    end = st["lens"][:, None] - s + 1 + torch.arange(s, device="cuda")  # [b, s]: each new token sees itself and what came before
    seen = torch.arange(n, device="cuda") < end[..., None]  # [b, s, n]
    if st["mask"] is not None:
        scores = scores + st["mask"].unsqueeze(1)
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(dim=-1, keepdim=True)
    p = (p / total.masked_fill(total == 0, 1.0)).view(b, hkv, -1, n)
    # pages behind a sequence's last token hold other data
    o = p @ gathered(st["v_pages"])
    return o.view(b, hkv, s, -1, d).permute(0, 2, 1, 3, 4).reshape(b, s, hq * d).to(q.dtype)


def _logits(st):
    if own:
        from oslo_b200.nn import functional as OF

        return OF.process_logits(st["logits"], tokens=st["tokens"], token_lengths=st["lens"], prompt_lengths=st["prompts"],
                                 repetition_penalty=st["rep"], presence_penalty=st["pres"], frequency_penalty=st["freq"],
                                 bias=st["bias"], allowed=st["allowed"])
    x = st["logits"].float()
    rows, v = x.shape
    t = torch.arange(st["tokens"].shape[1], device="cuda")
    held = (t < st["lens"][:, None]).float()
    made = held * (t >= st["prompts"][:, None])
    occurred = torch.zeros_like(x).scatter_add_(1, st["tokens"], held) > 0
    count = torch.zeros_like(x).scatter_add_(1, st["tokens"], made)
    rep, pres, freq = (p[:, None] if isinstance(p, torch.Tensor) else p for p in (st["rep"], st["pres"], st["freq"]))
    x = torch.where(occurred, torch.where(x > 0, x / rep, x * rep), x)
    x = x - pres * (count > 0) - freq * count
    if st["bias"] is not None:
        x = x + st["bias"]
    if st["allowed"] is not None:
        j = torch.arange(v, device="cuda")
        ok = (st["allowed"][:, j >> 5] >> (j & 31).to(torch.int32)) & 1
        x = x.masked_fill(ok == 0, -math.inf)
    return x.to(st["logits"].dtype)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "logits":
        rows, v, e = case["rows"], case["v"], SIZES[case["dtype"]]
        held = sum(_history(case)[0])
        n = 2 * rows * v * e + 8 * held + {"none": 0, "shared": 4 * v, "rows": 4 * rows * v}[case["bias"]]
        return dict(bytes=n + (rows * ((v + 31) // 32) * 4 if case["allowed"] else 0), flops=4 * rows * v)
    e, hq, hkv, d, s = SIZES[case["dtype"]], case["hq"], case["hkv"], case["d"], case["s"]
    lens = _lengths(case)
    if case["op"] == "append":
        tokens = sum(_counts(case))
        seen = len({n + i for n, c in zip(lens, _counts(case)) for i in range(c)})  # rows of the rotation's tables
        # padding's rows of the rotated queries are written (zeros), its inputs are not read
        return dict(bytes=e * d * (tokens * (hq + 4 * hkv) + case["b"] * s * hq) + seen * case["rot"] * 4, flops=3 * tokens * (hq + hkv) * case["rot"])
    n = 2 * sum(lens) * hkv * d * e + 2 * case["b"] * s * hq * d * e + (4 * sum(lens) if case["mask"] else 0)
    pairs = sum(max(0, n - i) for n in lens for i in range(s))
    return dict(bytes=n, flops=4 * pairs * hq * d)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logits": _exact_logits}[case["op"]](case, st)


def _exact_append(case, st):
    b, s, page, rot = case["b"], case["s"], case["page"], case["rot"]
    kp, vp = st["k_pages"].double(), st["v_pages"].double()
    qo = torch.zeros(b, s, case["hq"], case["d"], dtype=torch.float64, device="cuda")
    starts, counts, table = st["lens"].tolist(), _counts(case), st["table"].long()
    first, second = [], []
    for j in range(rot // 2):
        first.append(j if case["neox"] else 2 * j)
        second.append(j + rot // 2 if case["neox"] else 2 * j + 1)
    for r in range(b):
        n = counts[r]
        p = torch.arange(starts[r], starts[r] + n, device="cuda")
        q, k = st["q"][r, :n].double(), st["k"][r, :n].double()
        if rot:
            z = torch.complex(st["rope"][0][p].double(), st["rope"][1][p].double())[:, None]
            for x in (q, k):
                w = torch.complex(x[..., first], x[..., second]) * z
                x[..., first], x[..., second] = w.real, w.imag
        qo[r, :n] = q
        pages, offs = table[r, p // page], p % page
        kp[pages, :, offs] = k
        vp[pages, :, offs] = st["v"][r, :n].double()
    return qo, kp, vp


def _exact_attend(case, st):
    b, s, hq, hkv, d, page = (case[x] for x in ("b", "s", "hq", "hkv", "d", "page"))
    if 2.0 * sum(_lengths(case)) * hkv * d > 4e9:
        return None
    out = torch.zeros(b, s, hq, d, dtype=torch.float64, device="cuda")
    for r, n in enumerate(st["lens"].tolist()):
        rows = st["table"][r, : -(-n // page)].long()
        for h in range(hkv if n else 0):
            k = st["k_pages"][rows, h].reshape(-1, d)[:n].double()
            v = st["v_pages"][rows, h].reshape(-1, d)[:n].double()
            g = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            for i in range(s):
                m = n - s + i + 1
                x = st["q"][r, i, g].double() @ k[:m].T / math.sqrt(d)
                if st["mask"] is not None:
                    x = x + st["mask"][r, 0, 0, :m].double()
                out[r, i, g] = torch.softmax(x, dim=-1).nan_to_num(0.0) @ v[:m]
    return out.view(b, s, hq * d)


def _exact_logits(case, st):
    x = st["logits"].double()
    lens, prompts = _history(case)
    per_row = case["per_row"]
    for r in range(case["rows"]):
        rep, pres, freq = (float(st[p][r]) if per_row else float(st[p]) for p in ("rep", "pres", "freq"))
        seen = st["tokens"][r, : lens[r]].unique()
        x[r, seen] = torch.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
        made, n = st["tokens"][r, prompts[r] : lens[r]].unique(return_counts=True)
        x[r, made] -= pres + freq * n.double()
    if st["bias"] is not None:
        x += st["bias"].double()
    if st["allowed"] is not None:
        bits = (st["allowed"][..., None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
        x[bits.flatten(1)[:, : case["v"]] == 0] = -math.inf
    return x
