"""The paged-cache operators of the attention library as measurable cases.

Four operators work on one decoder cache that is kept in pages: ``append``
rotates new Q and K rows and writes K and V into the pages, ``attend`` is the
attention of a ragged batch of new tokens over it, ``score`` adds up the
attention weight that each cached row received, and ``evict`` keeps the rows
with the most weight and closes the gaps.

Where ``own`` is false, run() computes them from elementary torch operations;
where it is true, it calls the library.  A pool is (n_pages, n_head_kv,
page_size, D) halves, or Q8_0 blocks of 34 bytes per 32 values; the rows of a
stream are the pages its page-table row names, in order.
"""
import math
import os
import sys

import torch

own = False

BASE = 1e6            # the decoder's RoPE base
Q8_0_BLOCK = 34


# ---- cases --------------------------------------------------------------------

def _case(name, op, kv, n_seq, hq, hkv, d, page, lo, hi, new_lo, new_hi, **more):
    c = {"name": name, "op": op, "kv": kv, "n_seq": n_seq, "hq": hq, "hkv": hkv, "d": d, "page": page,
         "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi, "mixed": False, "window": 0, "softcap": 0.0,
         "observe": 0, "keep": 0, "sink": 0, "recent": 0}
    c.update(more)
    return c


def listed():
    return [
        # one stream, one token, the single-step decode length: pure latency
        _case("attend 1x1 f16 1k", "attend", "f16", 1, 32, 8, 128, 16, 1023, 1023, 1, 1),
        # a serving step of many ragged streams: K and V are read once
        _case("attend 64x1 f16 ragged", "attend", "f16", 64, 32, 8, 128, 16, 512, 16383, 1, 1),
        # the same step over a quantised cache
        _case("attend 64x1 q8_0 ragged", "attend", "q8_0", 64, 32, 8, 128, 32, 512, 16383, 1, 1),
        # a whole prompt (375 audio tokens and 16 of text) into an empty cache
        _case("attend prompt 391 f16", "attend", "f16", 1, 32, 8, 128, 64, 0, 0, 391, 391),
        # a chunk of a long prompt behind what is cached already: tensor-bound
        _case("attend chunk 2048 at 14k f16", "attend", "f16", 1, 32, 8, 128, 64, 14336, 14336, 2048, 2048),
        # a mixed step: chunks of prompts next to single tokens, ragged
        _case("attend mixed f16", "attend", "f16", 12, 32, 8, 128, 32, 130, 7500, 1, 251, mixed=True),
        # one decode step's new rows of 64 streams
        _case("append 64x1 f16", "append", "f16", 64, 32, 8, 128, 16, 1, 500, 1, 1),
        # prompts of four streams into a quantised cache
        _case("append 4 prompts q8_0", "append", "q8_0", 4, 32, 8, 128, 32, 0, 301, 1500, 2304),
        # a decode step's weights added to the running score
        _case("score 64x1 f16 ragged", "score", "f16", 64, 32, 8, 128, 16, 512, 8191, 1, 1),
        # the last tokens of a chunk vote on what a long prompt keeps
        _case("score chunk 500 at 15k f16", "score", "f16", 1, 32, 8, 128, 64, 15500, 15500, 500, 500),
        # a short cache trimmed to its budget: latency
        _case("evict 1 stream 1k f16", "evict", "f16", 1, 32, 8, 128, 16, 1024, 1024, 0, 0, keep=768, sink=4, recent=64),
        # many long caches brought back to one budget
        _case("evict 32 streams f16", "evict", "f16", 32, 32, 8, 128, 16, 1500, 8192, 0, 0, keep=2048, sink=4, recent=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "score", "evict"])
    kv = rng.choice(["f16", "f16", "q8_0"])
    hkv, g = rng.choice([(8, 4), (8, 4), (8, 4), (20, 1), (4, 8), (2, 2), (5, 3)])
    d = rng.choice([128, 128, 64])
    page = rng.choice([16, 32, 64, 128])
    more = {}
    if op == "attend":
        style = rng.choice(["decode", "chunk", "mixed"])
        if style == "decode":
            n = _log(rng, 1, 80)
            hi = _log(rng, 40, 16000)
            lo, new_lo, new_hi = rng.randint(0, hi), 1, rng.choice([1, 1, 2, 4])
            if n * hi > 600000:
                n = max(1, 600000 // hi)
        elif style == "chunk":
            n = rng.randint(1, 4)
            new_hi = _log(rng, 17, 1400)
            hi = _log(rng, 1, 13000) if rng.random() < 0.8 else 0
            if n * new_hi * (hi + new_hi) > 20000000:
                n = 1
            lo, new_lo = rng.randint(0, hi), max(1, new_hi - rng.randint(0, new_hi // 2))
        else:
            n = rng.randint(3, 14)
            new_lo, new_hi = 1, _log(rng, 20, 250)
            hi = _log(rng, 100, 6000)
            lo, more["mixed"] = rng.randint(0, hi), True
        if rng.random() < 0.25:
            more["window"] = _log(rng, 33, 1500)
        if rng.random() < 0.15:
            more["softcap"] = rng.choice([15.0, 30.0, 50.0])
    elif op == "append":
        n = _log(rng, 1, 100)
        new_lo, new_hi = 1, max(1, _log(rng, 1, 8000) // n)
        hi = rng.randint(0, 600)
        lo = rng.randint(0, hi)
    elif op == "score":
        n = rng.choice([1, 1, 2, 3, _log(rng, 1, 64)])
        new_lo, new_hi = 1, (1 if n > 3 else _log(rng, 1, 400))
        hi = _log(rng, 40, 14000)
        if n * hi > 250000:
            hi = 250000 // n
        lo = rng.randint(0, hi)
        more["observe"] = rng.choice([0, 0, 32])
    else:
        n = _log(rng, 1, 32)
        hi = _log(rng, 65, 16000)
        if n * hi > 250000:
            hi = max(65, 250000 // n)
        lo, new_lo, new_hi = rng.randint(0, hi), 0, 0
        keep = _log(rng, 40, hi)
        more.update(keep=keep, sink=rng.randint(0, 8), recent=rng.randint(0, max(0, keep - 8)) // 2)
    c = _case("", op, kv, n, hkv * g, hkv, d, page, lo, hi, new_lo, new_hi, **more)
    del c["name"]
    return c


def _spread(lo, hi, i, step=0.6180339887498949):
    """The i-th of a fixed sequence spread over [lo, hi]."""
    return lo + int((hi - lo + 1) * math.fmod((i + 0.5) * step, 1.0) * 0.999999)


def _lengths(case):
    """(new tokens, rows in the cache with them) of each stream."""
    n = case["n_seq"]
    new = [_spread(case["new_lo"], case["new_hi"], i, 0.7548776662466927) for i in range(n)]
    if case["mixed"]:                 # one stream in three brings a chunk, the others a token
        new = [max(1, case["new_hi"] - 7 * i) if i % 3 == 0 else 1 for i in range(n)]
    return new, [_spread(case["lo"], case["hi"], i) + new[i] for i in range(n)]


# ---- inputs --------------------------------------------------------------------

def _halves_to_q8(x):
    """Q8_0 bytes of (..., D) float values: d = amax / 127 as a half, then round(x * 127 / amax)."""
    b = x.float().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    q = torch.round(b * torch.where(amax > 0, 127.0 / amax, 0.0)).to(torch.int8)
    return torch.cat([(amax / 127.0).half().view(torch.uint8), q.view(torch.uint8)], -1).flatten(-2)


def _q8_values(raw):
    """(scales, integers) of Q8_0 bytes (..., D / 32 * 34): (..., D / 32, 1) halves and (..., D / 32, 32) int8."""
    b = raw.unflatten(-1, (-1, Q8_0_BLOCK))
    return b[..., :2].contiguous().view(torch.float16), b[..., 2:].view(torch.int8)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    n, hq, hkv, d, ps = case["n_seq"], case["hq"], case["hkv"], case["d"], case["page"]
    new, length = _lengths(case)
    pages = [-(-x // ps) for x in length]
    n_pages, most = sum(pages) + 3, max(max(pages), 1)
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    at = torch.zeros(n, most, dtype=torch.int64)
    first = 0
    for i, p in enumerate(pages):
        at[i, :p] = torch.arange(first, first + p)
        first += p
    table = order[at.to(dev)].contiguous()
    start = [0]
    for x in new:
        start.append(start[-1] + x)
    s = {"case": case, "table": table, "n_tokens": start[-1], "max_new": max(new), "max_len": max(length),
         "kv_len": torch.tensor(length, dtype=torch.int32, device=dev),
         "q_start": torch.tensor(start, dtype=torch.int32, device=dev), "scale": d ** -0.5}
    # cached rows: normal values, one key in fifty three times as long (what the weight gathers on)
    pools = []
    for k in range(2):
        x = torch.randn((n_pages, hkv, ps, d), generator=g, device=dev, dtype=torch.float16)
        if k == 0:
            x = x * torch.where(torch.rand((n_pages, hkv, ps, 1), generator=g, device=dev) < 0.02, 3.0, 1.0).half()
        pools.append(_halves_to_q8(x) if case["kv"] == "q8_0" else x)
    s["k_pool"], s["v_pool"] = pools
    t, cap = s["n_tokens"], most * ps
    # which stream and which row each new token is (the plain forms index with them)
    s["seq"] = torch.repeat_interleave(torch.arange(n, device=dev), torch.tensor(new, device=dev), output_size=t)
    s["row"] = (_nth(s) + (s["kv_len"] - s["q_start"].diff())[s["seq"]]).long()
    if case["op"] == "append":
        s["q"], s["k"], s["v"] = rnd(t, hq, d), rnd(t, hkv, d), rnd(t, hkv, d)
        # an evicted cache's rows are fewer than its positions
        s["positions"] = (s["row"] + torch.randint(0, 20000, (n,), generator=g, device=dev)[s["seq"]]).int()
        s["q_out"] = torch.empty(t, hq, d, dtype=torch.float16, device=dev)
        s["score"] = torch.rand(n, hkv, cap, generator=g, device=dev)
        s["row_pos"] = torch.randint(0, 1000, (n, hkv, cap), generator=g, device=dev, dtype=torch.int32)
    elif case["op"] in ("attend", "score"):
        s["q"] = rnd(t, hq, d).half()
        s["out"] = torch.empty(t, hq, d, dtype=torch.float16, device=dev)
        s["lse"] = torch.empty(t, hq, device=dev)
        if case["op"] == "score":
            s["lse"] = torch.logsumexp(_logits(s, _cached(s, "k_pool")), 3)[s["seq"], :, _nth(s)].contiguous()
            s["score"] = torch.rand(n, hkv, cap, generator=g, device=dev)
            s["score_out"] = torch.zeros_like(s["score"])
    else:
        keep = case["keep"]
        s["score"] = torch.exp(2.0 * rnd(n, hkv, cap)) * (torch.rand(n, hkv, cap, generator=g, device=dev) > 0.1)
        gap = torch.rand(n, hkv, cap, generator=g, device=dev) < 0.05    # rows that an earlier eviction dropped
        s["row_pos"] = (torch.arange(cap, device=dev) + gap.int().cumsum(-1)).int()
        s["next_pos"] = (s["kv_len"] + gap.sum((1, 2)).int() // hkv).int()
        s["score_out"] = torch.zeros(n, hkv, keep, device=dev)
        s["pos_out"] = torch.zeros(n, hkv, keep, dtype=torch.int32, device=dev)
        s["src_out"] = torch.zeros(n, hkv, keep, dtype=torch.int32, device=dev)
        s["kv_len_out"] = torch.zeros(n, dtype=torch.int32, device=dev)
    return s


# ---- the plain forms ------------------------------------------------------------

def _cached(s, pool):
    """(n_seq, n_head_kv, rows, D) float32 of every stream's pages."""
    x = s[pool][s["table"].long()].transpose(1, 2).flatten(2, 3)
    if s["case"]["kv"] == "q8_0":
        scale, q = _q8_values(x)
        return (scale.float() * q.float()).flatten(-2)
    return x.float()


def _nth(s):
    """Which of its stream's new tokens each token is."""
    return torch.arange(s["n_tokens"], device=s["q_start"].device) - s["q_start"][s["seq"]]


def _logits(s, k):
    """(n_seq, hq, new tokens, rows) scores of each stream's new tokens, -inf where a token does not see a row."""
    c = s["case"]
    n, hq, hkv, d = c["n_seq"], c["hq"], c["hkv"], c["d"]
    step = s["max_new"]
    pos = (s["kv_len"] - s["q_start"].diff())[:, None] + torch.arange(step, device=k.device)
    q = torch.zeros(n, step, hq, d, device=k.device)
    q[s["seq"], _nth(s)] = s["q"].float()
    q = q.unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"])
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    x = x.view(n, hq, step, -1)
    j = torch.arange(x.shape[3], device=k.device)
    hidden = (j > pos[..., None]) | (j >= s["kv_len"][:, None, None])
    if c["window"]:
        hidden |= j <= pos[..., None] - c["window"]
    return x.masked_fill_(hidden[:, None], -math.inf)


def _attend(s):
    c = s["case"]
    x = _logits(s, _cached(s, "k_pool"))
    top = x.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    x = x.sub_(top).exp_()
    total = x.sum(3, keepdim=True)
    n, hq, step, rows = x.shape
    o = torch.matmul(x.view(n, c["hkv"], -1, rows), _cached(s, "v_pool")).view(n, hq, step, -1)
    o = o / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total))[..., 0]
    i = _nth(s)
    s["out"].copy_(o[s["seq"], :, i])
    s["lse"].copy_(lse[s["seq"], :, i])
    return {"out": s["out"], "lse": s["lse"]}


def _append(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * BASE ** (-2.0 * torch.arange(c["d"] // 2, device=s["q"].device).double() / c["d"])
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def rotate(x):
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)

    page = s["table"][s["seq"], s["row"] // c["page"]].long()
    put = _halves_to_q8 if c["kv"] == "q8_0" else torch.Tensor.half
    s["q_out"].copy_(rotate(s["q"]))
    s["k_pool"][page, :, s["row"] % c["page"]] = put(rotate(s["k"]))
    s["v_pool"][page, :, s["row"] % c["page"]] = put(s["v"])
    s["score"][s["seq"], :, s["row"]] = 0.0
    s["row_pos"][s["seq"], :, s["row"]] = s["positions"][:, None]


def _score(s):
    c = s["case"]
    n, hq, hkv = c["n_seq"], c["hq"], c["hkv"]
    x = _logits(s, _cached(s, "k_pool"))
    i = _nth(s)
    lse = torch.full((n, s["max_new"], hq), math.inf, device=x.device)
    seen = i >= s["q_start"].diff()[s["seq"]] - c["observe"] if c["observe"] else i >= 0
    lse[s["seq"], i] = torch.where(seen[:, None], s["lse"], math.inf)
    x = x.sub_(lse.transpose(1, 2)[..., None]).exp_()
    got = x.view(n, hkv, -1, x.shape[3]).sum(2)
    live = torch.arange(x.shape[3], device=x.device) < s["kv_len"][:, None, None]
    s["score_out"].copy_(torch.where(live, s["score"] + got, s["score_out"]))
    return {"score": s["score_out"]}


def _evict(s):
    c = s["case"]
    n, hkv, cap = s["score"].shape
    dev = s["score"].device
    j = torch.arange(cap, device=dev)
    live = j < s["kv_len"][:, None, None]
    recent = s["row_pos"] >= (s["next_pos"] - c["recent"])[:, None, None]
    rank = torch.where(live, 1 + ((s["row_pos"] < c["sink"]) | recent).int(), 0)
    value = torch.where(rank == 2, 0.0, torch.nan_to_num(s["score"], nan=-math.inf, posinf=math.inf, neginf=-math.inf))
    order = torch.sort(value, dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, torch.sort(rank.gather(-1, order), dim=-1, descending=True, stable=True).indices)
    left = s["kv_len"].clamp(max=c["keep"])
    kept = torch.zeros_like(rank, dtype=torch.bool).scatter_(-1, order, (j < left[:, None, None]).expand(n, hkv, cap))
    # the i-th gap in front takes the i-th kept row behind it
    front = j < left[:, None, None]
    hole, late = front & ~kept, kept & ~front
    nth = torch.where(late, late.int().cumsum(-1) - 1, cap).long()
    by = torch.zeros(n, hkv, cap + 1, dtype=torch.int64, device=dev).scatter_(-1, nth, j.expand(n, hkv, cap))
    src = torch.where(hole, by.gather(-1, (hole.int().cumsum(-1) - 1).clamp(min=0).long()), j)
    a, h, to = torch.nonzero(hole, as_tuple=True)
    fro = src[a, h, to]
    for pool in ("k_pool", "v_pool"):
        s[pool][s["table"][a, to // c["page"]].long(), h, to % c["page"]] = \
            s[pool][s["table"][a, fro // c["page"]].long(), h, fro % c["page"]]
    m = min(c["keep"], cap)
    keep = front[..., :m].expand(n, hkv, m)
    for out, x in (("score_out", s["score"].gather(-1, src)), ("pos_out", s["row_pos"].gather(-1, src)), ("src_out", src.int())):
        s[out][..., :m] = torch.where(keep, x[..., :m], s[out][..., :m])
    s["kv_len_out"].copy_(left)


# ---- one pass --------------------------------------------------------------------

def _library(s):
    """The library's description of this cache, made once per cache as a program does."""
    if "kv" not in s:
        here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voxtral.cpp_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import vtx_attn
        s["kv"] = vtx_attn.PagedKv(s["k_pool"], s["v_pool"], s["table"], s["kv_len"], s["q_start"], s["case"]["hq"],
                                   n_tokens=s["n_tokens"], max_new=s["max_new"], max_kv_len=s["max_len"])
    return s["kv"]


def _call(s):
    c, kv = s["case"], _library(s)
    if c["op"] == "attend":
        kv.attend(s["q"], out=s["out"], lse=s["lse"], scale=s["scale"], window=c["window"], logit_softcap=c["softcap"])
    elif c["op"] == "append":
        kv.append(s["k"], s["v"], s["positions"], q=s["q"], q_out=s["q_out"], freq_base=BASE, score=s["score"], row_pos=s["row_pos"])
    elif c["op"] == "score":
        kv.score(s["q"], s["lse"], s["score"], score_out=s["score_out"], scale=s["scale"], observe=c["observe"])
    else:
        kv.evict(s["score"], c["keep"], s["kv_len_out"], n_sink=c["sink"], n_recent=c["recent"], row_pos=s["row_pos"],
                 next_pos=s["next_pos"], score_out=s["score_out"], pos_out=s["pos_out"], src_out=s["src_out"])


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        _call(s)
    else:
        {"attend": _attend, "append": _append, "score": _score, "evict": _evict}[op](s)
    if op == "attend":
        return {"out": s["out"], "lse": s["lse"]}
    if op == "score":
        return {"score": s["score_out"]}
    out = {"k": s["k_pool"], "v": s["v_pool"]}
    if op == "append":
        if s["case"]["kv"] == "q8_0":     # blocks as the values they stand for
            out = {k: torch.mul(*_q8_values(x)) for k, x in out.items()}
        out.update(q=s["q_out"], score=s["score"], row_pos=s["row_pos"])
    else:
        out.update(score=s["score_out"], pos=s["pos_out"], src=s["src_out"], kv_len=s["kv_len_out"])
    return out


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    new, length = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    row = hkv * (d // 32 * Q8_0_BLOCK if case["kv"] == "q8_0" else d * 2)      # one token's K (or V) of all heads
    t = sum(new)
    if case["op"] == "append":
        return {"bytes": t * ((hq + 2 * hkv) * d * 4 + hq * d * 2 + 2 * row + hkv * 8 + 4), "flops": t * (hq + hkv) * d * 3}
    if case["op"] == "evict":
        moved = rows = kept = 0
        for x in length:
            m = min(x, case["keep"])
            rows, kept = rows + x, kept + m
            moved += m * (x - m) / max(x, 1)         # about the share of the kept rows that stands behind the new end
        return {"bytes": hkv * (rows * 8 + kept * 12) + moved * row * 4, "flops": 0}
    pairs = seen = 0
    w = case["window"]
    for a, x in zip(new, length):
        o = min(a, case["observe"]) if case["observe"] else a
        pairs += sum(min(x - i, w) if w else x - i for i in range(o))
        seen += min(x, w + o - 1) if w else x
    if case["op"] == "attend":
        return {"bytes": 2 * seen * row + t * hq * (4 * d + 4), "flops": 4 * d * hq * pairs}
    return {"bytes": seen * row + sum(length) * hkv * 8 + t * hq * (2 * d + 4), "flops": 2 * d * hq * pairs}


# ---- the definition in 64 bits -------------------------------------------------------

def _rows64(s, pool, i):
    """(n_head_kv, rows, D) float64 rows of stream i's cache."""
    c, n = s["case"], int(s["kv_len"][i])
    x = torch.cat([s[pool][int(p)] for p in s["table"][i, :-(-n // c["page"])]] or [s[pool][0][:, :0]], 1)[:, :n]
    if c["kv"] != "q8_0":
        return x.double()
    b = x.reshape(c["hkv"], n, c["d"] // 32, Q8_0_BLOCK)
    low = b[..., 0].to(torch.int32) + 256 * b[..., 1].to(torch.int32)
    scale = torch.where(low > 32767, low - 65536, low).to(torch.int16).view(torch.float16).double()
    q = b[..., 2:].to(torch.int16)
    return (scale[..., None] * torch.where(q > 127, q - 256, q).double()).reshape(c["hkv"], n, c["d"])


def _weights64(s, i, h, first, count):
    """exp-ready scores of queries first .. first + count of stream i, head h: (count, rows) float64, -inf where unseen."""
    c, n = s["case"], int(s["kv_len"][i])
    q0, q1 = int(s["q_start"][i]), int(s["q_start"][i + 1])
    k = s["rows64"][h // (c["hq"] // c["hkv"])]
    x = s["q"][q0 + first:q0 + first + count, h].double() @ k.T / math.sqrt(c["d"])
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    p = n - (q1 - q0) + first + torch.arange(count, device=x.device)[:, None]
    j = torch.arange(n, device=x.device)[None]
    see = j <= p
    if c["window"]:
        see &= j > p - c["window"]
    return torch.where(see, x, -math.inf)


def _exact_attention(s):
    c = s["case"]
    out = torch.zeros(s["n_tokens"], c["hq"], c["d"], dtype=torch.float64, device="cuda")
    lse = torch.full((s["n_tokens"], c["hq"]), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(c["n_seq"]):
        a, b = int(s["q_start"][i]), int(s["q_start"][i + 1])
        if a == b:
            continue
        s["rows64"], v = _rows64(s, "k_pool", i), _rows64(s, "v_pool", i)
        for h in range(c["hq"]):
            x = _weights64(s, i, h, 0, b - a)
            lse[a:b, h] = torch.logsumexp(x, 1)
            out[a:b, h] = torch.nan_to_num(torch.exp(x - lse[a:b, h, None])) @ v[h // (c["hq"] // c["hkv"])]
    return {"out": out, "lse": lse}


def _exact_score(s):
    c = s["case"]
    got = s["score_out"].double()
    for i in range(c["n_seq"]):
        a, b, n = int(s["q_start"][i]), int(s["q_start"][i + 1]), int(s["kv_len"][i])
        got[i, :, :n] = s["score"][i, :, :n].double()
        s["rows64"] = _rows64(s, "k_pool", i)
        o = min(b - a, c["observe"]) if c["observe"] else b - a
        for h in range(c["hq"]):
            x = _weights64(s, i, h, b - a - o, o)
            got[i, h // (c["hq"] // c["hkv"]), :n] += torch.exp(x - s["lse"][b - o:b, h].double()[:, None]).sum(0)
    return {"score": got}


def _exact_append(s):
    c = s["case"]
    t, d = s["n_tokens"], c["d"]
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None, None] *
                    torch.exp(torch.arange(d // 2, device="cuda").double() * (-2.0 / d * math.log(BASE))))
    turn = lambda x: torch.view_as_real(torch.view_as_complex(x.double().reshape(t, -1, d // 2, 2).contiguous()) * z).reshape(t, -1, d)  # noqa: E731
    q8 = c["kv"] == "q8_0"

    def pool64(name):
        x = s[name]
        if not q8:
            return x.double()
        scale, q = _q8_values(x)
        return scale.double() * q.double()

    out = {"k": pool64("k_pool"), "v": pool64("v_pool"), "q": turn(s["q"]), "score": s["score"].double(), "row_pos": None}
    where = s["table"][s["seq"], torch.div(s["row"], c["page"], rounding_mode="floor")].long()
    for name, x in (("k", turn(s["k"])), ("v", s["v"].double())):
        if q8:
            x = x.reshape(t, -1, d // 32, 32)
            top = x.abs().amax(-1, keepdim=True)
            x = (top / 127).half().double() * torch.round(x * 127 / top.clamp(min=1e-300))
        out[name][where, :, s["row"] % c["page"]] = x
    out["score"][s["seq"], :, s["row"]] = 0
    return out


def _exact_evict(s):
    c = s["case"]
    keep, sc = c["keep"], s["score"].double().cpu()
    pos, nxt, table = s["row_pos"].cpu(), s["next_pos"].tolist(), s["table"].cpu()
    out = {"k": s["k_pool"].clone(), "v": s["v_pool"].clone(), "score": s["score_out"].double().cpu()}
    to_page, to_row, from_page, from_row, head = [], [], [], [], []
    for i, n in enumerate(s["kv_len"].tolist()):
        m = min(n, keep)
        for h in range(c["hkv"]):
            safe = (pos[i, h, :n] < c["sink"]) | (pos[i, h, :n] >= nxt[i] - c["recent"])
            want = torch.where(safe, math.inf, sc[i, h, :n])
            best = torch.argsort(-want, stable=True)[:m]
            inside = torch.zeros(n, dtype=torch.bool)
            inside[best] = True
            gaps, tail = torch.nonzero(~inside[:m]).flatten(), m + torch.nonzero(inside[m:]).flatten()
            moved = torch.arange(m)
            moved[gaps] = tail
            out["score"][i, h, :m] = sc[i, h, moved]
            to_page.append(table[i, gaps // c["page"]]); to_row.append(gaps % c["page"])
            from_page.append(table[i, tail // c["page"]]); from_row.append(tail % c["page"])
            head.append(torch.full((len(gaps),), h))
    tp, tr, fp, fr, hd = (torch.cat(x).long().cuda() for x in (to_page, to_row, from_page, from_row, head))
    for k in ("k", "v"):
        out[k][tp, hd, tr] = out[k][fp, hd, fr]
    q8 = c["kv"] == "q8_0"                        # bytes have no value in 64 bits
    return {"k": None if q8 else out["k"].double(), "v": None if q8 else out["v"].double(), "score": out["score"],
            "pos": None, "src": None, "kv_len": None}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attention, "append": _exact_append, "score": _exact_score, "evict": _exact_evict}[case["op"]](s)
