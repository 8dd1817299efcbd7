"""The paged key/value cache beside the feed-forward layer, as cases that can be timed and compared.

A case is one call an inference engine makes of ``biv_b200.cache.PagedCache`` in a decoder layer's
attention half:

  op      "extend"  pages for the new tokens of a batch of requests: block table, slot map, positions
          "store"   rotary positions of one or several axes on q and k; k and v into their pages
          "attend"  attention of each request's new tokens over its pages; with a window and first
                    tokens that stay visible (sinks) where the case has them

``run`` computes the same in elementary torch operations where ``own`` is false.  The lengths of a
batch's requests follow from the case alone, the values of all rows from the seed.
"""
import math
import random

import torch

own = False
_DEV = "cuda:0"
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------
def _extend(seqs, new, past, page):
    """`new` and `past`: the least and the most of a request, as texts "lo..hi"."""
    return dict(op="extend", seqs=seqs, new=new, past=past, page=page)


def _store(tokens, heads, heads_kv, dim, rot, axes, interleaved, adjacent, rows, type, page, order):
    return dict(op="store", tokens=tokens, heads=heads, heads_kv=heads_kv, dim=dim, rot=rot, axes=axes,
                interleaved=interleaved, adjacent=adjacent, rows=rows, type=type, page=page, order=order)


def _attend(seqs, new, past, heads, heads_kv, dim, type, page, order="token", window=0, sinks=0):
    return dict(op="attend", seqs=seqs, new=new, past=past, heads=heads, heads_kv=heads_kv, dim=dim, type=type,
                page=page, order=order, window=window, sinks=sinks)


def listed():
    return [
        # a server's decode step: one token for each of 64 conversations
        dict(_extend(64, "1..1", "1..8192", 16), name="tables_decode_64"),
        # a full server: prompts, chunks of prompts, decode steps and idle places together
        dict(_extend(1000, "0..64", "0..4096", 16), name="tables_mixed_1000"),
        # one token of one conversation, image-and-text positions on a quarter of the head
        dict(_store(1, 16, 2, 256, 64, 3, True, False, "f32", "bf16", 16, "token"), name="store_token_1"),
        # many prompts with images, at once: three axes in contiguous sections over the whole head
        dict(_store(16381, 32, 8, 128, 128, 3, False, False, "bf16", "bf16", 64, "head"), name="store_images_16381"),
        # one token of one conversation: latency
        dict(_attend(1, "1..1", "1000..1000", 16, 2, 256, "bf16", 16), name="decode_1"),
        # a server's decode step: the cache is read once
        dict(_attend(64, "1..1", "1..8192", 32, 8, 128, "bf16", 16), name="decode_64"),
        # 32 conversations x 5 drafted tokens verified
        dict(_attend(32, "5..5", "2000..16000", 16, 2, 256, "bf16", 64), name="verify_32x5"),
        # a chunk of a long prompt: the largest
        dict(_attend(1, "2048..2048", "30000..30000", 32, 8, 128, "bf16", 64), name="chunk_2048_at_30000"),
        # a whole prompt, wide heads
        dict(_attend(1, "4096..4096", "0..0", 16, 2, 256, "bf16", 16), name="prompt_4096_wide"),
        # ragged prompts and chunks, an odd number of heads to a group
        dict(_attend(9, "1..1500", "0..700", 14, 2, 64, "f16", 16, "head"), name="prompts_ragged_f16"),
        # a decode step of a model with windowed layers: long conversations, little of each in sight
        dict(_attend(128, "1..1", "1..30000", 64, 8, 64, "bf16", 16, "token", 1024, 4), name="window_decode_128"),
        # a long prompt through a windowed layer
        dict(_attend(1, "8192..8192", "0..0", 32, 4, 128, "f16", 32, "token", 1024, 4), name="window_prompt_8192"),
    ]


def _log_uniform(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _range(rng, hi):
    lo = rng.choice([0, hi // 3, hi])
    return "%d..%d" % (lo, hi)


def draw(rng):
    op = rng.choice(["extend", "store", "attend", "attend", "attend"])
    page = rng.choice([8, 16, 16, 32, 48, 64, 128, 256])
    type = rng.choice(["bf16", "bf16", "f16"])
    order = rng.choice(["token", "head"])
    if op == "extend":
        return _extend(_log_uniform(rng, 1, 1000), _range(rng, _log_uniform(rng, 1, 64)), _range(rng, _log_uniform(rng, 1, 8192)), page)
    dim = rng.choice([64, 128, 256])
    heads_kv = rng.choice([1, 2, 4, 8] if dim < 256 else [1, 2, 4])
    heads = heads_kv * rng.choice([1, 2, 4, 7, 8])
    if op == "store":
        rot = rng.choice([dim, dim // 2])
        axes = rng.choice([1, 3])
        return _store(_log_uniform(rng, 1, 16000 * 40 * 128 // ((heads + 2 * heads_kv) * dim) + 1), heads, heads_kv, dim, rot, axes,
                      rng.choice([False, True]), rng.choice([False, True]), rng.choice(["f32", type]), type, page, order)
    most = work(listed()[7])
    while True:
        seqs = _log_uniform(rng, 1, 128)
        new = rng.choice([1, 1, _log_uniform(rng, 2, 16), _log_uniform(rng, 16, 8192)])
        past = _log_uniform(rng, 1, 32000) * rng.choice([0, 1, 1, 1])
        window = rng.choice([0, 0, _log_uniform(rng, 16, 4096)])
        c = _attend(seqs, _range(rng, new), _range(rng, past), heads, heads_kv, dim, type, page, order, window,
                    rng.choice([0, 1, 4, 130]) if window else 0)
        w, (n, p) = work(c), _lengths(c)
        padded = seqs * (max(n) + 0) * max(a + b for a, b in zip(n, p)) * heads
        if w["flops"] > 0 and w["flops"] <= most["flops"] and w["bytes"] <= 2.5e9 and padded <= 2.2e9 and \
                seqs * max(a + b for a, b in zip(n, p)) * heads_kv * dim <= 1.5e9:
            return c


def _lengths(case):
    """(new, past) tokens of each request: a function of the case."""
    r = random.Random("lengths %d %s %s" % (case["seqs"], case["new"], case["past"]))

    def some(text):
        lo, hi = (int(v) for v in text.split(".."))
        return [r.randint(lo, hi) for _ in range(case["seqs"])]

    new, past = some(case["new"]), some(case["past"])
    if not any(new):
        new[0] = 1
    return new, past


def _sections(case):
    """Pairs of each axis: the first takes what the others leave."""
    pairs = case["rot"] // 2
    if case["axes"] == 1:
        return [pairs]
    part = pairs // 3
    return [pairs - 2 * part, part, part]


def _seen(p, window, sinks):
    """How many of the positions up to p a token at p sees."""
    if not window or p + 1 <= window:
        return p + 1
    return window + min(sinks, p + 1 - window)


def work(case):
    if case["op"] == "extend":
        new, past = _lengths(case)
        page = case["page"]
        pages = sum(-(-(n + p) // page) - -(-p // page) for n, p in zip(new, past))
        # lengths in, length and first token out; a free page read and its table entry written; slot and position of a token
        return {"bytes": 16 * case["seqs"] + 8 * pages + 12 * sum(new), "flops": 0}
    size = 2
    if case["op"] == "store":
        rows = case["tokens"] * (case["heads"] + 2 * case["heads_kv"]) * case["dim"]
        into = 4 if case["rows"] == "f32" else 2
        return {"bytes": rows * (into + size) + case["tokens"] * (8 + 4 * case["axes"]),
                "flops": 3 * case["tokens"] * (case["heads"] + case["heads_kv"]) * case["rot"]}
    new, past = _lengths(case)
    w, s = case["window"], case["sinks"]
    pairs = keys = 0
    for n, p in zip(new, past):
        if not n:
            continue
        if not w:
            pairs += n * p + n * (n + 1) // 2
            keys += n + p
        else:
            pairs += sum(_seen(x, w, s) for x in range(p, p + n))
            lo = max(0, p - w + 1)           # the first of the positions that some row's window reaches
            keys += n + p - lo + min(s, lo)
    return {"bytes": 2 * size * keys * case["heads_kv"] * case["dim"] + 2 * size * sum(new) * case["heads"] * case["dim"],
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- inputs --------------------------------------------------------------------------------------
def _pool(g, pages, case, type):
    """[pages, page, heads_kv, dim]; a head's tokens are neighbours in memory where the order is "head"."""
    page, h, d = case["page"], case["heads_kv"], case["dim"]
    if case["order"] == "head":
        return torch.randn((pages, h, page, d), generator=g, device=_DEV, dtype=type).transpose(1, 2)
    return torch.randn((pages, page, h, d), generator=g, device=_DEV, dtype=type)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=_DEV)


def _table(g, counts, width, spare=0):
    """Pages of each request, anywhere in the pool, -1 past them; and pages that are free."""
    total = sum(counts)
    order = torch.randperm(total + spare, generator=g, device=_DEV, dtype=torch.int32)
    have = _ints(counts)
    at = torch.arange(width, device=_DEV)
    start = (torch.cumsum(have, 0) - have)[:, None]
    table = torch.where(at[None] < have[:, None], order[(start + at[None]).clamp(max=total + spare - 1)], -1)
    return table.to(torch.int32).contiguous(), order[total:].contiguous()


def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 1000003 + 17)
    s = {"case": case}
    if case["op"] == "extend":
        new, past = _lengths(case)
        page = case["page"]
        width = max(-(-(n + p) // page) for n, p in zip(new, past)) + 2
        need = sum(-(-(n + p) // page) - -(-p // page) for n, p in zip(new, past))
        s["table"], s["free"] = _table(g, [-(-p // page) for p in past], width, need + 5)
        s.update(new=_ints(new), past=_ints(past), free_count=_ints([need + 5]), n=sum(new))
        _handle(s, 1, 1, 64, len(new), s["n"], torch.bfloat16, None)
        return s
    type = _TYPES[case["type"]]
    h, hk, d = case["heads"], case["heads_kv"], case["dim"]
    if case["op"] == "store":
        n, page = case["tokens"], case["page"]
        into = _TYPES[case["rows"]]
        # q, k and v as one product leaves them: neighbours in one row
        rows = torch.randn((n, h + 2 * hk, d), generator=g, device=_DEV, dtype=into)
        s["q"], s["k"], s["v"] = rows[:, :h], rows[:, h:h + hk], rows[:, h + hk:]
        pages = -(-n // page) + 3
        s["k_pool"], s["v_pool"] = _pool(g, pages, case, type), _pool(g, pages, case, type)
        order = torch.randperm(pages, generator=g, device=_DEV)
        at = torch.arange(n, device=_DEV)
        s["slots"] = order[at // page] * page + at % page
        # a conversation of up to 32768 tokens; an image's tokens share a time and have a row and a column
        start = torch.randint(0, 16384, (1,), generator=g, device=_DEV)
        time = start + at
        s["positions"] = (time[None] if case["axes"] == 1 else
                          torch.stack([time - at % 64, start + at // 64, start + at % 64])).to(torch.int32).contiguous()
        _handle(s, h, hk, d, 1, n, type, case)
        return s
    new, past = _lengths(case)
    page = case["page"]
    counts = [-(-(n + p) // page) for n, p in zip(new, past)]
    s["table"], _ = _table(g, counts, max(counts))
    pages = sum(counts)
    s["k_pool"], s["v_pool"] = _pool(g, pages, case, type), _pool(g, pages, case, type)
    n = sum(new)
    s["q"] = torch.randn((n, h, d), generator=g, device=_DEV, dtype=type)
    first = [0]
    for v in new:
        first.append(first[-1] + v)
    s.update(first=_ints(first), length=_ints([a + b for a, b in zip(new, past)]), max_new=max(new))
    _handle(s, h, hk, d, len(new), n, type, None)
    return s


def _handle(s, heads, heads_kv, dim, seqs, tokens, type, rope):
    """The framework's handle (geometry and workspace), which a user's program keeps."""
    if not own:
        return
    from biv_b200.cache import PagedCache, Rope
    if rope is not None:
        rope = Rope(rope["rot"], sections=_sections(rope), interleaved=rope["interleaved"], adjacent=rope["adjacent"])
    s["cache"] = PagedCache(heads, heads_kv, dim, s["case"]["page"], max_seqs=seqs, max_tokens=tokens, dtype=type, rope=rope)


# ---- one pass ------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if not own:
        return {"extend": _extend_plain, "store": _store_plain, "attend": _attend_plain}[op](s)
    c = s["cache"]
    if op == "extend":
        step = c.extend(s["past"], s["new"], s["free"], s["free_count"], s["table"], s["n"])
        return [s["table"], step.length, step.first, step.slots, step.positions, step.left]
    if op == "store":
        return [c.store(s["q"], s["k"], s["v"], s["k_pool"], s["v_pool"], s["slots"], s["positions"]), s["k_pool"], s["v_pool"]]
    return [c.attend(s["q"], s["k_pool"], s["v_pool"], s["table"], s["first"], s["length"], max_new=s["max_new"],
                     window=s["case"]["window"], sinks=s["case"]["sinks"])]


def _extend_plain(s):
    page, past, new, n, table = s["case"]["page"], s["past"], s["new"], s["n"], s["table"]
    length = past + new
    have = (past + page - 1) // page
    need = (length + page - 1) // page - have
    upto = torch.cumsum(need, 0, dtype=torch.int32)
    place = torch.arange(table.shape[1], device=_DEV, dtype=torch.int32)[None]
    i = (upto - need)[:, None] + place - have[:, None]          # which of the free pages
    taken = (place >= have[:, None]) & (place < (have + need)[:, None])
    free = s["free"][(s["free_count"] - 1 - i).clamp(0, s["free"].numel() - 1)]
    table.copy_(torch.where(taken, torch.where(i < s["free_count"], free, -1), table))
    first = torch.zeros(past.numel() + 1, dtype=torch.int32, device=_DEV)
    first[1:] = torch.cumsum(new, 0)
    t = torch.arange(n, device=_DEV, dtype=torch.int32)
    b = torch.searchsorted(first[1:], t, right=True)
    p = past[b] + t - first[b]
    at = table[b, p // page].long()
    slots = torch.where(at < 0, -1, at * page + p % page)
    left = torch.cat([(s["free_count"] - upto[-1:]).clamp(min=0), (upto[-1:] - s["free_count"]).clamp(min=0)])
    return [table, length, first, slots, p, left]


def _axis_of_pair(case):
    """Which axis turns each pair of the head's rotated part."""
    sec, pairs = _sections(case), case["rot"] // 2
    if case["interleaved"] and len(sec) > 1:
        a = len(sec)
        return [i % a if i % a and i < a * sec[i % a] else 0 for i in range(pairs)]
    return [k for k, v in enumerate(sec) for _ in range(v)]


def _turn(x, cos, sin, rot, adjacent):
    """x [n, heads, dim]; the pairs are neighbours, or half the rotated part apart."""
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if adjacent else (r[..., :rot // 2], r[..., rot // 2:])
    u, v = a * cos - b * sin, a * sin + b * cos
    r = torch.stack([u, v], -1).flatten(-2) if adjacent else torch.cat([u, v], -1)
    return torch.cat([r, rest], -1)


def _store_plain(s):
    case = s["case"]
    rot, type = case["rot"], s["k_pool"].dtype
    axis = torch.tensor(_axis_of_pair(case), device=_DEV)
    freq = torch.pow(10000.0, torch.arange(rot // 2, device=_DEV, dtype=torch.float32) * (-2.0 / rot))
    angle = (s["positions"].float()[axis] * freq[:, None]).T[:, None]    # [n, 1, pairs]
    cos, sin = torch.cos(angle), torch.sin(angle)
    q = _turn(s["q"].float(), cos, sin, rot, case["adjacent"]).to(type)
    k = _turn(s["k"].float(), cos, sin, rot, case["adjacent"]).to(type)
    page, at = s["slots"] // case["page"], s["slots"] % case["page"]
    s["k_pool"][page, at] = k
    s["v_pool"][page, at] = s["v"].to(type)
    return [q, s["k_pool"], s["v_pool"]]


def _attend_plain(s):
    case, q, table, first, length = s["case"], s["q"], s["table"], s["first"], s["length"]
    hk, d, page, w = case["heads_kv"], case["dim"], case["page"], case["window"]
    g, b, n = case["heads"] // hk, table.shape[0], s["max_new"]
    keys = table.shape[1] * page
    pages = table.clamp(min=0).long()
    k = s["k_pool"][pages].reshape(b, keys, hk, d).permute(0, 2, 3, 1).float()      # [b, hk, d, keys]
    v = s["v_pool"][pages].reshape(b, keys, hk, d).permute(0, 2, 1, 3).float()
    i = torch.arange(n, device=_DEV)[None]
    new = (first[1:] - first[:-1])[:, None]
    rows = (first[:-1, None] + i).clamp(max=q.shape[0] - 1).long()
    qp = q[rows].reshape(b, n, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, n * g, d).float()
    p = ((length[:, None] - new + i))[:, :, None]                                   # [b, n, 1]
    j = torch.arange(keys, device=_DEV)[None, None]
    see = (j <= p) & (i < new)[:, :, None]
    if w:
        see &= (j > p - w) | (j < case["sinks"])
    hide = ~see[:, None, :, None, :]
    x = torch.matmul(qp, k).mul_(1.0 / math.sqrt(d)).view(b, hk, n, g, keys)
    x.masked_fill_(hide, float("-inf"))
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hk, n * g, keys), v).view(b, hk, n, g, d) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 2, 1, 3, 4).reshape(b * n, hk * g, d)
    t = torch.arange(q.shape[0], device=_DEV, dtype=torch.int32)
    of = torch.searchsorted(first[1:].contiguous(), t, right=True)
    return [o[of * n + (t - first[of])].to(q.dtype)]


# ---- the same in 64 bits ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False       # the inputs alone: no handle
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "extend":
        return None
    if case["op"] == "store":
        sec, rot, n = _sections(case), case["rot"], case["tokens"]
        c = torch.empty((n, rot // 2), dtype=torch.float64, device=_DEV)
        for i in range(rot // 2):
            if not case["interleaved"] or len(sec) == 1:
                axis = sum(i >= sum(sec[:k + 1]) for k in range(len(sec)))
            else:
                axis = i % len(sec)
                axis = axis if i < len(sec) * sec[axis] else 0
            c[:, i] = s["positions"][axis].double() * 10000.0 ** (-2.0 * i / rot)
        z = torch.polar(torch.ones_like(c), c)[:, None]

        def turned(x):
            x = x.double().clone()
            one, two = ((slice(0, rot, 2), slice(1, rot, 2)) if case["adjacent"] else (slice(0, rot // 2), slice(rot // 2, rot)))
            y = torch.complex(x[..., one], x[..., two]) * z
            x[..., one], x[..., two] = y.real, y.imag
            return x

        kp, vp = s["k_pool"].double(), s["v_pool"].double()
        page, at = torch.div(s["slots"], case["page"], rounding_mode="floor"), torch.remainder(s["slots"], case["page"])
        kp.index_put_((page, at), turned(s["k"]))
        vp.index_put_((page, at), s["v"].double())
        return [turned(s["q"]), kp, vp]
    new, past = _lengths(case)
    g, d, w = case["heads"] // case["heads_kv"], case["dim"], case["window"]
    if work(case)["flops"] > 4e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    at = 0
    for b, (n, p) in enumerate(zip(new, past)):
        if not n:
            continue
        used = s["table"][b, :-(-(n + p) // case["page"])].long()
        mine = torch.arange(p, p + n, device=_DEV)[:, None] - torch.arange(n + p, device=_DEV)[None]   # how far back a key lies
        see = mine >= 0
        if w:
            see &= (mine < w) | (torch.arange(n + p, device=_DEV)[None] < case["sinks"])
        for h in range(case["heads_kv"]):
            kk = s["k_pool"][used, :, h].reshape(-1, d)[:n + p].double()
            vv = s["v_pool"][used, :, h].reshape(-1, d)[:n + p].double()
            for r in range(h * g, (h + 1) * g):
                x = s["q"][at:at + n, r].double() @ kk.T / math.sqrt(d)
                out[at:at + n, r] = torch.softmax(x.masked_fill_(~see, -math.inf), -1) @ vv
        at += n
    return [out]
