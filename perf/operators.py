"""Measured cases of the batched-serving operators: step planning, the 8-bit paged K/V cache
(write, read back), attention over that cache, and the rules applied to logits.

Every operator has a plain form here (elementary torch operations in 32 bits) and the
framework's call; ``own`` chooses. Head layouts are those of the repository's configurations:
16 heads of 64 (311M), 16 query / 4 key heads of 128 (1.3B), 32 / 8 of 128 (8B).
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DEV = "cuda"
_QMAX = {"e4m3": 448.0, "int8": 127.0}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a small interactive server: launch latency only
        {"name": "plan 8 requests", "op": "plan", "requests": 8, "context": 500, "new": 1,
         "page": 64, "pattern": 1},
        # a large server's mixed step: mostly decoding, some prompts arriving
        {"name": "plan 700 mixed", "op": "plan", "requests": 700, "context": 4096, "new": 48,
         "page": 16, "pattern": 2},
        # decode step of a busy server, 1.3B heads: one token into a partly filled page each
        {"name": "append decode 64", "op": "append", "requests": 64, "context": 2048, "new": 1,
         "q_heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "codes": "e4m3", "pattern": 3},
        # prompts of the 311M model arriving together, ragged, int8 codes, small pages
        {"name": "append prompts 311M", "op": "append", "requests": 24, "context": 0, "new": 512,
         "q_heads": 16, "kv_heads": 16, "dim": 64, "page": 16, "codes": "int8", "pattern": 4},
        # a long prompt and a few shorter ones in the 8B head layout, continued mid-page
        {"name": "append long 8B", "op": "append", "requests": 4, "context": 777, "new": 32768,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "codes": "e4m3", "pattern": 5},
        # one user of the 311M model, next token: latency
        {"name": "decode 1 x 512", "op": "attend", "requests": 1, "context": 500, "new": 1,
         "q_heads": 16, "kv_heads": 16, "dim": 64, "page": 64, "codes": "e4m3", "pattern": 6},
        # one user with a 32k context on the 1.3B model: the long axis is split over the GPU
        {"name": "decode 1 x 32k", "op": "attend", "requests": 1, "context": 32767, "new": 1,
         "q_heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "codes": "int8", "pattern": 7},
        # a full server of the 8B shape, ragged contexts: cache bandwidth
        {"name": "decode 128 ragged", "op": "attend", "requests": 128, "context": 4096, "new": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "codes": "e4m3", "pattern": 8},
        # prompts of the 311M model in odd lengths, attended after being written
        {"name": "prefill 311M", "op": "attend", "requests": 16, "context": 0, "new": 509,
         "q_heads": 16, "kv_heads": 16, "dim": 64, "page": 16, "codes": "int8", "pattern": 9},
        # chunks of long prompts of the 8B shape over what is cached already: tensor cores
        {"name": "prefill 8B chunks", "op": "attend", "requests": 3, "context": 2048, "new": 2048,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "codes": "e4m3", "pattern": 10},
        # next token of one request, small vocabulary: latency
        {"name": "logits 1 x 8192", "op": "logits", "requests": 1, "vocab": 8192, "history": 500,
         "bias": 4, "mask": True, "half": True, "pattern": 11},
        # next tokens of a full server with long histories
        {"name": "logits 128 x 32768", "op": "logits", "requests": 128, "vocab": 32768,
         "history": 4096, "bias": 32, "mask": True, "half": True, "pattern": 12},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    largest = {}
    for c in listed():
        w = _cost(c)
        largest[c["op"]] = max(largest.get(c["op"], 0.0), w)
    while True:
        op = rng.choice(["plan", "append", "attend", "attend", "logits"])
        c = {"op": op, "pattern": rng.randrange(1 << 20)}
        if op == "logits":
            c.update(requests=_spread(rng, 1, 128), vocab=_spread(rng, 1000, 60000),
                     history=_spread(rng, 1, 8192), bias=rng.choice([0, 1, 7, 64]),
                     mask=rng.random() < 0.6, half=rng.random() < 0.7)
        elif op == "plan":
            c.update(requests=_spread(rng, 1, 1000), context=_spread(rng, 1, 8192),
                     new=rng.choice([1, 1, _spread(rng, 2, 64)]), page=rng.choice([16, 32, 64, 128]))
        else:
            hq, hkv, d = rng.choice([(16, 16, 64), (16, 4, 128), (32, 8, 128), (12, 4, 64),
                                     (8, 8, 128), (14, 2, 64), (16, 1, 128), (40, 8, 128)])
            decode = rng.random() < 0.5
            c.update(requests=_spread(rng, 1, 128), context=_spread(rng, 1, 32768) - 1,
                     new=rng.choice([1, 1, 1, 2, 5]) if decode else _spread(rng, 6, 4096),
                     q_heads=hq, kv_heads=hkv, dim=d, page=rng.choice([16, 32, 64, 128]),
                     codes=rng.choice(["e4m3", "int8"]))
        w = _cost(c)
        if largest[op] >= w and w * 4000 >= largest[op]:
            return c


def _lens(c):
    """(context lengths, new lengths) of the requests, from the case alone."""
    rng = random.Random(c["pattern"])
    n, ctx, new = c["requests"], c["context"], c["new"]
    if n == 1:
        return [ctx], [new]
    # contexts from an eighth of the largest to the largest; every fourth at its full length
    contexts = [ctx if i % 4 == 0 else int(ctx * rng.uniform(0.125, 1.0)) for i in range(n)]
    if c["op"] == "plan" and new > 1:    # mixed steps: three in four decode
        news = [1 if i % 4 else rng.randint(1, 4 * new) for i in range(n)]
    elif new <= 8:
        news = [new] * n
    else:
        news = [new if i == 0 else max(1, int(new * rng.uniform(0.125, 1.0))) for i in range(n)]
    return contexts, news


def _cost(c):
    """The plain form's weight of a case, to keep drawn cases below the listed ones."""
    if c["op"] == "logits":
        return c["requests"] * (c["vocab"] + c["history"])
    ctx, new = _lens(c)
    if c["op"] == "plan":
        return c["requests"] + sum(new)
    rows, pages = sum(new), c["kv_heads"] * c["dim"]
    if c["op"] == "append":
        return pages * (rows + c["page"] * len(ctx))
    longest = max(a + b for a, b in zip(ctx, new))
    # padded scores and padded keys of the plain form
    return len(ctx) * longest * (2 * pages + c["q_heads"] * max(new) * 1.5)


# ------------------------------------------------------------------------------ inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=_DEV)


def _plan_host(contexts, news, tables, page):
    """Step plan of host lists: (q_starts, kv_lens, positions, slots, touched)."""
    starts, pos, slots, touched = [0], [], [], []
    for b, (c, n) in enumerate(zip(contexts, news)):
        row = starts[-1]
        starts.append(row + n)
        at = c
        while at < c + n:
            stop = min(c + n, (at // page + 1) * page)
            touched.append((tables[b][at // page], row + at - c, at % page, stop - at))
            slots.extend(tables[b][at // page] * page + i % page for i in range(at, stop))
            pos.extend(range(at, stop))
            at = stop
    return starts, [c + n for c, n in zip(contexts, news)], pos, slots, touched


def _power(e):
    """Exactly 2**e in fp32 (the library's pow may be an ulp away)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise_pages(x, codes):
    """Codes and power-of-two scales of pages x [N, H, page, D]."""
    amax = x.abs().amax((2, 3))
    m, e = torch.frexp(amax / _QMAX[codes])
    e = torch.where(m == 0.5, e - 1, e).clamp(-60, 60)
    s = _power(e)
    y = x / s[:, :, None, None]
    y = y.to(torch.float8_e4m3fn) if codes == "e4m3" else y.round().to(torch.int8)
    return y, s


def prepare(case, seed):
    c = case
    g = torch.Generator(device=_DEV).manual_seed(seed)
    rng = random.Random(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=_DEV)

    if c["op"] == "logits":
        b, v, h = c["requests"], c["vocab"], c["history"]
        lens = [h if i % 4 == 0 else max(1, int(h * rng.uniform(0.125, 1.0))) for i in range(b)]
        prompts = [int(n * rng.uniform(0.0, 1.0)) for n in lens]
        # token frequencies fall off as in text: many repeats of few tokens
        u = torch.rand(b, h, generator=g, device=_DEV)
        history = ((v ** u - 1) * (v / max(1, v - 1))).long().clamp(0, v - 1).to(torch.int32)
        s = {"case": c, "logits": (normal(b, v) * 3).to(torch.bfloat16 if c["half"] else torch.float32),
             "history": history, "lens": _ints(lens), "prompts": _ints(prompts),
             "repetition": 1.0 + 0.3 * torch.rand(b, generator=g, device=_DEV),
             "presence": 0.5 * torch.rand(b, generator=g, device=_DEV),
             "frequency": 0.2 * torch.rand(b, generator=g, device=_DEV),
             "bias_ids": None, "bias": None, "allowed": None}
        if c["bias"]:
            s["bias_ids"] = torch.stack([torch.randperm(v, generator=g, device=_DEV)[:c["bias"]]
                                         for _ in range(b)]).to(torch.int32)
            s["bias"] = normal(b, c["bias"]) * 2
        if c["mask"]:
            s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (b, (v + 31) // 32), generator=g,
                                         device=_DEV).to(torch.int32)
        return s

    contexts, news = _lens(c)
    page, n = c["page"], c["requests"]
    used = [(a + b + page - 1) // page for a, b in zip(contexts, news)]
    width, total = max(used) + 1, sum(used)
    order = list(range(total + 8))
    rng.shuffle(order)
    if c["op"] == "plan":
        tables = [[-1] * width for _ in range(n)]
        at = 0
        for b in range(n):
            k = (contexts[b] + page - 1) // page
            tables[b][:k] = order[at:at + k]
            at += k
        free = order[at:] + [0] * at
        return {"case": c, "context": _ints(contexts), "new": _ints(news), "tables": _ints(tables),
                "free": _ints(free), "count": _ints([len(order) - at]), "tokens": sum(news)}

    tables = [[-1] * width for _ in range(n)]
    at = 0
    for b in range(n):
        tables[b][:used[b]] = order[at:at + used[b]]
        at += used[b]
    starts, kv, _, _, touched = _plan_host(contexts, news, tables, page)
    hkv, d, pages = c["kv_heads"], c["dim"], len(order)
    s = {"case": c, "tables": _ints(tables), "starts": _ints(starts), "kv": _ints(kv),
         "max_new": max(news)}
    for name in ("k", "v"):
        # keys have a few large channels, values do not; every page has its own level
        channel = 1.0 + 3.0 * (torch.rand(hkv, 1, d, generator=g, device=_DEV) < 0.06) * (name == "k")
        level = torch.exp(0.3 * normal(pages, hkv, 1, 1))
        s[name + "_pages"], s[name + "_scale"] = _quantise_pages(
            normal(pages, hkv, page, d) * channel * level, c["codes"])
    tokens = sum(news)
    if c["op"] == "append":
        # k and v are slices of one projection output, as the model gives them
        wide = normal(tokens, (c["q_heads"] + 2 * hkv) * d).to(torch.bfloat16)
        a = c["q_heads"] * d
        s["k"] = wide[:, a:a + hkv * d].view(tokens, hkv, d)
        s["v"] = wide[:, a + hkv * d:].view(tokens, hkv, d)
        s["touched"] = _ints(touched)
        # the touched pages up to their last token, which come back as values
        s["slots"] = _ints([p * page + i for p, _, off, cnt in touched for i in range(off + cnt)])
    else:
        s["q"] = normal(tokens, c["q_heads"], d).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------------- plain forms
def _plain_plan(s):
    page, tables = s["case"]["page"], s["tables"]
    ctx, new, tokens = s["context"].long(), s["new"].long(), s["tokens"]
    n = ctx.numel()
    dev = ctx.device
    ends = new.cumsum(0)
    starts = ends - new
    kv = ctx + new
    old = (ctx + page - 1) // page
    take = (kv + page - 1) // page - old
    first = take.cumsum(0) - take
    col = torch.arange(tables.shape[1], device=dev)[None]
    fresh = (col >= old[:, None]) & (col < (old + take)[:, None])
    pick = s["count"].long() - 1 - (first[:, None] + col - old[:, None])
    tables = torch.where(fresh, s["free"].long()[pick.clamp(0, s["free"].numel() - 1)], tables.long())
    rows = torch.arange(tokens, device=dev)
    req = torch.searchsorted(ends, rows, right=True)
    pos = ctx[req] + rows - starts[req]
    slots = tables[req, pos // page] * page + pos % page
    # touched pages: one entry for each (request, page) that gets tokens
    lead = ctx // page
    per = torch.where(new > 0, (kv - 1) // page - lead + 1, 0)
    tends = per.cumsum(0)
    room = min(tokens, tokens // page + 2 * n)
    u = torch.arange(room, device=dev)
    ureq = torch.searchsorted(tends, u, right=True)
    live = ureq < n
    r = ureq.clamp(max=n - 1)
    lp = (lead[r] + u - (tends - per)[r]).clamp(max=tables.shape[1] - 1)
    a = torch.maximum(lp * page, ctx[r])
    b = torch.minimum((lp + 1) * page, kv[r])
    touched = torch.stack([tables[r, lp], starts[r] + a - ctx[r], a - lp * page, b - a], 1)
    touched = torch.where(live[:, None], touched, torch.tensor([-1, 0, 0, 0], device=dev))
    i = torch.int32
    return {"q_starts": torch.cat([starts, ends[-1:]]).to(i), "kv_lens": kv.to(i),
            "positions": pos.to(i), "slots": slots.to(i), "touched": touched.to(i),
            "tables": tables.to(i), "free_count": (s["count"] - take.sum()).to(i)}


def _plain_values(codes, scale):
    return codes.float() * scale[..., None, None]


def _plain_append(s):
    c = s["case"]
    page, qmax = c["page"], _QMAX[c["codes"]]
    at, row, off, cnt = s["touched"].long().unbind(1)
    i = torch.arange(page, device=at.device)[None]
    is_new = (i >= off[:, None]) & (i < (off + cnt)[:, None])
    src = (row[:, None] + i - off[:, None]).clamp(0, s["k"].shape[0] - 1)
    is_old = (i < off[:, None])[:, None, :, None]
    keep = (i >= (off + cnt)[:, None])[:, None, :, None]
    out = {}
    slots = s["slots"].long()
    for name in ("k", "v"):
        pages, scale = s[name + "_pages"], s[name + "_scale"]
        x = s[name][src].float().transpose(1, 2) * is_new[:, None, :, None]    # [U, H, page, D]
        amax = x.abs().amax((2, 3))
        m, e = torch.frexp(amax / qmax)
        e = torch.where(m == 0.5, e - 1, e).clamp(-60, 60)
        grown = _power(e)
        before = scale[at]
        now = torch.where(off[:, None] > 0, torch.maximum(before, grown), grown)
        codes = pages.view(torch.uint8)[at].view(pages.dtype)
        old = torch.where(is_old, codes.float() * (before / now)[:, :, None, None], 0.0)
        y = torch.where(is_old, old, x / now[:, :, None, None]).clamp(-qmax, qmax)
        y = y.to(pages.dtype) if c["codes"] == "e4m3" else y.round().to(pages.dtype)
        pages.view(torch.uint8)[at] = torch.where(keep, codes.view(torch.uint8), y.view(torch.uint8))
        scale[at] = now
        got = pages.view(torch.uint8)[slots // page, :, slots % page].view(pages.dtype)
        out[name] = (got.float() * scale[slots // page][:, :, None]).to(torch.bfloat16)
        out[name + "_scale"] = scale
    return out


def _plain_attend(s):
    c = s["case"]
    q, starts, kv = s["q"].float(), s["starts"].long(), s["kv"].long()
    n, hkv, d = c["requests"], c["kv_heads"], c["dim"]
    group, most = c["q_heads"] // hkv, s["max_new"]
    tables = s["tables"].long().clamp(min=0)
    length = tables.shape[1] * c["page"]
    seen = (torch.arange(length, device=q.device) < kv[:, None])[:, None, :, None]

    def dense(name):
        pages = s[name + "_pages"]
        x = pages.view(torch.uint8)[tables].view(pages.dtype).float()
        x = x * s[name + "_scale"][tables][..., None, None]                # [B, P, H, page, D]
        return torch.where(seen, x.transpose(1, 2).reshape(n, hkv, length, d), 0.0)

    new = starts[1:] - starts[:-1]
    t = torch.arange(most, device=q.device)
    rows = (starts[:-1, None] + t).clamp(max=q.shape[0] - 1)               # [B, most]
    x = q[rows].view(n, most, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, most * group, d)
    p = (x @ dense("k").transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    limit = (kv - new)[:, None] + t + 1                                    # keys row t sees
    hidden = torch.arange(length, device=q.device) >= limit[:, :, None]
    p.masked_fill_(hidden.repeat_interleave(group, 1)[:, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = (p @ dense("v")) / p.sum(-1, keepdim=True)
    o = o.view(n, hkv, most, group, d).permute(0, 2, 1, 3, 4).reshape(n, most, c["q_heads"], d)
    return o[t < new[:, None]].to(torch.bfloat16)


def _plain_logits(s):
    z = s["logits"].float()
    b, v = z.shape
    h = s["history"].long()
    i = torch.arange(h.shape[1], device=z.device)[None]
    live = i < s["lens"][:, None]
    made = live & (i >= s["prompts"][:, None])
    seen = torch.zeros(b, v, device=z.device).scatter_add_(1, h, live.float()) > 0
    count = torch.zeros(b, v, device=z.device).scatter_add_(1, h, made.float())
    r = s["repetition"][:, None]
    z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
    z = z - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        z = z.scatter_add(1, s["bias_ids"].long(), s["bias"])
    if s["allowed"] is not None:
        j = torch.arange(v, device=z.device)
        z = torch.where(((s["allowed"][:, j // 32] >> (j % 32)) & 1) > 0, z, float("-inf"))
    return z


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend,
                "logits": _plain_logits}[op](s)
    from nano_megatron_b200.ops import serving

    if op == "plan":
        p = serving.plan_step(s["context"], s["new"], s["tables"], s["free"], s["count"],
                              page_size=s["case"]["page"], num_tokens=s["tokens"])
        return {"q_starts": p.q_starts, "kv_lens": p.kv_lens, "positions": p.positions,
                "slots": p.slots, "touched": p.touched, "tables": s["tables"],
                "free_count": p.free_count}
    if op == "logits":
        return serving.adjust_logits(
            s["logits"], s["history"], s["lens"], s["prompts"], repetition=s["repetition"],
            presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"],
            bias=s["bias"], allowed=s["allowed"])
    cache = serving.PagedKV(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if op == "append":
        serving.append_kv(cache, s["k"], s["v"], s["touched"])
        k, v = serving.read_kv(cache, s["slots"])
        return {"k": k, "k_scale": cache.k_scale, "v": v, "v_scale": cache.v_scale}
    return serving.paged_attention(s["q"], cache, s["tables"], s["starts"], s["kv"],
                                   max_new=s["max_new"])


# -------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "logits":
        b, v = c["requests"], c["vocab"]
        byte = b * v * ((2 if c["half"] else 4) + 4) + b * c["history"] * 0.65 * 4
        byte += b * (v // 8) * bool(c["mask"]) + b * c["bias"] * 8
        return {"bytes": byte, "flops": 6 * b * v}
    ctx, new = _lens(c)
    page, n, tokens = c["page"], len(ctx), sum(new)
    used = sum((a + b + page - 1) // page for a, b in zip(ctx, new))
    if c["op"] == "plan":
        touched = sum((a + b - 1) // page - a // page + 1 for a, b in zip(ctx, new))
        return {"bytes": 4 * (4 * n + 2 * tokens + 4 * touched + 2 * used), "flops": 4 * tokens}
    row = c["kv_heads"] * c["dim"]
    if c["op"] == "append":
        back = sum(b + a % page for a, b in zip(ctx, new))
        pages = sum((a + b - 1) // page - a // page + 1 for a, b in zip(ctx, new))
        return {"bytes": 2 * row * (3 * tokens + 3 * back) + pages * 2 * c["kv_heads"] * 8,
                "flops": 4 * row * tokens}
    keys = sum(a + b for a, b in zip(ctx, new))
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(ctx, new))
    return {"bytes": 2 * row * keys + 4 * tokens * c["q_heads"] * c["dim"]
            + used * (8 * c["kv_heads"] + 4),
            "flops": 4 * c["dim"] * c["q_heads"] * pairs}


# ------------------------------------------------------------------- results in 64 bits
def _decode_table(codes):
    """Value of each of the 256 bytes, from the format's definition."""
    if codes == "int8":
        return [float(i if i < 128 else i - 256) for i in range(256)]
    table = []
    for i in range(256):
        sign, e, m = -1.0 if i & 128 else 1.0, (i >> 3) & 15, i & 7
        v = math.nan if (e, m) == (15, 7) else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        table.append(sign * v)
    return table


def _power64(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None
    s = prepare(case, seed)
    f64 = torch.float64
    if c["op"] == "logits":
        out = s["logits"].to(f64)
        for b in range(c["requests"]):
            h = s["history"][b, :int(s["lens"][b])].long()
            z = out[b]
            r = s["repetition"][b].to(f64)
            ids = h.unique()
            z[ids] = torch.where(z[ids] > 0, z[ids] / r, z[ids] * r)
            ids, cnt = h[int(s["prompts"][b]):].unique(return_counts=True)
            z[ids] -= s["frequency"][b].to(f64) * cnt + s["presence"][b].to(f64)
            if c["bias"]:
                z[s["bias_ids"][b].long()] += s["bias"][b].to(f64)
            if c["mask"]:
                bits = (s["allowed"][b].long()[:, None] >> torch.arange(32, device=z.device)) & 1
                z[bits.reshape(-1)[:c["vocab"]] == 0] = -math.inf
        return out
    page = c["page"]
    table = torch.tensor(_decode_table(c["codes"]), dtype=f64, device=_DEV)
    if c["op"] == "append":
        out = {}
        at, row, off, cnt = (x.tolist() for x in s["touched"].unbind(1))
        if len(at) > 4000:
            return None
        for name in ("k", "v"):
            scale, pages, values = s[name + "_scale"].to(f64).clone(), s[name + "_pages"].view(torch.uint8), []
            for p, r, o, m in zip(at, row, off, cnt):
                x = s[name][r:r + m].to(f64).transpose(0, 1)                       # [H, m, D]
                top = x.abs().amax((1, 2))
                e = torch.ceil(torch.log2(top / _QMAX[c["codes"]])).clamp(-60, 60)
                now = _power64(e)
                if o:
                    now = torch.maximum(now, scale[p])
                    x = torch.cat([table[pages[p, :, :o].long()] * scale[p][:, None, None], x], 1)
                y = x / now[:, None, None]
                if c["codes"] == "int8":
                    y = y.round()
                else:    # nearest multiple of the spacing of e4m3 at that size, ties to even
                    step = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3
                    step = _power64(step)
                    y = (y / step).round() * step
                values.append((y * now[:, None, None]).transpose(0, 1))
                scale[p] = now
            out[name], out[name + "_scale"] = torch.cat(values), scale
        return out
    q, group = s["q"].to(f64), c["q_heads"] // c["kv_heads"]
    out = torch.empty_like(q)
    starts = s["starts"].tolist()
    for b in range(c["requests"]):
        n, r0, r1 = int(s["kv"][b]), starts[b], starts[b + 1]
        ids = s["tables"][b, :(n + page - 1) // page].long()
        limit = n - (r1 - r0) + 1 + torch.arange(r1 - r0, device=_DEV)
        for h in range(c["kv_heads"]):
            k, v = ((table[s[x + "_pages"].view(torch.uint8)[ids, h].long()]
                     * s[x + "_scale"][ids, h].to(f64)[:, None, None]).reshape(-1, c["dim"])[:n]
                    for x in ("k", "v"))
            for j in range(h * group, (h + 1) * group):
                z = q[r0:r1, j] @ k.T / math.sqrt(c["dim"])
                z.masked_fill_(torch.arange(n, device=_DEV)[None] >= limit[:, None], -math.inf)
                out[r0:r1, j] = torch.softmax(z, -1) @ v
    return out
