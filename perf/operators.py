"""What the exact paged serving step is measured on: block tables and slot maps, the norm and rotation of queries and
keys with their cache write, attention of one new token over a paged cache, and attention of prompt chunks over it."""

import math
import random

import torch

own = False

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = {"f32": F32, "f16": F16, "bf16": BF16}
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step's bookkeeping for the 64-request paged serving batch: one new token each, two requests ended
        dict(name="tables_decode", op="tables", batch=64, ending=2, ctx_lo=1024, ctx_hi=65536, new_lo=1, new_hi=1, block=16, short=False),
        # a mixed step of a busy server: decodes beside prompt chunks of up to 2K tokens, a pool that runs out near the end
        dict(name="tables_mixed", op="tables", batch=1001, ending=37, ctx_lo=1, ctx_hi=8192, new_lo=1, new_hi=2048, block=16, short=True),
        # one decode step of 16 requests: 28/4 heads, normed queries and keys, rows written to the cache
        dict(name="rope_decode", op="rope", tokens=16, hq=28, hkv=4, dim=128, rotary=128, interleaved=False, norm=True, cache=True, dtype="bf16"),
        # a prompt of 8192 tokens at 32/8 heads, normed, half layout, written to the cache
        dict(name="rope_prompt", op="rope", tokens=8192, hq=32, hkv=8, dim=128, rotary=128, interleaved=False, norm=True, cache=True, dtype="bf16"),
        # a ragged step whose model rotates half of each head in the interleaved layout and norms nothing; keys go on to the codec
        dict(name="rope_part", op="rope", tokens=4099, hq=32, hkv=8, dim=128, rotary=64, interleaved=True, norm=False, cache=False, dtype="f16"),
        # one user's chat turn: a single request of 1001 tokens
        dict(name="decode_one", op="decode", batch=1, lo=1001, hi=1001, hq=32, hkv=8, dim=128, block=16, window=0, cap=0.0, slopes=False, dtype="bf16"),
        # the paged serving batch: 64 requests of 1K to 64K tokens at 28/4 heads
        dict(name="decode_paged", op="decode", batch=64, lo=1024, hi=65536, hq=28, hkv=4, dim=128, block=16, window=0, cap=0.0, slopes=False, dtype="bf16"),
        # long contexts at 64/8 heads with capped scores
        dict(name="decode_long_cap", op="decode", batch=4, lo=131072, hi=131072, hq=64, hkv=8, dim=128, block=16, window=0, cap=30.0, slopes=False, dtype="f16"),
        # a windowed layer with a distance bias, 32-bit cache, heads of 64, ragged lengths
        dict(name="decode_window_f32", op="decode", batch=33, lo=100, hi=32768, hq=12, hkv=4, dim=64, block=32, window=4096, cap=0.0, slopes=True, dtype="f32"),
        # a ragged batch of short prompts
        dict(name="prefill_short", op="prefill", batch=9, new_lo=1, new_hi=301, ctx_lo=0, ctx_hi=0, hq=28, hkv=4, dim=128, block=16, window=0, prefix=0, cap=0.0, slopes=False, dtype="bf16"),
        # one long prompt at 32/8 heads
        dict(name="prefill_long", op="prefill", batch=1, new_lo=8192, new_hi=8192, ctx_lo=0, ctx_hi=0, hq=32, hkv=8, dim=128, block=16, window=0, prefix=0, cap=0.0, slopes=False, dtype="bf16"),
        # chunks behind cached context, a prefix all rows see, a window and capped scores
        dict(name="prefill_chunk", op="prefill", batch=4, new_lo=501, new_hi=1024, ctx_lo=2000, ctx_hi=8000, hq=64, hkv=8, dim=128, block=16, window=4096, prefix=256, cap=30.0, slopes=False, dtype="f16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def span(lo, hi):
        a, b = log(lo, hi), log(lo, hi)
        return min(a, b), max(a, b)

    op = rng.choice(["tables", "rope", "decode", "prefill"])
    heads = [(32, 8), (28, 4), (64, 8), (12, 4), (16, 16), (8, 1)]
    while True:
        if op == "tables":
            (clo, chi), (nlo, nhi) = span(1, 65536), span(1, 2048)
            n = log(1, 1500)
            c = dict(op=op, batch=n, ending=rng.choice([0, n // 20, n // 4]), ctx_lo=clo, ctx_hi=chi, new_lo=nlo, new_hi=nhi, block=rng.choice([8, 16, 24, 64, 128]), short=rng.random() < 0.3)
            if work(c)["bytes"] <= work(listed()[1])["bytes"]:
                return c
        elif op == "rope":
            (hq, hkv), dim = rng.choice(heads), rng.choice([64, 128, 256])
            c = dict(op=op, tokens=log(1, 16384), hq=hq, hkv=hkv, dim=dim, rotary=dim // rng.choice([1, 1, 2, 4]), interleaved=rng.random() < 0.4,
                     norm=rng.random() < 0.6, cache=rng.random() < 0.6, dtype=rng.choice(["bf16", "f16", "f32"]))
            if work(c)["bytes"] <= work(listed()[3])["bytes"]:
                return c
        elif op == "decode":
            (hq, hkv), (lo, hi) = rng.choice(heads), span(1, 131072)
            c = dict(op=op, batch=log(1, 128), lo=lo, hi=hi, hq=hq, hkv=hkv, dim=rng.choice([64, 128, 128, 256]), block=rng.choice([8, 16, 24, 64, 128]),
                     window=rng.choice([0, 0, log(16, 8192)]), cap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
            if work(c)["bytes"] <= work(listed()[7])["bytes"] and c["batch"] * hi * hkv * c["dim"] <= 1 << 30:
                return c
        else:
            (hq, hkv), (nlo, nhi), (clo, chi) = rng.choice(heads), span(1, 8192), span(1, 16384)
            if rng.random() < 0.5:
                clo = chi = 0
            c = dict(op=op, batch=log(1, 16), new_lo=nlo, new_hi=nhi, ctx_lo=clo, ctx_hi=chi, hq=hq, hkv=hkv, dim=rng.choice([64, 128, 128, 256]), block=rng.choice([8, 16, 24, 64, 128]),
                     window=rng.choice([0, 0, log(64, 8192)]), prefix=rng.choice([0, 0, log(1, 512)]), cap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.3, dtype=rng.choice(["bf16", "f16"]))
            if work(c)["flops"] <= work(listed()[10])["flops"] and c["batch"] * hq * nhi * (nhi + chi) <= 1 << 31:
                return c


def spread(count, lo, hi, salt=0):
    """`count` lengths from lo to hi, even over their logarithm, in an order of the case's own."""
    got = [lo if lo == hi else int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** ((i + 0.5) / count))) - 1 for i in range(count)]
    got = [min(hi, max(lo, x)) for x in got]
    random.Random(1000 * count + salt).shuffle(got)
    return got


def rows_of(c):
    """(context, new tokens) of each request of a tables or prefill case; a tables case's first `ending` requests have ended."""
    rows = list(zip(spread(c["batch"], c["ctx_lo"], c["ctx_hi"]), spread(c["batch"], c["new_lo"], c["new_hi"], 1)))
    return [(x, 0 if i < c.get("ending", 0) else n) for i, (x, n) in enumerate(rows)]


def blocks_for(n, block):
    return -(-n // block)


def pairs(c, n, ctx):
    """Visible (row, token) pairs of a request with n new tokens behind ctx cached ones."""
    L, p, w = ctx + n, min(c["prefix"], ctx + n), c["window"]
    total = 0
    for i in range(ctx, L):
        lo = max(0, i - w + 1) if w else 0
        total += p + max(0, i + 1 - max(lo, p))
    return total


def work(c):
    if c["op"] == "tables":
        rows = rows_of(c)
        total = sum(n for _, n in rows)
        blocks = sum(blocks_for(x + n, c["block"]) - (x // c["block"] if n else 0) for x, n in rows)
        return {"bytes": 12.0 * total + 8.0 * blocks + 18.0 * len(rows), "flops": 0.0}
    size = DTYPES[c["dtype"]].itemsize
    if c["op"] == "rope":
        T, heads = c["tokens"], c["hq"] + (2 if c["cache"] else 1) * c["hkv"]
        flops = T * (c["hq"] + c["hkv"]) * (3.0 * c["rotary"] + (4.0 * c["dim"] if c["norm"] else 0.0))
        return {"bytes": 2.0 * T * heads * c["dim"] * size + T * (4.0 * c["rotary"] + 12.0), "flops": flops}
    if c["op"] == "decode":
        seen = sum(min(n, c["window"]) if c["window"] else n for n in spread(c["batch"], c["lo"], c["hi"]))
        return {"bytes": 2.0 * seen * c["hkv"] * c["dim"] * size + 2.0 * c["batch"] * c["hq"] * c["dim"] * size, "flops": 4.0 * seen * c["hq"] * c["dim"]}
    rows = rows_of(c)
    seen = sum(pairs(c, n, x) for x, n in rows)
    held = sum(min(x + n, n + c["window"] + c["prefix"]) if c["window"] else x + n for x, n in rows)
    return {"bytes": 2.0 * held * c["hkv"] * c["dim"] * size + 2.0 * sum(n for _, n in rows) * c["hq"] * c["dim"] * size, "flops": 4.0 * seen * c["hq"] * c["dim"]}


# ------------------------------------------------------------------ inputs
def cached(c, lens, gen, dtype):
    """A paged cache of requests of these lengths: (k_cache, v_cache, block_table). Pages are handed out in a random order; the
    slots behind a request's last token hold what memory held before (NaN here)."""
    b = c["block"]
    need = [blocks_for(n, b) for n in lens]
    total, width = sum(need), max(1, max(need))
    order = torch.randperm(total + 3, generator=gen, device=DEV, dtype=torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device=DEV)
    counts = torch.tensor(need, device=DEV)
    table[torch.arange(width, device=DEV)[None, :] < counts[:, None]] = order[:total]
    shape = (total + 3, b, c["hkv"], c["dim"])
    # keys carry a spectrum over the head's channels, as trained ones do; values are plain
    spectrum = torch.linspace(1.8, 0.4, c["dim"], device=DEV)
    k = (torch.randn(shape, generator=gen, device=DEV, dtype=F32 if dtype == F32 else BF16) * spectrum).to(dtype)
    v = torch.randn(shape, generator=gen, device=DEV, dtype=F32 if dtype == F32 else BF16).to(dtype)
    ends = [(i, n) for i, n in enumerate(lens) if n % b]
    if ends:
        page = table[[i for i, _ in ends], [n // b for _, n in ends]].long()
        past = torch.arange(b, device=DEV)[None, :] >= torch.tensor([n % b for _, n in ends], device=DEV)[:, None]
        at = (page[:, None].expand(-1, b)[past], torch.arange(b, device=DEV)[None, :].expand(len(ends), -1)[past])
        k[at], v[at] = float("nan"), float("nan")
    return k, v, table


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def prepare(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c}
    if c["op"] == "tables":
        rows = [(x, n, i < c["ending"]) for i, (x, n) in enumerate(rows_of(c))]
        random.Random(seed).shuffle(rows)
        ended, rows = [e for _, _, e in rows], [(x, n) for x, n, _ in rows]
        b = c["block"]
        held = [blocks_for(x, b) for x, _ in rows]
        need = [blocks_for(x + n, b) - h for (x, n), h in zip(rows, held)]
        back = sum(h for h, e in zip(held, ended) if e)
        width = max(blocks_for(x + n, b) for x, n in rows)
        free = max(1, int(0.8 * sum(need)) - back) if c["short"] else sum(need) + 7
        order = torch.randperm(sum(held) + free, generator=gen, device=DEV, dtype=torch.int32)
        table = torch.zeros(len(rows), width, dtype=torch.int32, device=DEV)
        table[torch.arange(width, device=DEV)[None, :] < ints(held)[:, None]] = order[free:]
        s.update(context=ints([x for x, _ in rows]), new=ints([n for _, n in rows]), table=table, free_blocks=torch.cat([order[:free], torch.full_like(order[free:], -1)]), free_count=ints([free]),
                 ended=torch.tensor(ended, device=DEV) if c["ending"] else None, tokens=sum(n for _, n in rows))
        return s
    dtype = DTYPES[c["dtype"]]
    if c["op"] == "rope":
        T, hq, hkv, D, R = c["tokens"], c["hq"], c["hkv"], c["dim"], c["rotary"]
        qkv = (torch.randn(T, hq + 2 * hkv, D, generator=gen, device=DEV) * torch.linspace(2.0, 0.3, D, device=DEV)).to(dtype)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        longest = 32768
        s["positions"] = torch.randint(0, longest, (T,), generator=gen, device=DEV, dtype=torch.int32)
        angle = torch.arange(longest, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
        s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).to(F32)
        s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(2, D, generator=gen, device=DEV)).unbind(0)) if c["norm"] else (None, None)
        if c["cache"]:
            pages = blocks_for(T, 16) + 1
            s["k_cache"], s["v_cache"] = torch.zeros(2, pages, 16, hkv, D, dtype=dtype, device=DEV).unbind(0)
            s["slots"] = torch.randperm(pages * 16, generator=gen, device=DEV)[:T]
        return s
    s["slopes"] = (2.0 ** (-8.0 * (torch.arange(c["hq"], device=DEV, dtype=F32) + 1) / c["hq"])) if c["slopes"] else None
    if c["op"] == "decode":
        lens = spread(c["batch"], c["lo"], c["hi"])
        news = [1] * len(lens)
    else:
        rows = rows_of(c)
        lens, news = [x + n for x, n in rows], [n for _, n in rows]
        s["cu"] = ints([sum(news[:i]) for i in range(len(news) + 1)])
        s["prefix"] = ints([min(c["prefix"], n) for n in lens]) if c["prefix"] else None
    s["k_cache"], s["v_cache"], s["table"] = cached(c, lens, gen, dtype)
    s["lens"] = ints(lens)
    s["longest"], s["most"] = max(lens), max(news)  # what the plain form pads to
    s["q"] = torch.randn(sum(news), c["hq"], c["dim"], generator=gen, device=DEV).to(dtype)
    return s


# ------------------------------------------------------------------ the calls
def run(s):
    return (run_own if own else run_plain)(s)


def run_own(s):
    from smaq_b200 import ops
    c = s["case"]
    if c["op"] == "tables":
        t = ops.step_tables(s["free_blocks"], s["free_count"], s["context"], s["new"], s["table"], block_size=c["block"], num_tokens=s["tokens"], finished=s["ended"])
        return {"pool": s["free_blocks"], "cu": t.cu_query, "lens": t.seq_lens, "positions": t.positions, "slots": t.slots, "free": t.free_count, "admitted": t.admitted, "table": s["table"]}
    if c["op"] == "rope":
        more = dict(v=s["v"], k_cache=s["k_cache"], v_cache=s["v_cache"], slots=s["slots"]) if c["cache"] else {}
        q, k = ops.norm_rope(s["q"], s["k"], s["positions"], s["rope"], q_weight=s["wq"], k_weight=s["wk"], eps=1e-6, interleaved=c["interleaved"], **more)
        return {"q": q, "k": s["k_cache"], "v": s["v_cache"]} if c["cache"] else {"q": q, "k": k}
    more = dict(window=c["window"] or None, softcap=c["cap"] or None, slopes=s["slopes"])
    if c["op"] == "decode":
        return ops.paged_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], **more)
    return ops.paged_prefill(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"], prefix_lens=s["prefix"], **more)


def run_plain(s):
    return {"tables": plain_tables, "rope": plain_rope, "decode": plain_attention, "prefill": plain_attention}[s["case"]["op"]](s)


def plain_tables(s):
    c, ctx, new, table, pool = s["case"], s["context"], s["new"], s["table"], s["free_blocks"]
    b, (B, M) = c["block"], s["table"].shape
    ended = torch.zeros_like(new, dtype=torch.bool) if s["ended"] is None else s["ended"]
    start = (ctx + b - 1) // b
    # the stack of free blocks, with the ended requests' blocks on top
    back = torch.where(ended, start, torch.zeros_like(start)).cumsum(0, dtype=torch.int32)
    F = s["free_count"]
    at = torch.arange(pool.numel(), device=DEV, dtype=torch.int32)
    giver = torch.searchsorted(back, (at - F).clamp(min=0), right=True).clamp(max=B - 1)
    nth = (at - F - back[giver] + start[giver]).clamp(min=0, max=M - 1)
    stack = torch.where(at < F, pool, table[giver, nth.long()])
    top = F + back[-1:]
    # what each running request needs, in the requests' order while the stack lasts
    new = torch.where(ended, torch.zeros_like(new), new)
    end = (ctx + new + b - 1) // b
    fits = (end <= M) & ~ended
    need = torch.where(fits & (new > 0), end - start, torch.zeros_like(end))
    upto = need.cumsum(0, dtype=torch.int32)
    admitted = fits & ((need == 0) | (upto <= top))
    left = top - torch.where(admitted & (need > 0), upto, torch.zeros_like(upto)).amax(0, keepdim=True)
    col = torch.arange(M, device=DEV, dtype=torch.int32)[None, :]
    fresh = admitted[:, None] & (col >= start[:, None]) & (col < end[:, None]) & (need > 0)[:, None]
    take = top - 1 - (upto - need)[:, None] - (col - start[:, None])
    table.copy_(torch.where(fresh, stack[take.clamp(min=0, max=pool.numel() - 1).long()], table))
    pool.copy_(torch.where((at >= F) & (at < left), stack, pool))
    cu = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0, dtype=torch.int32)])
    t = torch.arange(s["tokens"], device=DEV, dtype=torch.int32)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=B - 1)
    pos = ctx[r] + t - cu[r]
    page = table[r, (pos // b).clamp(max=M - 1).long()].long()
    slots = torch.where(admitted[r], page * b + pos % b, torch.full_like(page, -1))
    lens = torch.where(admitted, ctx + new, torch.zeros_like(ctx))
    return {"pool": pool, "cu": cu, "lens": lens, "positions": pos, "slots": slots, "free": left, "admitted": admitted, "table": table}


def plain_rope(s):
    c = s["case"]
    R, half = c["rotary"], c["rotary"] // 2
    row = s["rope"][s["positions"].long()][:, None, :]
    cos, sin = row[..., :half], row[..., half:]

    def turned(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w
        a, b = (y[..., 0:R:2], y[..., 1:R:2]) if c["interleaved"] else (y[..., :half], y[..., half:R])
        p = (a * cos - b * sin, b * cos + a * sin)
        p = torch.stack(p, -1).flatten(-2) if c["interleaved"] else torch.cat(p, -1)
        return torch.cat([p, y[..., R:]], -1).to(x.dtype)

    q, k = turned(s["q"], s["wq"]), turned(s["k"], s["wk"])
    if not c["cache"]:
        return {"q": q, "k": k}
    s["k_cache"].view(-1, c["hkv"], c["dim"])[s["slots"]] = k
    s["v_cache"].view(-1, c["hkv"], c["dim"])[s["slots"]] = s["v"]
    return {"q": q, "k": s["k_cache"], "v": s["v_cache"]}


def plain_attention(s):
    c = s["case"]
    B, L, N, b, G = c["batch"], s["longest"], s["most"], c["block"], c["hq"] // c["hkv"]
    j = torch.arange(L, device=DEV)
    held = j[None, :] < s["lens"][:, None]
    at = s["table"].long()[:, j // b] * b + j % b
    k, v = (torch.where(held[:, :, None, None], x.view(-1, c["hkv"], c["dim"])[at], torch.zeros((), dtype=x.dtype, device=DEV)).float().permute(0, 2, 1, 3) for x in (s["k_cache"], s["v_cache"]))
    n = s["cu"].diff() if "cu" in s else torch.ones_like(s["lens"])
    first = s["cu"][:-1] if "cu" in s else torch.arange(B, device=DEV)
    r = torch.arange(N, device=DEV)
    mine = (first[:, None] + torch.minimum(r[None, :], n[:, None] - 1)).long()
    q = s["q"][mine].float().view(B, N, c["hkv"], G, c["dim"]).permute(0, 2, 3, 1, 4).reshape(B, c["hkv"], G * N, c["dim"])
    x = (q @ k.transpose(-1, -2) * (1.0 / math.sqrt(c["dim"]))).view(B, c["hkv"], G, N, L)
    if c["cap"]:
        x = torch.tanh(x.div_(c["cap"])).mul_(c["cap"])
    i = s["lens"][:, None] - n[:, None] + r[None, :]
    gap = (i[:, :, None] - j[None, None, :])[:, None, None]
    if s["slopes"] is not None:
        x.sub_(s["slopes"].view(1, c["hkv"], G, 1, 1) * gap.abs())
    seen = gap >= 0
    if c["window"]:
        seen = seen & (gap < c["window"])
    if s.get("prefix") is not None:
        seen = seen | (j[None, :] < s["prefix"][:, None])[:, None, None, None, :]
    x.masked_fill_(~(seen & held[:, None, None, None, :]), float("-inf"))
    x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    out = (x.view(B, c["hkv"], G * N, L) @ v).view(B, c["hkv"], G, N, c["dim"]) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4).reshape(B, N, c["hq"], c["dim"])
    if "cu" not in s:
        return out[:, 0].to(s["q"].dtype)
    t = torch.arange(s["q"].shape[0], device=DEV)
    row = torch.searchsorted(s["cu"][1:].contiguous(), t.int(), right=True)
    return out[row, t - s["cu"][row]].to(s["q"].dtype)


# ------------------------------------------------------------------ 64 bits
def exact(c, seed):
    if c["op"] == "tables":
        return None
    s = prepare(c, seed)
    if c["op"] == "rope":
        return exact_rope(c, s)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lens = s["lens"].tolist()
    cu = s["cu"].tolist() if "cu" in s else list(range(len(lens) + 1))
    G, b = c["hq"] // c["hkv"], c["block"]
    for e, L in enumerate(lens):
        pages = s["table"][e, :blocks_for(L, b)].long()
        for h in range(c["hkv"]):
            K = s["k_cache"][pages, :, h].reshape(-1, c["dim"])[:L].double()
            V = s["v_cache"][pages, :, h].reshape(-1, c["dim"])[:L].double()
            step = max(1, (1 << 26) // max(1, G * L))
            for r0 in range(cu[e], cu[e + 1], step):
                r1 = min(cu[e + 1], r0 + step)
                z = torch.einsum("tgd,jd->tgj", s["q"][r0:r1, h * G:(h + 1) * G].double(), K) / math.sqrt(c["dim"])
                if c["cap"]:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                i = torch.arange(L - (cu[e + 1] - r0), L - (cu[e + 1] - r1), device=DEV)[:, None, None]
                j = torch.arange(L, device=DEV)[None, None, :]
                if s["slopes"] is not None:
                    z = z - s["slopes"][h * G:(h + 1) * G].double()[None, :, None] * (i - j).abs()
                ok = j <= i
                if c["window"]:
                    ok = ok & (j > i - c["window"])
                if s.get("prefix") is not None:
                    ok = ok | (j < int(s["prefix"][e]))
                out[r0:r1, h * G:(h + 1) * G] = torch.softmax(z.masked_fill(~ok, float("-inf")), -1) @ V
    return out


def exact_rope(c, s):
    R = c["rotary"]
    at = s["positions"].long()
    turn = torch.complex(s["rope"][at, :R // 2].double(), s["rope"][at, R // 2:].double())[:, None, :]

    def go(x, w):
        y = x.double()
        if w is not None:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        y = y.clone()
        if c["interleaved"]:
            z = torch.view_as_complex(y[..., :R].reshape(*y.shape[:-1], R // 2, 2).contiguous()) * turn
            y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
        else:
            z = torch.complex(y[..., :R // 2].contiguous(), y[..., R // 2:R].contiguous()) * turn
            y[..., :R // 2], y[..., R // 2:R] = z.real, z.imag
        return y

    q, k = go(s["q"], s["wq"]), go(s["k"], s["wk"])
    if not c["cache"]:
        return {"q": q, "k": k}
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    page, off = s["slots"] // 16, s["slots"] % 16
    kc[page, off], vc[page, off] = k, s["v"].double()
    return {"q": q, "k": kc, "v": vc}
