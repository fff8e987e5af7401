"""Plain restatements of the exact paged step in 64 bits, and random cases for its tests."""

import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half an ulp of 1
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def paged_case(dev, lens, Hkv, D, page, dtype, seed=0, fill=float("nan"), spare=2):
    """K and V caches with the requests' tokens on shuffled pages; every other slot holds ``fill``."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g).tolist()
    M = max(need + [1]) + 1
    table = torch.zeros(len(lens), M, dtype=torch.int32)
    k = torch.full((P, page, Hkv, D), fill)
    v = torch.full((P, page, Hkv, D), fill)
    at = 0
    for b, n in enumerate(lens):
        pages = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = torch.tensor(pages, dtype=torch.int32)
        for i, pg in enumerate(pages):
            m = min(page, n - i * page)
            k[pg, :m] = torch.randn(m, Hkv, D, generator=g) * 1.3
            v[pg, :m] = torch.randn(m, Hkv, D, generator=g)
    return k.to(dev, dtype), v.to(dev, dtype), table.to(dev)


def attention64(q, k, v, table, lens, cu, *, scale=None, window=None, softcap=None, slopes=None, prefix=None):
    """(out, lse, bound) in 64 bits; ``bound(u_p)`` is the elementwise error that weights rounded by
    ``u_p`` and 32-bit scores allow (before the output's own rounding)."""
    T, Hq, D = q.shape
    page, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    mass, eps = torch.zeros_like(out), torch.zeros(T, Hq, 1, dtype=torch.float64, device=q.device)
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if L == 0 or n == 0:
            continue
        pages = table[b, :-(-L // page)].long()
        K = k[pages].reshape(-1, Hkv, D)[:L].double().repeat_interleave(G, 1)
        V = v[pages].reshape(-1, Hkv, D)[:L].double().repeat_interleave(G, 1)
        Q = q[cu[b]:cu[b + 1]].double()
        i = (L - n + torch.arange(n, device=q.device))[:, None]
        j = torch.arange(L, device=q.device)[None]
        see = j <= i
        if window:
            see &= j > i - window
        if prefix is not None:
            see |= j < prefix[b]
        x = torch.einsum("thd,jhd->htj", Q, K) * scale
        size = torch.einsum("thd,jhd->htj", Q.abs(), K.nan_to_num(0, 0, 0).abs()) * abs(scale)
        if softcap:
            x = softcap * torch.tanh(x / softcap)
            size = size + 8 * softcap
        if slopes is not None:
            x = x - slopes.double()[:, None, None] * (i - j).abs()
            size = size + (slopes.double()[:, None, None] * (i - j).abs()).masked_fill(~see, 0)
        x = x.masked_fill(~see, -math.inf)
        big = x.amax(-1, keepdim=True)
        w = torch.exp(x - torch.where(big == -math.inf, torch.zeros_like(big), big))
        s = w.sum(-1, keepdim=True)
        w = torch.where(s > 0, w / s, torch.zeros_like(w))
        Vz = torch.where(torch.isfinite(V), V, torch.zeros_like(V))
        o = torch.einsum("htj,jhd->thd", w, Vz)
        bad = (see[:, :, None, None] & ~torch.isfinite(V)[None]).any(1)        # [t, h, d]
        out[cu[b]:cu[b + 1]] = torch.where(bad, torch.full_like(o, math.nan), o)
        lse[cu[b]:cu[b + 1]] = (big + s.log()).squeeze(-1).transpose(0, 1)
        mass[cu[b]:cu[b + 1]] = torch.einsum("htj,jhd->thd", w, Vz.abs())
        eps[cu[b]:cu[b + 1]] = (size.masked_fill(~see, 0).amax(-1) * 2.0 ** -24 * (D / 8 + 16)).transpose(0, 1)[..., None]
    return out, lse, lambda u_p: (u_p + 2 * eps + 2.0 ** -20) * mass


def check_attention(got, ref, bound, dtype, u_p):
    """Every element within the output's rounding of the 64-bit value plus ``bound(u_p)``; NaN where it is NaN."""
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), "NaN in other places"
    ok = ~torch.isnan(ref)
    tol = UNIT[dtype] * ref.abs() + bound(u_p) * (1 + UNIT[dtype]) + TINY[dtype]
    over = ((g - ref).abs() - tol)[ok]
    assert over.numel() == 0 or float(over.max()) <= 0, float(((g - ref).abs() / tol)[ok].max())


def tables_ref(free, F, ctx, new, table, page, T, finished):
    """step_tables in plain Python; returns what it returns plus the updated stack and table."""
    B, M = len(ctx), len(table[0]) if table else 0
    table = [row[:] for row in table]
    free = free[:]
    stack = free[:F]
    for b in range(B):
        if finished and finished[b]:
            stack += table[b][:-(-ctx[b] // page)]
    top, used = len(stack), 0
    cu, lens, adm, pos, slots = [0], [], [], [], []
    taken = 0
    for b in range(B):
        n = 0 if finished and finished[b] else new[b]
        cu.append(cu[-1] + n)
        held, end = -(-ctx[b] // page), -(-(ctx[b] + n) // page)
        fits = end <= M and not (finished and finished[b])
        need = end - held if fits and n > 0 else 0
        taken += need
        ok = fits and (need == 0 or taken <= top)
        if ok and need:
            used = taken
            for i in range(need):
                table[b][held + i] = stack[top - 1 - (taken - need) - i]
        adm.append(ok)
        lens.append(ctx[b] + n if ok else 0)
        for t in range(n):
            p = ctx[b] + t
            pos.append(p)
            slots.append(table[b][p // page] * page + p % page if ok else -1)
    left = top - used
    for i in range(F, left):
        free[i] = stack[i]
    pos, slots = (pos + [0] * T)[:T], (slots + [-1] * T)[:T]
    return dict(cu=cu, lens=lens, positions=pos, slots=slots, left=left, admitted=adm, free=free, table=table)


def norm_rope_ref(x, w, eps, pos, table, interleaved):
    """One of q, k in 64 bits: norm, then rotation with the table's row; and the sum of magnitudes of each output."""
    R = table.shape[1]
    y = x.double()
    if w is not None:
        y = y * (y.square().mean(-1, keepdim=True) + eps).rsqrt() * w.double()
    row = table[pos.long()].double()[:, None, :]
    c, s = row[..., :R // 2], row[..., R // 2:]
    out, mag = y.clone(), y.abs()
    ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia], mag[..., ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, mag
