"""Norm and rotation of queries and keys with the cache write, against the formula in 64 bits.

Tolerance of an output of magnitude y made of terms of magnitude s: the output's own rounding u|y|, and 32-bit
arithmetic on the terms: the sum of squares (D/16 + 6 additions, halved by the root), root, quotient, two
weight products, two products and an addition, (D/32 + 10) 2^-24 s in all."""

import pytest
import torch

from paged_ref import TINY, UNIT, norm_rope_ref

pytestmark = pytest.mark.gpu


def near(got, ref, mag, D):
    u = UNIT[got.dtype]
    tol = u * ref.abs() + (D / 32 + 10) * 2.0 ** -24 * mag * (1 + u) + TINY[got.dtype]
    over = (got.double() - ref).abs() - tol
    assert float(over.max()) <= 0, float(((got.double() - ref).abs() / tol).max())


def case(cuda, T, Hq, Hk, D, R, dtype, norm, seed=0, P=500):
    from smaq_b200 import ops
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(T, Hq + 2 * Hk, D, generator=g) * torch.linspace(3, 0.1, D)).to(cuda, dtype)
    pos = torch.randint(0, P, (T,), generator=g, dtype=torch.int32).to(cuda)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(cuda) if norm else None for _ in range(2)]
    table = ops.rope_table(P, R, device=cuda) if R else torch.zeros(P, 0, device=cuda)
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], pos, table, w


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,R,norm", [
    (1, 32, 8, 128, 128, True), (5, 28, 4, 128, 64, True), (1000, 28, 4, 128, 128, False), (37, 12, 3, 64, 16, True),
    (9, 4, 4, 256, 256, True), (3, 2, 1, 512, 128, True), (11, 3, 1, 80, 32, True), (7, 5, 1, 96, 96, False),
    (6, 2, 2, 72, 72, True), (4, 3, 3, 20, 6, True), (2, 2, 1, 33, 10, True), (8, 2, 1, 1040, 32, True), (3, 4, 2, 64, 0, True)])
def test_formula(cuda, dtype, interleaved, T, Hq, Hk, D, R, norm):
    from smaq_b200 import ops
    q, k, _, pos, table, (wq, wk) = case(cuda, T, Hq, Hk, D, R, dtype, norm)
    qo, ko = ops.norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk, eps=1e-5, interleaved=interleaved)
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        assert got.shape == x.shape and got.dtype == dtype
        near(got, *norm_rope_ref(x, w, 1e-5, pos, table, interleaved), D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hk,D,R,norm,interleaved,cache", [
    (11999, 6, 2, 128, 128, True, False, True), (12003, 4, 1, 64, 32, True, True, True), (11901, 2, 2, 256, 64, True, False, False),
    (12500, 3, 1, 80, 48, False, True, False), (6201, 28, 4, 128, 128, False, False, True), (11877, 2, 1, 512, 512, True, True, True),
    (1201, 4, 2, 128, 128, True, False, True), (14300, 6, 2, 128, 128, True, False, True), (14301, 2, 2, 256, 64, True, False, False),
    (3700, 28, 4, 128, 128, False, True, True), (7203, 24, 6, 64, 32, True, True, True), (7105, 12, 4, 80, 48, True, True, False)])
def test_many_tokens(cuda, dtype, T, Hq, Hk, D, R, norm, interleaved, cache):
    """Enough tokens for the staged kernel: several batches a block, a ragged last one, positions and slots outside."""
    from smaq_b200 import ops
    q, k, v, pos, table, (wq, wk) = case(cuda, T, Hq, Hk, D, R, dtype, norm, seed=7)
    pos[5], pos[T - 1], pos[1000] = 500, -3, 2 ** 31 - 1
    kw = dict(q_weight=wq, k_weight=wk, eps=1e-5, interleaved=interleaved)
    if cache:
        P = T // 16 + 2
        kc, vc = torch.full((2, P, 16, Hk, D), 7.0, device=cuda, dtype=dtype).unbind(0)
        slots = torch.randperm(P * 16, generator=torch.Generator().manual_seed(1))[:T].to(cuda)
        slots[7], slots[T - 2] = -1, P * 16
        qo, _ = ops.norm_rope(q, k, pos, table, v=v, k_cache=kc, v_cache=vc, slots=slots, **kw)
        keep = (slots >= 0) & (slots < P * 16)
        ko = kc.view(-1, Hk, D)[slots.clamp(0, P * 16 - 1)]
        assert torch.equal(vc.view(-1, Hk, D)[slots[keep]], v[keep])
        left = torch.ones(P * 16, dtype=torch.bool, device=cuda)
        left[slots[keep]] = False
        assert bool((kc.view(-1, Hk, D)[left] == 7).all()) and bool((vc.view(-1, Hk, D)[left] == 7).all())
    else:
        qo, ko = ops.norm_rope(q, k, pos, table, **kw)
        keep = torch.ones(T, dtype=torch.bool, device=cuda)
    ops.exact_status()
    bad = (pos < 0) | (pos >= 500)
    ok = ~bad
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        rows = ok & keep if got is ko else ok
        near(got[rows], *norm_rope_ref(x[rows], w, 1e-5, pos[rows], table, interleaved), D)
        rows = bad & keep if got is ko else bad
        assert bool(torch.isnan(got[rows][..., :R]).all()) and not bool(torch.isnan(got[rows][..., R:]).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 24), (36, 5)])
def test_cache_write(cuda, dtype, D, page):
    """Rows land in their slots, skipped slots and all others keep what they held; strided caches."""
    from smaq_b200 import ops
    T, Hq, Hk, R = 50, 6, 2, D // 4 * 2
    q, k, v, pos, table, (wq, wk) = case(cuda, T, Hq, Hk, D, R, dtype, True, seed=3)
    P = T // page + 3
    both = torch.full((P, 2, page, Hk, D), 7.0, device=cuda, dtype=dtype)
    kc, vc = both[:, 0], both[:, 1]
    slots = torch.randperm(P * page, generator=torch.Generator().manual_seed(1))[:T].to(cuda)
    slots[3], slots[17], slots[20] = -1, P * page, 2 ** 40
    qo, ko = ops.norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk, v=v, k_cache=kc, v_cache=vc, slots=slots)
    assert ko is None
    qr, kr = ops.norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk)
    assert torch.equal(qo, qr)
    want = torch.full_like(both, 7.0)
    for t in range(T):
        s = int(slots[t])
        if 0 <= s < P * page:
            want[s // page, 0, s % page], want[s // page, 1, s % page] = kr[t], v[t]
    assert torch.equal(both, want)


def test_weights_of_the_model_dtype_and_bare_side(cuda):
    from smaq_b200 import ops
    q, k, _, pos, table, (wq, _) = case(cuda, 20, 4, 2, 128, 128, torch.bfloat16, True)
    wq = wq.bfloat16()
    qo, ko = ops.norm_rope(q, k, pos, table, q_weight=wq)
    near(qo, *norm_rope_ref(q, wq, 1e-6, pos, table, False), 128)
    near(ko, *norm_rope_ref(k, None, 1e-6, pos, table, False), 128)


def test_rows_of_zeros_and_infinities(cuda):
    from smaq_b200 import ops
    q, k, _, pos, table, (wq, wk) = case(cuda, 6, 2, 1, 128, 128, torch.float32, True)
    q, k = q.clone(), k.clone()
    q[0] = 0
    k[1, 0, 5] = float("inf")
    pos[2], pos[3] = 500, -1     # outside the table
    qo, ko = ops.norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk)
    assert bool((qo[0] == 0).all()) and bool(torch.isnan(ko[1]).any())
    assert bool(torch.isnan(qo[2:4]).all()) and bool(torch.isfinite(qo[4:]).all()) and bool(torch.isfinite(ko[4:]).all())


def test_empty_and_other_stream(cuda):
    from smaq_b200 import ops
    q, k, _, pos, table, (wq, wk) = case(cuda, 300, 8, 2, 128, 128, torch.bfloat16, True)
    e, _ = ops.norm_rope(q[:0], k[:0], pos[:0], table)
    assert e.shape == (0, 8, 128)
    want, _ = ops.norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, _ = ops.norm_rope(q, k, pos, table, q_weight=wq, k_weight=wk)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(cuda):
    from smaq_b200 import ops
    q, k, v, pos, table, _ = case(cuda, 4, 4, 2, 64, 32, torch.bfloat16, False)
    c = torch.zeros(2, 16, 2, 64, device=cuda, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="k must be"):
        ops.norm_rope(q, k.float(), pos, table)
    with pytest.raises(ValueError, match="positions"):
        ops.norm_rope(q, k, pos[:3], table)
    with pytest.raises(ValueError, match="positions"):
        ops.norm_rope(q, k, pos.float(), table)
    with pytest.raises(ValueError, match="table"):
        ops.norm_rope(q, k, pos, torch.zeros(9, 65, device=cuda))
    with pytest.raises(ValueError, match="q_weight"):
        ops.norm_rope(q, k, pos, table, q_weight=torch.ones(32, device=cuda))
    with pytest.raises(ValueError, match="together"):
        ops.norm_rope(q, k, pos, table, v=v)
    with pytest.raises(ValueError, match="caches must be"):
        ops.norm_rope(q, k, pos, table, v=v, k_cache=c.float(), v_cache=c.float(), slots=pos.long())
    with pytest.raises(ValueError, match="heads"):
        ops.norm_rope(q, k, pos, table, v=v, k_cache=c[:, :, :1], v_cache=c[:, :, :1], slots=pos.long())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.norm_rope(q, k, pos.cpu(), table)
