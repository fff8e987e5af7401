"""Decode and prefill attention over the exact paged cache, against softmax attention in 64 bits.

Tolerance per element (paged_ref.check_attention): the output's rounding; 32-bit scores (their size times
(D/8 + 16) 2^-24); weights rounded to the cache's type before the second product where a kernel does so
(prefill: one rounding; decode: hi + lo parts, u^2).  Slots that nobody wrote hold NaN throughout."""

import math

import pytest
import torch

from paged_ref import UNIT, attention64, check_attention, paged_case

pytestmark = pytest.mark.gpu
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def queries(cuda, T, Hq, D, dtype, seed=5):
    return torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(seed)).to(cuda, dtype)


def slopes_of(Hq, cuda):
    return (2.0 ** (-8.0 * torch.arange(1, Hq + 1) / Hq)).to(cuda)


def check_lse(lse, ref):
    assert torch.equal(torch.isinf(lse), torch.isinf(ref))
    ok = torch.isfinite(ref)
    assert bool(((lse.double() - ref)[ok].abs() <= 2e-5 * (1 + ref[ok].abs())).all())


def decode(cuda, lens, Hq, Hkv, D, page, dtype, slopes=False, u_p=None, **kw):
    from smaq_b200 import ops
    k, v, table = paged_case(cuda, lens, Hkv, D, page, dtype)
    q = queries(cuda, len(lens), Hq, D, dtype)
    sl = slopes_of(Hq, cuda) if slopes else None
    n = torch.tensor(lens, dtype=torch.int32, device=cuda)
    out, lse = ops.paged_decode(q, k, v, table, n, slopes=sl, return_lse=True, **kw)
    ref, rl, bound = attention64(q, k, v, table, lens, list(range(len(lens) + 1)), slopes=sl, **kw)
    assert out.shape == q.shape and out.dtype == dtype
    check_attention(out, ref, bound, dtype, UNIT[dtype] ** 2 if dtype != SF else 0.0)
    check_lse(lse, rl)
    assert torch.equal(out, ops.paged_decode(q, k, v, table, n, slopes=sl, **kw))  # and the same again, bit for bit


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("lens,Hq,Hkv,D,page", [
    ([1], 1, 1, 64, 16), ([0, 1, 2, 0], 8, 2, 128, 16), ([63, 64, 65, 129], 28, 4, 128, 16), ([1001], 32, 8, 128, 16),
    ([5000, 17, 300], 64, 8, 128, 24), ([700, 33], 40, 1, 64, 8), ([257, 900], 12, 4, 256, 64), ([90], 20, 1, 256, 128),
    ([40, 77], 6, 2, 96, 16), ([33, 100], 4, 2, 36, 7), ([19], 5, 5, 33, 4), ([50, 1], 3, 1, 200, 16)])
def test_decode(cuda, dtype, lens, Hq, Hkv, D, page):
    decode(cuda, lens, Hq, Hkv, D, page, dtype)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=100), dict(window=64, slopes=True), dict(softcap=5.0),
                                dict(softcap=30.0, window=999, slopes=True), dict(scale=0.3), dict(scale=-0.1, softcap=2.0)])
def test_decode_scores(cuda, dtype, kw):
    decode(cuda, [700, 1, 99, 100, 101], 8, 2, 128, 16, dtype, **kw)


def test_decode_many_requests(cuda):
    """More requests than the search handles at once, most of them short or empty."""
    decode(cuda, [(i * 7) % 40 if i % 3 else 0 for i in range(300)] + [900], 4, 2, 64, 16, BF)


@pytest.mark.parametrize("dtype", [BF, SF])
def test_decode_all_empty(cuda, dtype):
    decode(cuda, [0, 0, 0], 8, 2, 128, 16, dtype)


@pytest.mark.parametrize("dtype", [BF, SF])
def test_decode_infinities(cuda, dtype):
    """NaN keys and infinite values outside the window change nothing; inside they reach their own heads only."""
    from smaq_b200 import ops
    k, v, table = paged_case(cuda, [300, 200], 2, 128, 16, dtype)
    q = queries(cuda, 2, 4, 128, dtype)
    n = torch.tensor([300, 200], dtype=torch.int32, device=cuda)
    a = ops.paged_decode(q, k, v, table, n, window=50)
    k[table[0, 3].long(), 2], v[table[0, 4].long(), 1] = math.nan, math.inf
    assert torch.equal(a, ops.paged_decode(q, k, v, table, n, window=50))
    v[table[0, 18].long(), 1, 1, 5] = math.inf
    b = ops.paged_decode(q, k, v, table, n, window=50)
    assert torch.equal(b[1], a[1]) and torch.equal(b[0, :2], a[0, :2]) and bool((b[0, 2:, 5] == math.inf).all())
    keep = [c for c in range(128) if c != 5]
    assert torch.equal(b[0, 2:][:, keep], a[0, 2:][:, keep])


def prefill(cuda, news, ctx, Hq, Hkv, D, page, dtype, slopes=False, prefix=None, pad=0, mutate=None, **kw):
    from smaq_b200 import ops
    lens = [n + c for n, c in zip(news, ctx)]
    k, v, table = paged_case(cuda, lens, Hkv, D, page, dtype)
    if mutate:
        mutate(k, v, table)
    cu = [sum(news[:i]) for i in range(len(news) + 1)]
    q = queries(cuda, cu[-1] + pad, Hq, D, dtype)
    sl = slopes_of(Hq, cuda) if slopes else None
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    pre = None if prefix is None else i32(prefix)
    out, lse = ops.paged_prefill(q, k, v, table, i32(lens), i32(cu), slopes=sl, prefix_lens=pre, return_lse=True, **kw)
    ref, rl, bound = attention64(q, k, v, table, lens, cu, slopes=sl, prefix=prefix, **kw)
    assert out.shape == q.shape and out.dtype == dtype
    check_attention(out, ref, bound, dtype, UNIT[dtype] if dtype != SF else 0.0)
    check_lse(lse, rl)
    assert torch.equal(out.nan_to_num(7), ops.paged_prefill(q, k, v, table, i32(lens), i32(cu), slopes=sl, prefix_lens=pre, **kw).nan_to_num(7))


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("news,ctx,Hq,Hkv,D,page", [
    ([1], [0], 1, 1, 64, 16), ([3, 0, 1], [0, 5, 9], 8, 2, 128, 16), ([130, 64, 65], [0, 0, 0], 28, 4, 128, 16),
    ([300], [777], 32, 8, 128, 16), ([513, 40], [0, 200], 8, 8, 64, 24), ([200, 7], [31, 0], 12, 4, 256, 16),
    ([100], [0], 40, 1, 128, 128), ([33, 60], [10, 0], 6, 2, 96, 16), ([20, 9], [3, 8], 4, 2, 36, 7), ([17], [2], 3, 1, 33, 4)])
def test_prefill(cuda, dtype, news, ctx, Hq, Hkv, D, page):
    prefill(cuda, news, ctx, Hq, Hkv, D, page, dtype)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=70), dict(softcap=5.0), dict(slopes=True), dict(prefix=[100, 0, 9999]),
                                dict(window=33, prefix=[257, 3, 1], softcap=20.0, slopes=True), dict(scale=0.25)])
def test_prefill_scores(cuda, dtype, D, kw):
    prefill(cuda, [260, 1, 90], [140, 300, 0], 8, 2, D, 16, dtype, **kw)


@pytest.mark.parametrize("dtype", [BF, SF])
def test_prefill_padding_rows_and_many_requests(cuda, dtype):
    prefill(cuda, [(i * 5) % 9 for i in range(200)], [(i * 11) % 30 for i in range(200)], 4, 2, 64, 16, dtype, pad=37)


@pytest.mark.parametrize("dtype", [BF, SF])
def test_prefill_more_requests_than_threads(cuda, dtype):
    prefill(cuda, [(i * 5) % 4 for i in range(1500)], [(i * 11) % 20 for i in range(1500)], 2, 1, 64, 16, dtype, pad=5)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_prefill_infinities_reach_only_rows_that_see_them(cuda, dtype):
    """A later token's infinite or NaN value or key in the same block leaves the rows before it as they are."""
    def mutate(k, v, table):
        v[table[0, 6].long(), 3, 0, 7] = math.nan      # token 99 of request 0
        k[table[1, 1].long(), 0, 1] = math.nan         # token 16 of request 1: rows from it on are NaN in head 1
    prefill(cuda, [150, 40], [20, 0], 4, 2, 128, 16, dtype) if dtype == SF else None
    from smaq_b200 import ops
    k, v, table = paged_case(cuda, [170, 40], 2, 128, 16, dtype)
    q = queries(cuda, 190, 4, 128, dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    args = (table, i32([170, 40]), i32([0, 150, 190]))
    a = ops.paged_prefill(q, k, v, *args)
    mutate(k, v, table)
    b = ops.paged_prefill(q, k, v, *args)
    assert torch.isnan(b[79:150, :2, 7]).all() and not torch.isnan(b[:79]).any() and not torch.isnan(b[:150, 2:]).any()
    assert torch.isnan(b[166:, 2:]).all() and not torch.isnan(b[150:166]).any() and not torch.isnan(b[150:, :2]).any()
    tol = 4 * UNIT[dtype] if dtype != SF else 1e-5
    same = torch.isfinite(b)
    assert float((b.float() - a.float())[same].abs().max()) <= tol * float(a.float().abs().max())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("news,ctx,Hq,Hkv,D,page,kw", [
    ([16], [3000], 8, 2, 128, 16, {}), ([1, 0, 5], [2999, 10, 700], 8, 2, 64, 8, dict(slopes=True)),
    ([70], [1500], 4, 4, 128, 24, dict(softcap=9.0)), ([3, 130], [513, 2000], 7, 1, 128, 128, dict(window=900, prefix=[40, 300])),
    ([200], [900], 4, 1, 64, 256, dict(window=200)), ([33], [2500], 2, 1, 128, 1, {})])
def test_prefill_shared_walks(cuda, dtype, news, ctx, Hq, Hkv, D, page, kw):
    """Few rows behind long contexts: several CTAs share a tile's walk and their parts are joined."""
    from smaq_b200 import ops
    assert ops.paged_prefill_workspace_bytes(sum(news), len(news), Hq, Hkv, D) > 0
    prefill(cuda, news, ctx, Hq, Hkv, D, page, dtype, pad=3, **kw)


def test_prefill_shared_walks_infinities(cuda):
    """An infinite value in a window's edge block leaves rows that do not see it as they are, whichever share met it."""
    from smaq_b200 import ops
    k, v, table = paged_case(cuda, [2000], 1, 128, 16, BF)
    q = queries(cuda, 40, 2, 128, BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    args = (table, i32([2000]), i32([0, 40]))
    a = ops.paged_prefill(q, k, v, *args, window=1000)
    v[table[0, 60].long(), 12, 0, 3] = math.inf            # token 972: rows of positions 1960 .. 1971 see it
    b = ops.paged_prefill(q, k, v, *args, window=1000)
    assert bool((b[:12, :, 3] == math.inf).all()) and bool(torch.isfinite(b[12:]).all())
    assert float((b[12:].float() - a[12:].float()).abs().max()) <= 4 * UNIT[BF] * float(a.float().abs().max())
    with pytest.raises(RuntimeError, match="WORKSPACE"):
        ops.paged_prefill(q, k, v, *args, workspace=torch.empty(64, dtype=torch.uint8, device=cuda))


def test_not_admitted_and_broken_tables_stay_inside(cuda):
    """A request of length 0 with query rows gives zeros; page numbers and lengths past the cache read in bounds."""
    from smaq_b200 import ops
    k, v, table = paged_case(cuda, [64, 64], 2, 64, 16, BF, fill=0.0)
    q = queries(cuda, 20, 4, 64, BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    out, lse = ops.paged_prefill(q, k, v, table, i32([0, 64]), i32([0, 10, 20]), return_lse=True)
    assert not out[:10].any() and bool((lse[:10] == -math.inf).all()) and bool(out[10:].any())
    table[0, 0], table[1, 2] = -5, 1 << 30
    for lens in ([10 ** 9, 2 ** 31 - 1], [-4, 70]):
        o1 = ops.paged_prefill(q, k, v, table, i32(lens), i32([0, 10, 20]))
        o2 = ops.paged_decode(q[:2], k, v, table, i32(lens))
        assert bool(torch.isfinite(o1).all()) and bool(torch.isfinite(o2).all())
    assert bool(torch.isfinite(ops.paged_prefill(q, k, v, table, i32([64, 64]), i32([-3, 10, 10 ** 6]))).all())


@pytest.mark.parametrize("dtype,D", [(SF, 64), (SF, 128), (SF, 256), (SF, 96), (SF, 33), (BF, 96), (HF, 36), (BF, 201)])
@pytest.mark.parametrize("news,ctx,Hq,Hkv,page,kw", [
    ([260, 0, 90], [140, 300, 0], 8, 2, 16, {}), ([1, 700], [90, 0], 7, 1, 24, dict(window=70, slopes=True)),
    ([333], [500], 12, 12, 7, dict(window=33, prefix=[257], softcap=20.0)), ([100], [63], 28, 4, 64, dict(window=1, pad=70))])
def test_prefill_many_rows_in_32_bits(cuda, dtype, D, news, ctx, Hq, Hkv, page, kw):
    """fp32 and the head dims that the tensor cores do not take, with rows enough for tiles of 64."""
    prefill(cuda, news, ctx, Hq, Hkv, D, page, dtype, **kw)


@pytest.mark.parametrize("dtype,D", [(SF, 128), (SF, 256), (BF, 96), (SF, 33)])
def test_prefill_many_rows_infinities(cuda, dtype, D):
    from smaq_b200 import ops
    k, v, table = paged_case(cuda, [400, 90], 2, D, 16, dtype)
    q = queries(cuda, 470, 8, D, dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    args = (table, i32([400, 90]), i32([0, 380, 470]))
    a = ops.paged_prefill(q, k, v, *args)
    v[table[0, 6].long(), 3, 0, 7] = math.inf       # token 99 of request 0: rows from 79 on, head 0 of the cache
    v[table[0, 20].long(), 0, 1, 1] = math.nan      # token 320: rows from 300 on, head 1
    k[table[1, 1].long(), 0, 1] = math.nan          # token 16 of request 1: rows from 396 on are NaN, head 1
    b = ops.paged_prefill(q, k, v, *args)
    good = torch.ones_like(b, dtype=torch.bool)
    good[79:380, :4, 7] = False
    good[300:380, 4:, 1] = False
    good[396:, 4:] = False
    assert bool((b[79:380, :4, 7] == math.inf).all()) and bool(torch.isnan(b[300:380, 4:, 1]).all()) and bool(torch.isnan(b[396:, 4:]).all())
    assert bool(torch.isfinite(b[good]).all())
    tol = 4 * UNIT[dtype] if dtype != SF else 1e-5
    assert float((b.float() - a.float())[good].abs().max()) <= tol * float(a.float().abs().max())


@pytest.mark.parametrize("dtype", [BF, SF])
def test_strides_streams_workspace(cuda, dtype):
    """Queries and outputs as views of wider buffers, caches as the halves of one buffer, another stream, a kept workspace."""
    from smaq_b200 import ops
    lens, D = [500, 81, 7], 128
    k, v, table = paged_case(cuda, lens, 2, D, 16, dtype)
    q = queries(cuda, 3, 8, D, dtype)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda)
    want = ops.paged_decode(q, k, v, table, n)
    both = torch.stack([k, v]).transpose(1, 3).contiguous().transpose(1, 3)     # heads outside slots
    wide = torch.zeros(3, 12, D, device=cuda, dtype=dtype)
    wide[:, 4:] = q
    out = torch.zeros(3, 20, D, device=cuda, dtype=dtype)
    ws = torch.empty(ops.paged_decode_workspace_bytes(3, 8, 2, D), dtype=torch.uint8, device=cuda)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(3):
            ops.paged_decode(wide[:, 4:], both[0], both[1], table, n, out=out[:, 5:13], workspace=ws)
    s.synchronize()
    assert torch.equal(out[:, 5:13], want) and not out[:, :5].any() and not out[:, 13:].any()
    # one off 16-byte alignment: the general kernels
    odd = torch.zeros(3 * 8 * D + 1, device=cuda, dtype=dtype)[1:].view(3, 8, D)
    odd.copy_(q)
    got = ops.paged_decode(odd, k, v, table, n)
    assert float((got.float() - want.float()).abs().max()) <= 4 * UNIT[dtype] * float(want.float().abs().max()) + 1e-6
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda)
    a = ops.paged_prefill(q, k, v, table, n, cu)
    b = ops.paged_prefill(odd, k, v, table, n, cu)
    ops.paged_prefill(wide[:, 4:], both[0], both[1], table, n, cu, out=out[:, 5:13])
    assert torch.equal(out[:, 5:13], a)
    for x in (a, b):
        assert float((x.float() - want.float()).abs().max()) <= 4 * UNIT[dtype] * float(want.float().abs().max()) + 1e-6


def test_offsets_past_32_bits(cuda):
    from smaq_b200 import ops
    P, page, H, D = 140000, 16, 8, 128                       # 2.3e9 elements a cache
    k = torch.empty(P, page, H, D, dtype=BF, device=cuda)
    v = torch.empty_like(k)
    lens = [200]
    ks, vs, ts = paged_case(cuda, lens, H, D, page, BF)
    far = torch.arange(P - 14, P, dtype=torch.int32, device=cuda)[None]
    for i in range(13):
        k[P - 14 + i], v[P - 14 + i] = ks[ts[0, i].long()], vs[ts[0, i].long()]
    n = torch.tensor(lens, dtype=torch.int32, device=cuda)
    q = queries(cuda, 40, 16, D, BF)
    assert torch.equal(ops.paged_decode(q[:1], k, v, far, n), ops.paged_decode(q[:1], ks, vs, ts, n))
    cu = torch.tensor([0, 40], dtype=torch.int32, device=cuda)
    assert torch.equal(ops.paged_prefill(q, k, v, far, n, cu), ops.paged_prefill(q, ks, vs, ts, n, cu))
    x = torch.randn(3, 2 * H + 16, D, device=cuda, dtype=BF)
    slots = torch.tensor([0, P * page - 1, P * page - 40], device=cuda)
    table = ops.rope_table(8, D, device=cuda)
    pos = torch.zeros(3, dtype=torch.int32, device=cuda)
    ops.norm_rope(x[:, :16], x[:, 16:16 + H], pos, table, v=x[:, 16 + H:], k_cache=k, v_cache=v, slots=slots)
    assert torch.equal(k[-1, -1], x[1, 16:16 + H]) and torch.equal(v.view(-1, H, D)[P * page - 40], x[2, 16 + H:])


def test_refusals(cuda):
    from smaq_b200 import ops
    k, v, table = paged_case(cuda, [20, 30], 2, 64, 16, BF)
    q = queries(cuda, 2, 4, 64, BF)
    n = torch.tensor([20, 30], dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="rows for"):
        ops.paged_decode(q[:1], k, v, table, n)
    with pytest.raises(ValueError, match="do not divide"):
        ops.paged_decode(q[:, :3], k, v, table, n)
    with pytest.raises(ValueError, match="caches must be"):
        ops.paged_decode(q.half(), k, v, table, n)
    with pytest.raises(ValueError, match="same strides"):
        ops.paged_decode(q, k, v.transpose(1, 2).contiguous().transpose(1, 2), table, n)
    with pytest.raises(ValueError, match="window"):
        ops.paged_decode(q, k, v, table, n, window=0)
    with pytest.raises(ValueError, match="softcap"):
        ops.paged_decode(q, k, v, table, n, softcap=-1.0)
    with pytest.raises(ValueError, match="slopes"):
        ops.paged_decode(q, k, v, table, n, slopes=torch.ones(3, device=cuda))
    with pytest.raises(ValueError, match="seq_lens"):
        ops.paged_decode(q, k, v, table, n[:1])
    with pytest.raises(ValueError, match="out must be"):
        ops.paged_decode(q, k, v, table, n, out=q.float())
    with pytest.raises(RuntimeError, match="WORKSPACE"):
        ops.paged_decode(q, k, v, table, n, workspace=torch.empty(16, dtype=torch.uint8, device=cuda))
    with pytest.raises(ValueError, match="cu_query"):
        ops.paged_prefill(q, k, v, table, n, n)
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        big = torch.zeros(1, 16, 2, 264, device=cuda, dtype=BF)
        ops.paged_decode(torch.zeros(2, 4, 264, device=cuda, dtype=BF), big, big, table, n)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.paged_decode(q, k, v, table.cpu(), n)
