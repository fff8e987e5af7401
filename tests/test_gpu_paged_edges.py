"""Decode and prefill attention over the exact paged cache where sizes, strides and values are at an edge."""

import pytest
import torch

from paged_ref import UNIT, attention64, check_attention, paged_case
from test_gpu_paged_attention import BF, HF, SF, check_lse, decode, prefill, queries, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("D", [33, 65, 127, 201, 255])
@pytest.mark.parametrize("lens,Hq,Hkv", [([700, 1, 300, 64, 65], 4, 4), ([900, 0, 129], 8, 2), ([2000], 3, 1), ([513, 70], 5, 1)])
def test_odd_head_dims_join_their_parts(cuda, dtype, D, lens, Hq, Hkv):
    """A slot of an odd head_dim starts its maximum and sum at any float."""
    decode(cuda, lens, Hq, Hkv, D, 16, dtype)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [8, 16, 64, 128, 256])
@pytest.mark.parametrize("news,ctx,kw", [
    ([250, 3, 130], [900, 700, 0], dict(window=130)), ([40], [1000], dict(window=90, prefix=[70])), ([300, 300], [260, 0], dict(window=20, prefix=[150, 5])),
    ([1, 1, 1, 1], [129, 255, 383, 511], dict(window=129))])
def test_prefill_neighbouring_blocks_with_cleared_rows(cuda, D, page, news, ctx, kw):
    """A window's two edges, or a prefix's end and the diagonal, in blocks side by side: one box of the next block or none."""
    from smaq_b200 import ops
    prefill(cuda, news, ctx, 8, 2, D, page, BF, **kw)
    ops.exact_status()


def ints(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def test_tables_whose_rows_overlap(cuda):
    """One row expanded over the requests, and rows a single column apart: as with a copy of the table."""
    from smaq_b200 import ops
    k, v, table = paged_case(cuda, [500], 2, 64, 16, BF, fill=0.0)
    q, n, cu = queries(cuda, 6, 4, 64, BF), ints([500, 490, 17], cuda), ints([0, 1, 4, 6], cuda)
    row = table[0]
    for shared in (row.expand(3, -1), row.as_strided((3, 20), (1, 1)), row[:1].expand(3, 1), table.expand(3, -1)):
        copy = shared.contiguous()
        assert torch.equal(ops.paged_decode(q[:3], k, v, shared, n), ops.paged_decode(q[:3], k, v, copy, n))
        assert torch.equal(ops.paged_prefill(q, k, v, shared, n, cu), ops.paged_prefill(q, k, v, copy, n, cu))


def test_a_workspace_with_gaps_is_refused(cuda):
    """Its size in bytes is counted from its elements, which have to lie side by side."""
    from smaq_b200 import ops
    k, v, table = paged_case(cuda, [500, 90], 2, 64, 16, BF)
    q, n = queries(cuda, 2, 4, 64, BF), ints([500, 90], cuda)
    need = ops.paged_decode_workspace_bytes(2, 4, 2, 64)
    for gappy in (torch.empty(need, 2, dtype=torch.uint8, device=cuda)[:, 0], torch.empty(1, dtype=torch.uint8, device=cuda).expand(need)):
        with pytest.raises(ValueError, match="contiguous"):
            ops.paged_decode(q, k, v, table, n, workspace=gappy)
        with pytest.raises(ValueError, match="contiguous"):
            ops.paged_prefill(q, k, v, table, n, ints([0, 1, 2], cuda), workspace=gappy)
    whole = torch.empty(need // 4 + 1, dtype=torch.float32, device=cuda)
    assert torch.equal(ops.paged_decode(q, k, v, table, n, workspace=whole), ops.paged_decode(q, k, v, table, n))


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("D", [64, 128, 96, 256])
def test_decode_nan_reaches_those_who_see_it(cuda, dtype, D):
    """A NaN query, and a NaN key at the newest token, alone in its warp's share or not, make their rows NaN and no others."""
    from smaq_b200 import ops
    lens = [1, 17, 65, 700, 1025, 33]
    k, v, table = paged_case(cuda, lens, 2, D, 16, dtype)
    q, n = queries(cuda, len(lens), 8, D, dtype), ints(lens, cuda)
    want, lse = ops.paged_decode(q, k, v, table, n, return_lse=True)
    bad = q.clone()
    bad[:, 5, D // 2] = float("nan")
    got, gl = ops.paged_decode(bad, k, v, table, n, return_lse=True)
    others = [h for h in range(8) if h != 5]
    assert bool(torch.isnan(got[:, 5]).all()) and bool(torch.isnan(gl[:, 5]).all())
    assert torch.equal(got[:, others], want[:, others]) and torch.equal(gl[:, others], lse[:, others])
    for b, L in enumerate(lens):
        k[table[b, (L - 1) // 16].long(), (L - 1) % 16, 1, 3] = float("nan")
    got, gl = ops.paged_decode(q, k, v, table, n, return_lse=True)
    assert bool(torch.isnan(got[:, 4:]).all()) and bool(torch.isnan(gl[:, 4:]).all())
    assert torch.equal(got[:, :4], want[:, :4]) and torch.equal(gl[:, :4], lse[:, :4])


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("cap", [50.0, 65.0, 3000.0, 1e6])
@pytest.mark.parametrize("D,slopes,scale", [(64, False, None), (128, False, 0.6), (128, True, None), (96, False, None), (256, False, -0.1)])
def test_caps_far_above_the_scores(cuda, dtype, cap, D, slopes, scale):
    """A score far below the cap is as exact as one without a cap: within 2^-24 of the sum of its products' sizes, D/8 + 16 times.
    (A tanh of fixed absolute error would be off by that error times the cap.)"""
    from smaq_b200 import ops
    sl = slopes_of(8, cuda) if slopes else None
    u = UNIT[dtype] if dtype != SF else 0.0

    def check(got, lse, q, k, v, table, lens, cu, u_p):
        ref, rl, capped = attention64(q, k, v, table, lens, cu, softcap=cap, slopes=sl, scale=scale)
        plain = attention64(q, k, v, table, lens, cu, slopes=sl, scale=scale)[2]
        mass, share = capped(1.0) - capped(0.0), plain(0.0) / (plain(1.0) - plain(0.0))   # of the capped weights; what scores without a cap allow
        # capped at 50 and 65 the absolute error 2^-22 of tanh counts too, in the weight and in the sum, as long as it stays below the output's rounding
        more = 2.0 ** -20 * cap if cap < 100 else 0.0
        check_attention(got, ref, lambda x: (x + share + more) * mass, dtype, u_p)
        check_lse(lse, rl)
    lens = [700, 1, 99]
    k, v, table = paged_case(cuda, lens, 2, D, 16, dtype)
    q, n = queries(cuda, 3, 8, D, dtype), ints(lens, cuda)
    check(*ops.paged_decode(q, k, v, table, n, softcap=cap, slopes=sl, scale=scale, return_lse=True), q, k, v, table, lens, [0, 1, 2, 3], u * u)
    for lens, news in (([400, 130, 9], [300, 130, 1]), ([100, 64], [90, 64])):       # the second: a table of one block
        k, v, table = paged_case(cuda, lens, 2, D, 16, dtype)
        cu = [sum(news[:i]) for i in range(len(news) + 1)]
        q = queries(cuda, cu[-1], 8, D, dtype)
        got = ops.paged_prefill(q, k, v, table, ints(lens, cuda), ints(cu, cuda), softcap=cap, slopes=sl, scale=scale, return_lse=True)
        check(*got, q, k, v, table, lens, cu, u)


def one_score_above_the_others(cuda, L, D, dtype, gap, value):
    """A cache whose token 0 scores `gap` (natural) above all others for a query along channel 0; its value is 0, theirs `value`."""
    page = 16
    pages = -(-L // page)
    k = torch.zeros(pages, page, 1, D, device=cuda, dtype=dtype)
    v = torch.full_like(k, value)
    k[0, 0, 0, 0], v[0, 0] = 8.0, 0.0
    q0 = gap * D ** 0.5 / 8.0
    return k, v, torch.arange(pages, dtype=torch.int32, device=cuda)[None], q0


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256, 96])
@pytest.mark.parametrize("gap", [9.0, 14.0, 18.5, 20.0])
def test_small_weights_add_up(cuda, dtype, D, gap):
    """Many tokens far below one that outweighs each of them: together they count, in either 16-bit type.

    The weights relative to the largest are e^-gap, about 2^-13 to 2^-29.  Decode keeps them in two parts, each a multiple of 2^-24
    2^-15 of the largest; prefill rounds them once, to a multiple of 2^-24 2^-12 of the largest or of one up to 2^3 below."""
    from smaq_b200 import ops
    L, value = 30000, 1000.0
    k, v, table, q0 = one_score_above_the_others(cuda, L, D, dtype, gap, value)
    q = torch.zeros(40, 2, D, device=cuda, dtype=dtype)
    q[:, 0, 0], q[:, 1, 0] = q0, q0 / 2
    n = ints([L], cuda)

    def check(got, rows, tokens, u_p, grain):
        x = q[rows].double()[..., 0] * k[0, 0, 0, 0].double() / D ** 0.5      # the score of token 0; the others' is 0
        w = torch.exp(-x)
        ref = (tokens - 1) * w / (1 + (tokens - 1) * w) * v[-1, 0, 0, 0].double()
        # one rounding of the output, 32-bit scores and sums, the weights' own rounding and their grain
        tol = (UNIT[dtype] + u_p + (D / 8 + 16) * 2.0 ** -24 * x.abs() + 2.0 ** -16) * ref + tokens * grain * value + 2.0 ** -25
        over = (got.double() - ref[..., None]).abs() - tol[..., None]
        assert float(over.max()) <= 0, (got.double()[0, :, 0].tolist(), ref[0].tolist(), tol[0].tolist())
    u, half = UNIT[dtype], dtype == HF
    check(ops.paged_decode(q[:1], k, v, table, n), slice(0, 1), L, u * u, 2.0 ** -39 if half else 0.0)
    out = ops.paged_prefill(q, k, v, table, n, ints([0, 40], cuda))              # rows 0 .. 39 see L - 39 .. L tokens
    for r in (0, 39):
        check(out[r:r + 1], slice(r, r + 1), L - 39 + r, u, 2.0 ** -36 if half else 0.0)
    many = torch.zeros(4000, 2, D, device=cuda, dtype=dtype) + q[:1]             # rows enough for walks of their own
    out = ops.paged_prefill(many, k, v, table, n, ints([0, 4000], cuda))
    for r in (0, 3999):
        check(out[r:r + 1], slice(0, 1), L - 3999 + r, u, 2.0 ** -36 if half else 0.0)
    out = ops.paged_prefill(q[:2], k, v, table[:, :8].contiguous(), ints([128], cuda), ints([0, 2], cuda))   # a table of one block
    for r in (0, 1):
        check(out[r:r + 1], slice(0, 1), 127 + r, u, 2.0 ** -36 if half else 0.0)


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("D", [64, 128, 256, 96])
@pytest.mark.parametrize("prefix", [None, [100, 0, 270]])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 100, 400])
def test_windows_wider_than_any_request(cuda, dtype, D, prefix, window):
    """As without one, up to the widest that an int holds."""
    from smaq_b200 import ops
    lens, news = [400, 90, 301], [260, 90, 1]
    k, v, table = paged_case(cuda, lens, 2, D, 16, dtype)
    q, n, cu = queries(cuda, 351, 8, D, dtype), ints(lens, cuda), ints([0, 260, 350, 351], cuda)
    pre = None if prefix is None else ints(prefix, cuda)
    want, lse = ops.paged_prefill(q, k, v, table, n, cu, prefix_lens=pre, return_lse=True)
    got, gl = ops.paged_prefill(q, k, v, table, n, cu, prefix_lens=pre, window=window, return_lse=True)
    assert torch.equal(got, want) and torch.equal(gl, lse)
    one = ops.paged_decode(q[:3], k, v, table, n)
    assert torch.equal(one, ops.paged_decode(q[:3], k, v, table, n, window=window))


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("D", [64, 128, 256, 96])
@pytest.mark.parametrize("width", [25, 5])     # tables of 400 and 80 tokens
def test_more_rows_than_tokens_under_a_wide_window(cuda, dtype, D, width):
    """Rows before a request's first token see nothing, and the others are not disturbed by their positions below zero."""
    from smaq_b200 import ops
    lens = [70, 33]
    k, v, table = paged_case(cuda, [400, 90], 2, D, 16, dtype)
    table = table[:, :width].contiguous()
    q, n, cu = queries(cuda, 300, 8, D, dtype), ints(lens, cuda), ints([0, 200, 300], cuda)
    want, lse = ops.paged_prefill(q, k, v, table, n, cu, return_lse=True)
    assert not want[:130].any() and bool(want[130:200].any()) and not want[200:267].any()
    for window in (2 ** 31 - 1, 2 ** 31 - 70):
        got, gl = ops.paged_prefill(q, k, v, table, n, cu, window=window, return_lse=True)
        assert torch.equal(got, want) and torch.equal(gl, lse)


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("D", [64, 256, 96])
@pytest.mark.parametrize("width,news,heads", [(20, [3, 5], 8), (20, [90, 100], 8), (5, [40, 33], 2)])
def test_rows_before_the_first_requests(cuda, dtype, D, width, news, heads):
    """cu_query may start behind the first row: rows of no request give zeros at either end."""
    from smaq_b200 import ops
    lens = [80, 70]
    k, v, table = paged_case(cuda, [300, 70], 2, D, 16, dtype)
    table, n, (a, b) = table[:, :width].contiguous(), ints(lens, cuda), news
    q = queries(cuda, 19 + a + b + 6, heads, D, dtype)
    want, lse = ops.paged_prefill(q[19:19 + a + b].contiguous(), k, v, table, n, ints([0, a, a + b], cuda), return_lse=True)
    out = torch.full_like(q, 7.0)
    got, gl = ops.paged_prefill(q, k, v, table, n, ints([19, 19 + a, 19 + a + b], cuda), out=out, return_lse=True)
    mine = slice(19, 19 + a + b)
    tol = 4 * UNIT[dtype] * float(want.float().abs().max()) if dtype != SF else 1e-5
    assert float((got[mine].float() - want.float()).abs().max()) <= tol
    none = torch.ones(q.shape[0], dtype=torch.bool, device=cuda)
    none[mine] = False
    assert not got[none].any() and bool((gl[none] == -float("inf")).all())
    check_lse(gl[mine], lse.double())


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("D", [64, 96])
@pytest.mark.parametrize("kw", [dict(window=2 ** 31), dict(window=10 ** 18), dict(softcap=1e32), dict(softcap=1e37), dict(softcap=1e200),
                                dict(softcap=float("inf")), dict(softcap=float("inf"), window=2 ** 63)])
def test_limits_beyond_every_score_and_length(cuda, dtype, D, kw):
    """A window or a cap too large for the C types is none."""
    from smaq_b200 import ops
    lens, news = [400, 90], [260, 90]
    k, v, table = paged_case(cuda, lens, 2, D, 16, dtype)
    q, n, cu, sl = queries(cuda, 350, 8, D, dtype), ints(lens, cuda), ints([0, 260, 350], cuda), slopes_of(8, cuda)
    for slopes in (None, sl):
        want, lse = ops.paged_prefill(q, k, v, table, n, cu, slopes=slopes, return_lse=True)
        got, gl = ops.paged_prefill(q, k, v, table, n, cu, slopes=slopes, return_lse=True, **kw)
        assert torch.equal(got, want) and torch.equal(gl, lse)
        assert torch.equal(ops.paged_decode(q[:2], k, v, table, n, slopes=slopes), ops.paged_decode(q[:2], k, v, table, n, slopes=slopes, **kw))
