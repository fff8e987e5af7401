"""Bounded waits of the exact step's kernels that run out: reported by ``exact_status``, and nothing looks like an answer.

A limit of no polls at all makes every wait run out at once, copies under way or not; a few polls make some of them."""

import pytest
import torch

from paged_ref import paged_case

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture
def limit(cuda):
    from smaq_b200 import ops
    ops.exact_status()
    yield ops.exact_wait_limit
    torch.cuda.synchronize()
    ops.exact_wait_limit()
    try:
        ops.exact_status()
    except RuntimeError:
        pass
    ops.exact_status()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news,ctx,kw", [([700, 90], [300, 0], {}), ([30], [3000], dict(softcap=20.0)), ([300], [260], dict(window=20, prefix=[150]))])
@pytest.mark.parametrize("page", [16, 24])
def test_prefill(cuda, limit, D, news, ctx, kw, page):
    from smaq_b200 import ops
    lens = [n + c for n, c in zip(news, ctx)]
    k, v, table = paged_case(cuda, lens, 2, D, page, BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.randn(sum(news), 8, D, device=cuda).to(BF)
    kw = {a: i32(b) if a == "prefix" else b for a, b in kw.items()}
    kw["prefix_lens"] = kw.pop("prefix", None)
    args = (q, k, v, table, i32(lens), i32([sum(news[:i]) for i in range(len(news) + 1)]))
    want, lse = ops.paged_prefill(*args, return_lse=True, **kw)
    ops.exact_status()
    for polls in (0, 1, 2):
        limit(polls)
        got, gl = ops.paged_prefill(*args, return_lse=True, **kw)
        torch.cuda.synchronize()
        whole = ~torch.isnan(got)
        assert torch.equal(got[whole], want[whole]) and torch.equal(gl[~torch.isnan(gl)], lse[~torch.isnan(gl)])
        if polls == 0:
            assert not whole.any() and bool(torch.isnan(gl).all())
        if not whole.all():
            with pytest.raises(RuntimeError, match="paged_prefill"):
                ops.exact_status()
    limit()
    try:
        ops.exact_status()
    except RuntimeError:
        pass
    assert torch.equal(ops.paged_prefill(*args, **kw), want)
    ops.exact_status()


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_norm_rope(cuda, limit, dtype):
    from smaq_b200 import ops
    T, Hq, Hk, D = 16384, 6, 2, 128                       # enough tokens for the staged kernel
    x = torch.randn(T, Hq + 2 * Hk, D, device=cuda).to(dtype)
    table, pos = ops.rope_table(500, D, device=cuda), torch.randint(0, 500, (T,), device=cuda, dtype=torch.int32)
    slots = torch.randperm(T, device=cuda)
    w = torch.ones(D, device=cuda)

    def call(cache):
        out, _ = ops.norm_rope(x[:, :Hq], x[:, Hq:Hq + Hk], pos, table, q_weight=w, k_weight=w, v=x[:, Hq + Hk:],
                               k_cache=cache[0], v_cache=cache[1], slots=slots)
        return out
    good = torch.full((2, T // 16, 16, Hk, D), 7.0, device=cuda, dtype=dtype)
    want = call(good)
    ops.exact_status()
    limit(0)
    cache = torch.full_like(good, 7.0)
    call(cache)
    assert bool((cache == 7).all())
    with pytest.raises(RuntimeError, match="norm_rope"):
        ops.exact_status()
    limit(1)
    call(cache)
    assert bool(((cache == 7) | (cache == good)).all())
    limit()
    assert torch.equal(call(cache), want) and torch.equal(cache, good)
