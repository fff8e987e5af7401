"""The exact serving step as a whole: requests come and go on shared pages over several steps, and every answer is
checked against attention in 64 bits over histories that the test keeps densely."""

import importlib.util
import os

import pytest
import torch

from conftest import REPO
from paged_ref import UNIT, attention64, check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_requests_come_and_go(cuda, dtype):
    from smaq_b200 import ops
    from smaq_b200.integration.exact import ExactPagedCache, RequestPool
    R, Hq, Hkv, D, page = 4, 6, 2, 64, 8
    pool = RequestPool(30, page, R, 20, cuda)
    cache = ExactPagedCache(30, page, Hkv, D, dtype=dtype, device=cuda)
    cache.kv.fill_(float("nan"))
    rope = ops.rope_table(200, D, device=cuda)
    g = torch.Generator().manual_seed(2)
    hist = [([], []) for _ in range(R)]
    # (new tokens of each row, rows that ended before): prompts, decodes, a prompt chunk beside decodes, reuse of pages
    plan = [([50, 1, 0, 70], []), ([1, 1, 1, 1], []), ([9, 1, 0, 1], []), ([1, 60, 30, 0], [1, 3]), ([1, 1, 1, 1], []),
            ([400, 1, 1, 0], [3]), ([1, 1, 1, 5], [])]
    for news, ended in plan:
        fin = torch.tensor([b in ended for b in range(R)], device=cuda)
        news = [0 if b in ended else n for b, n in enumerate(news)]
        before = pool.context.tolist()
        T = sum(news)
        t = pool.step(torch.tensor(news, dtype=torch.int32, device=cuda), T, finished=fin if ended else None)
        for b in ended:
            hist[b] = ([], [])
        x = torch.randn(T, Hq + 2 * Hkv, D, generator=g).to(cuda, dtype)
        q = cache.project(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], t, rope)
        _, k = ops.norm_rope(x[:, :Hq], x[:, Hq:Hq + Hkv], t.positions, rope)
        adm, cu = t.admitted.tolist(), t.cu_query.tolist()
        assert adm == [b not in ended and not (news[b] == 400) for b in range(R)]
        for b in range(R):
            if adm[b]:
                hist[b][0].append(k[cu[b]:cu[b + 1]])
                hist[b][1].append(x[cu[b]:cu[b + 1], Hq + Hkv:])
        lens = t.seq_lens.tolist()
        held = pool.context.tolist()
        assert held == [0 if b in ended else before[b] + (news[b] if adm[b] else 0) for b in range(R)]
        out = cache.prefill(q, pool.block_table, t)
        for b in range(R):
            rows = out[cu[b]:cu[b + 1]]
            if not adm[b] or not news[b]:
                assert not rows.any()
                continue
            K, V = torch.cat(hist[b][0])[None], torch.cat(hist[b][1])[None]
            assert K.shape[1] == lens[b]
            zero = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
            ref, _, bound = attention64(q[cu[b]:cu[b + 1]], K, V, zero, [lens[b]], [0, news[b]])
            check_attention(rows, ref, bound, dtype, UNIT[dtype] if dtype != torch.float32 else 0.0)
        if all(n == 1 for n in news):
            one = cache.decode(q, pool.block_table, t.seq_lens)
            assert float((one.float() - out.float()).abs().max()) <= 8 * UNIT[dtype] * float(out.float().abs().max()) + 1e-5
    pool.step(torch.zeros(R, dtype=torch.int32, device=cuda), 0, finished=torch.ones(R, dtype=torch.bool, device=cuda))
    assert int(pool.free_count) == 30 and sorted(pool.free_blocks.tolist()) == list(range(30))


def test_example_runs(cuda, capsys):
    spec = importlib.util.spec_from_file_location("exact_step", os.path.join(REPO, "examples", "exact_step.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    gaps = m.main(["--steps", "5", "--prompts", "200,7,90"])
    assert len(gaps) == 5 and all(0 <= x < 0.6 for x in gaps)
    assert "pages free" in capsys.readouterr().out


def test_step_in_a_cuda_graph(cuda):
    """The whole step captured once and replayed with other lengths in the same buffers."""
    from smaq_b200 import ops
    from smaq_b200.integration.exact import ExactPagedCache
    B, Hq, Hkv, D, page, blocks = 3, 8, 2, 128, 16, 64
    cache = ExactPagedCache(blocks, page, Hkv, D, device=cuda)
    free = torch.arange(blocks, dtype=torch.int32, device=cuda)
    count = torch.full((1,), blocks, dtype=torch.int32, device=cuda)
    table = torch.zeros(B, 20, dtype=torch.int32, device=cuda)
    ctx, new = torch.zeros(B, dtype=torch.int32, device=cuda), torch.tensor([40, 3, 20], dtype=torch.int32, device=cuda)
    x = torch.randn(64, Hq + 2 * Hkv, D, device=cuda).to(torch.bfloat16)
    rope = ops.rope_table(100, D, device=cuda)

    def step():
        t = ops.step_tables(free, count, ctx, new, table, block_size=page, num_tokens=64)
        q = cache.project(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], t, rope)
        return cache.prefill(q, table, t), cache.decode(q[:B], table, t.seq_lens)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for lens in ([40, 3, 20], [1, 1, 1], [0, 64, 0], [64, 0, 0]):
        new.copy_(torch.tensor(lens, dtype=torch.int32, device=cuda))
        graph.replay()
        want = step()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
