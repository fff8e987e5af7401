"""RequestPool over many steps: captured once and replayed, and with masks of both kinds."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_captured_step_grows_like_the_eager_one(cuda):
    """step, project and decode captured once and replayed across page boundaries, against the same steps run eagerly."""
    from smaq_b200 import ops
    from smaq_b200.integration.exact import ExactPagedCache, RequestPool
    R, Hq, Hkv, D, page, blocks = 3, 8, 2, 128, 4, 40
    rope = ops.rope_table(200, D, device=cuda)
    prompts = torch.tensor([5, 11, 1], dtype=torch.int32, device=cuda)
    rows = torch.randn(30, R, Hq + 2 * Hkv, D, device=cuda).to(torch.bfloat16)
    first = torch.randn(17, Hq + 2 * Hkv, D, device=cuda).to(torch.bfloat16)

    class Side:
        def __init__(self):
            self.pool = RequestPool(blocks, page, R, 20, cuda)
            self.cache = ExactPagedCache(blocks, page, Hkv, D, device=cuda)
            self.x = torch.zeros_like(rows[0])
            self.new = torch.ones(R, dtype=torch.int32, device=cuda)
            self.ended = torch.zeros(R, dtype=torch.bool, device=cuda)
            t = self.pool.step(prompts, 17)
            self.cache.project(first[:, :Hq], first[:, Hq:Hq + Hkv], first[:, Hq + Hkv:], t, rope)

        def step(self):
            t = self.pool.step(self.new, R, finished=self.ended)
            q = self.cache.project(self.x[:, :Hq], self.x[:, Hq:Hq + Hkv], self.x[:, Hq + Hkv:], t, rope)
            return self.cache.decode(q, self.pool.block_table, t.seq_lens), t

    eager, replayed = Side(), Side()
    state = [replayed.pool.context, replayed.pool.free_count, replayed.pool.free_blocks, replayed.pool.block_table, replayed.cache.kv]
    kept = [x.clone() for x in state]
    replayed.step()                                        # a run before the capture, taken back
    torch.cuda.synchronize()
    for x, y in zip(state, kept):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, t = replayed.step()
    for x, y in zip(state, kept):
        x.copy_(y)
    for i in range(20):
        for side in (eager, replayed):
            side.x.copy_(rows[i])
            side.ended[1] = i == 9                         # its pages are used again
        want, w = eager.step()
        graph.replay()
        assert torch.equal(out, want) and torch.equal(t.slots, w.slots) and torch.equal(t.seq_lens, w.seq_lens)
        assert torch.equal(replayed.pool.context, eager.pool.context) and torch.equal(replayed.pool.free_count, eager.pool.free_count)
        assert torch.equal(replayed.pool.block_table, eager.pool.block_table)
    assert eager.pool.context.tolist() == [25, 10, 21] and int(eager.pool.free_count) == blocks - 7 - 3 - 6


def test_a_step_keeps_no_other_buffers_alive(cuda):
    from smaq_b200.integration.exact import RequestPool
    pool = RequestPool(8, 4, 2, 4, cuda)
    pool.step(torch.tensor([3, 1], dtype=torch.int32, device=cuda), 4)
    assert pool.free_count.untyped_storage().nbytes() == 4 and pool.context.untyped_storage().nbytes() == 8


@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8])
def test_masks_of_ended_rows(cuda, dtype):
    from smaq_b200.integration.exact import RequestPool
    pool = RequestPool(8, 4, 3, 4, cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    pool.step(i32([9, 4, 3]), 16)
    assert pool.context.tolist() == [9, 4, 3] and int(pool.free_count) == 3
    for ended in ([1, 0, 0], [0, 0, 2 if dtype == torch.uint8 else 1]):
        pool.step(i32([0, 1, 0]), 1, finished=torch.tensor(ended, device=cuda).to(dtype))
    assert pool.context.tolist() == [0, 6, 0] and int(pool.free_count) == 6
    held = pool.block_table[1, :2].tolist()
    assert sorted(held + pool.free_blocks[:6].tolist()) == list(range(8))
