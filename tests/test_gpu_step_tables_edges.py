"""Block bookkeeping at the edges of its sizes, strides and lengths."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def test_table_rows_that_overlap_are_refused(cuda):
    """The table is written in place: one row expanded over the requests has no room of its own for each."""
    from smaq_b200 import ops
    row = ints([5, -1, -1], cuda)
    for shared in (row[None].expand(2, -1), row.as_strided((2, 2), (1, 1))):
        with pytest.raises(ValueError, match="rows of their own"):
            ops.step_tables(ints([1, 2, 3], cuda), ints([3], cuda), ints([0, 0], cuda), ints([4, 4], cuda), shared, block_size=16, num_tokens=8)
    assert row.tolist() == [5, -1, -1]
    t = ops.step_tables(ints([1, 2, 3], cuda), ints([3], cuda), ints([0], cuda), ints([4], cuda), row[None].expand(1, -1), block_size=16, num_tokens=4)
    assert t.slots.tolist() == [48, 49, 50, 51] and row.tolist() == [3, -1, -1]


BIG = 2 ** 31 - 1


def walk(ctx, new, page, M, stack, table):
    """One step in plain Python; sums stop at 2^31 - 1, and a request that reaches it is not admitted."""
    cu, adm, lens, slots, taken, used = [0], [], [], [], 0, 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        cu.append(min(cu[-1] + n, BIG))
        room = min(page * M, BIG - 1)
        held, end = -(-c // page), -(-(c + n) // page)
        need = end - held if n and c + n <= room else 0
        taken = min(taken + need, BIG)
        ok = c + n <= room and cu[-1] < BIG and (need == 0 or taken <= len(stack))
        if ok and need:
            used = taken
            table[b][held:end] = [stack[len(stack) - 1 - (taken - need) - i] for i in range(need)]
        adm.append(ok)
        lens.append(c + n if ok else 0)
        for i in range(c, c + min(n, 50)):
            slots.append(table[b][i // page] * page + i % page if ok else -1)
    return cu, adm, lens, slots, len(stack) - used, table


@pytest.mark.parametrize("page,M", [(1, 8), (16, 4), (24, 3), (1 << 30, 4), (2 ** 31 - 1, 2)])
def test_lengths_that_no_row_holds(cuda, page, M):
    """Lengths and sums past 2^31 admit nobody, and the others are served as without them."""
    from smaq_b200 import ops
    ctx, new = [0, 3, BIG, BIG, 2 ** 30, 5, 0, -9, 7], [2, 1, 1, 0, 2 ** 30, BIG, BIG, 4, 1]
    free, stack = list(range(100, 120)), list(range(100, 120))
    table = torch.full((len(ctx), M), 55, dtype=torch.int32, device=cuda)
    want = walk(ctx, new, page, M, stack, table.tolist())
    t = ops.step_tables(ints(free, cuda), ints([20], cuda), ints(ctx, cuda), ints(new, cuda), table, block_size=page, num_tokens=9)
    assert (t.cu_query.tolist(), t.admitted.tolist(), t.seq_lens.tolist()) == want[:3]
    assert t.slots.tolist() == want[3][:9] and t.free_count.tolist() == [want[4]] and table.tolist() == want[5]
    # ended requests give back what their row holds, at most
    pool = torch.cat([ints(free, cuda), torch.full((20,), -1, dtype=torch.int32, device=cuda)])
    t = ops.step_tables(pool, ints([20], cuda), ints([BIG, -4], cuda), ints([1, 1], cuda), table[:2].clone(), block_size=page, num_tokens=2,
                        finished=torch.tensor([True, True], device=cuda))
    assert t.free_count.tolist() == [20 + min(M, -(-BIG // page))] and t.seq_lens.tolist() == [0, 0] and t.cu_query.tolist() == [0, 0, 0]


def test_slow_garbage_does_not_disturb_the_next_step(cuda):
    from smaq_b200 import ops
    for _ in range(3):
        free = torch.arange(8, dtype=torch.int32, device=cuda)
        table = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
        ops.step_tables(free, ints([BIG], cuda), ints([-2 ** 31, BIG], cuda), ints([BIG, BIG], cuda), table, block_size=4, num_tokens=5)
        t = ops.step_tables(free, ints([8], cuda), ints([0, 0], cuda), ints([4, 5], cuda), table, block_size=4, num_tokens=9)
        assert t.slots.tolist() == [28, 29, 30, 31, 24, 25, 26, 27, 20] and t.free_count.tolist() == [5]


@pytest.mark.parametrize("B", [4096, 4079, 4080, 4081, 4097, 16384])   # 4096 before any larger batch of the process
def test_batches_around_the_default_limit_of_shared_memory(cuda, B):
    from smaq_b200 import ops
    page, M = 16, 4
    ctx, new = [b % 40 for b in range(B)], [(b * 7) % 5 for b in range(B)]
    stack = list(range(3 * B, 3 * B + B // 8))
    table = torch.arange(3 * B, dtype=torch.int32).view(B, 3)
    table = torch.cat([table, torch.full((B, 1), -1, dtype=torch.int32)], 1).to(cuda)
    want = walk(ctx, new, page, M, stack, table.tolist())
    t = ops.step_tables(ints(stack, cuda), ints([len(stack)], cuda), ints(ctx, cuda), ints(new, cuda), table, block_size=page, num_tokens=sum(new))
    assert (t.cu_query.tolist(), t.admitted.tolist(), t.seq_lens.tolist()) == want[:3]
    assert t.slots.tolist() == want[3] and t.free_count.tolist() == [want[4]] and table.tolist() == want[5]
