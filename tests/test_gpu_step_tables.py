"""Block tables and slot maps on the GPU against a plain Python walk: every output is a whole number and equal."""

import random

import pytest
import torch

from paged_ref import tables_ref

pytestmark = pytest.mark.gpu


def run(cuda, ctx, new, page, M, F, *, T=None, finished=None, extra=0, seed=0):
    from smaq_b200 import ops
    rnd = random.Random(seed)
    held = [-(-c // page) for c in ctx]
    ids = list(range(sum(min(h, M) for h in held) + F + extra))
    rnd.shuffle(ids)
    free = ids[:F] + [-7] * (len(ids) - F)
    at, table = F, []
    for h in held:
        h = min(h, M)
        table.append(ids[at:at + h] + [-3] * (M - h))
        at += h
    total = sum(n for b, n in enumerate(new) if not (finished and finished[b]))
    T = total if T is None else T
    want = tables_ref(free, F, ctx, new, table, page, T, finished)
    dev_i = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    wide = torch.full((len(ctx), M + 5), -9, dtype=torch.int32, device=cuda)      # rows are a view of a wider buffer
    wide[:, :M] = dev_i(table).reshape(len(ctx), M)
    bt, fb = wide[:, :M], dev_i(free)
    fin = None if finished is None else torch.tensor(finished, device=cuda)
    for _ in range(2):  # the same call again writes the same values
        r = ops.step_tables(fb, dev_i([F]), dev_i(ctx), dev_i(new), bt, block_size=page, num_tokens=T, finished=fin)
        assert r.cu_query.tolist() == want["cu"]
        assert r.seq_lens.tolist() == want["lens"]
        assert r.admitted.tolist() == want["admitted"]
        assert r.free_count.tolist() == [want["left"]]
        assert r.positions.tolist() == want["positions"]
        assert r.slots.tolist() == want["slots"]
        assert bt.tolist() == want["table"] and bool((wide[:, M:] == -9).all())
        assert fb.tolist() == want["free"]
    return want


@pytest.mark.parametrize("page", [1, 16, 24])
def test_decode_step(cuda, page):
    ctx = [0, 1, 15, 16, 17, 47, 48, 100]
    run(cuda, ctx, [1] * 8, page, 110, 20)


@pytest.mark.parametrize("seed", range(6))
def test_random_steps(cuda, seed):
    rnd = random.Random(seed)
    B = rnd.choice([1, 3, 64, 513, 1100])
    page = rnd.choice([1, 8, 16, 24, 128])
    ctx = [rnd.choice([0, rnd.randint(0, 300)]) for _ in range(B)]
    new = [rnd.choice([0, 1, 1, rnd.randint(0, 200)]) for _ in range(B)]
    need = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(ctx, new))
    finished = [rnd.random() < 0.2 for _ in range(B)] if seed % 2 else None
    F = rnd.choice([need + 3, max(1, need // 2)])
    M = max(-(-(c + n) // page) for c, n in zip(ctx, new)) + (0 if seed % 3 else 1)
    run(cuda, ctx, new, page, max(M, 1), F, finished=finished, seed=seed, extra=3)


def test_shortage_is_in_order_and_does_not_stop_those_who_need_nothing(cuda):
    w = run(cuda, [16, 5, 16, 3, 32], [1, 2, 40, 1, 1], 16, 8, 2)
    assert w["admitted"] == [True, True, False, True, False] and w["left"] == 1


def test_pool_empty_and_row_too_narrow(cuda):
    w = run(cuda, [0, 4, 64], [5, 1, 1], 16, 4, 0)
    assert w["admitted"] == [False, True, False]
    w = run(cuda, [60, 10], [10, 10], 16, 4, 9)
    assert w["admitted"] == [False, True]


def test_all_finished_and_empty_batch(cuda):
    from smaq_b200 import ops
    run(cuda, [20, 33], [1, 1], 16, 4, 2, finished=[True, True])
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)  # noqa: E731
    r = ops.step_tables(z(4), z(1) + 3, z(0), z(0), z(0, 2), block_size=16, num_tokens=5)
    assert r.cu_query.tolist() == [0] and r.slots.tolist() == [-1] * 5 and r.free_count.tolist() == [3]


def test_padding_and_cutting(cuda):
    run(cuda, [3, 0], [4, 6], 4, 4, 9, T=17)
    run(cuda, [3, 0], [4, 6], 4, 4, 9, T=7)
    run(cuda, [3, 0], [4, 6], 4, 4, 9, T=0)


def test_wide_slots(cuda):
    """Slots past 32 bits: page numbers near 2^27 of 64 tokens."""
    from smaq_b200 import ops
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    base = 2 ** 27
    bt = i([[base + 5, -1]])
    r = ops.step_tables(i([base + 9]), i([1]), i([63]), i([3]), bt, block_size=64, num_tokens=3)
    assert r.slots.tolist() == [(base + 5) * 64 + 63, (base + 9) * 64, (base + 9) * 64 + 1]


def test_refusals(cuda):
    from smaq_b200 import ops
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)  # noqa: E731
    ok = dict(block_size=16, num_tokens=2)
    with pytest.raises(ValueError, match="free_blocks"):
        ops.step_tables(z(4).long(), z(1), z(2), z(2), z(2, 3), **ok)
    with pytest.raises(ValueError, match="block_table"):
        ops.step_tables(z(4), z(1), z(2), z(2), z(3, 3), **ok)
    with pytest.raises(ValueError, match="query_lens"):
        ops.step_tables(z(4), z(1), z(2), z(3), z(2, 3), **ok)
    with pytest.raises(ValueError, match="block_size"):
        ops.step_tables(z(4), z(1), z(2), z(2), z(2, 3), block_size=0, num_tokens=2)
    with pytest.raises(ValueError, match="finished"):
        ops.step_tables(z(4), z(1), z(2), z(2), z(2, 3), finished=z(2), **ok)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.step_tables(z(4), z(1).cpu(), z(2), z(2), z(2, 3), **ok)
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        ops.step_tables(z(4), z(1), z(16385), z(16385), z(16385, 1), **ok)
