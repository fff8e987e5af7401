"""Argument checks of the exact step's C entry points, on the host and without a GPU."""

import pytest


def call(name, mirror, **fields):
    from smaq_b200 import _lib
    lib = _lib.load()
    a = mirror()
    for k, v in fields.items():
        setattr(a, k, v)
    st = getattr(lib, name)(bytes(a), None)
    return st, lib.smaq_last_error().decode()


def test_sizes_match_the_library():
    import ctypes
    from smaq_b200 import _lib
    lib = _lib.load()
    for which, m in enumerate((_lib.TablesArgs, _lib.NormRopeArgs, _lib.PagedArgs)):
        assert lib.smaq_paged_args_size(which) == ctypes.sizeof(m)
    assert lib.smaq_paged_args_size(3) == 0
    assert len(_lib.pack_paged(*([0] * 30 + [0.0, 0.0]))) == ctypes.sizeof(_lib.PagedArgs)


def test_step_tables_refusals():
    from smaq_b200._lib import TablesArgs as A
    ok = dict(batch=2, max_blocks=4, page_size=16, table_stride=4, pool_size=8, n_tokens=0, free_blocks=4096, free_count=4096,
              context_lens=4096, query_lens=4096, block_table=4096, cu_query=4096, seq_lens=4096, admitted=4096, free_count_out=4096)
    for bad, word in ((dict(page_size=0), "page_size"), (dict(batch=-1), "batch"), (dict(batch=20000), "above"), (dict(seq_lens=0), "null"),
                      (dict(table_stride=3), "stride"), (dict(n_tokens=5), "null"), (dict(n_tokens=5, positions=4100, slots=4096), "aligned"),
                      (dict(pool_size=-1), "sizes")):
        st, msg = call("smaq_step_tables", A, **{**ok, **bad})
        assert st in (1, 2) and word in msg, (bad, msg)


def test_norm_rope_refusals():
    from smaq_b200._lib import NormRopeArgs as A
    ok = dict(q=4096, k=4096, positions=4096, table=4096, q_out=4096, k_out=4096, n_tokens=3, n_positions=10, dtype=1, n_q_heads=4,
              n_kv_heads=2, head_dim=64, rotary_dim=64)
    for bad, word in ((dict(dtype=9), "dtype"), (dict(head_dim=0), "sizes"), (dict(rotary_dim=65), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"),
                      (dict(q=0), "null"), (dict(k_out=0), "neither"), (dict(slots=4096), "cache write"), (dict(v=4096, k_cache=4096), "cache write")):
        st, msg = call("smaq_norm_rope", A, **{**ok, **bad})
        assert st == 1 and word in msg, (bad, msg)
    assert call("smaq_norm_rope", A, **{**ok, "n_tokens": 0})[0] == 0


@pytest.mark.parametrize("entry", ["smaq_paged_decode", "smaq_paged_prefill"])
def test_paged_refusals(entry):
    from smaq_b200._lib import PagedArgs as A
    ok = dict(q=4096, k_cache=4096, v_cache=4096, block_table=4096, table_stride=4, seq_lens=4096, cu_query=4096, out=4096, n_pages=8,
              n_rows=2, batch=2, max_blocks=4, page_size=16, n_q_heads=4, n_kv_heads=2, head_dim=128, dtype=1, scale=0.1)
    for bad, word in ((dict(dtype=-1), "dtype"), (dict(n_q_heads=5), "head counts"), (dict(head_dim=257), "head_dim"), (dict(head_dim=0), "head_dim"),
                      (dict(page_size=0), "sizes"), (dict(window=-2), "window"), (dict(softcap=-1.0), "softcap"), (dict(scale=float("nan")), "scale"),
                      (dict(table_stride=2), "stride"), (dict(q=0), "null"), (dict(seq_lens=0), "null"), (dict(block_table=0), "null"),
                      (dict(n_rows=2 ** 30), "2^31")):
        st, msg = call(entry, A, **{**ok, **bad})
        assert st in (1, 2) and word in msg, (bad, st, msg)
    if entry == "smaq_paged_decode":
        assert call(entry, A, **{**ok, "n_rows": 3})[0] == 1
        st, msg = call(entry, A, **{**ok, "workspace": 4096, "workspace_bytes": 8})
        assert st == 4 and "workspace" in msg
        assert call(entry, A, **{**ok, "n_rows": 0, "batch": 0})[0] == 0
    else:
        assert call(entry, A, **{**ok, "cu_query": 0})[0] == 1
        assert call(entry, A, **{**ok, "n_rows": 0})[0] == 0
    st, msg = call(entry, A, dtype=7)
    assert st == 1


def test_workspace_sizes():
    from smaq_b200 import ops
    assert ops.paged_decode_workspace_bytes(0, 8, 2, 128) == 0
    assert ops.paged_decode_workspace_bytes(4, 32, 8, 128) > ops.paged_decode_workspace_bytes(1, 32, 8, 128) > 0
    assert ops.paged_prefill_workspace_bytes(16, 1, 32, 8, 128) > 0
    assert ops.paged_prefill_workspace_bytes(16, 1, 32, 8, 128, 256) == 0      # a table too narrow to share
    assert ops.paged_prefill_workspace_bytes(100000, 1, 32, 8, 128) == 0       # rows enough to fill the GPU
    assert ops.paged_prefill_workspace_bytes(16, 1, 32, 8, 96) == 0
