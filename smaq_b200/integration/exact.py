"""The exact side of a paged serving step: pages for requests, and one layer's exact keys and values.

``RequestPool`` owns the pages of a cache and the requests on them.  A step says how many tokens each
request adds and which requests ended; ``ops.step_tables`` turns that into block tables, slots,
positions and lengths on the GPU, so the host reads nothing back.

``ExactPagedCache`` holds one layer's exact keys and values in the engine's layout
``[2, num_blocks, block_size, Hkv, D]``.  ``project`` norms and rotates a step's queries and keys and
writes keys and values to their slots (``ops.norm_rope``); ``decode`` and ``prefill`` attend over the
pages (``ops.paged_decode``, ``ops.paged_prefill``).

The compressed rows of ``PagedCompressedCache`` (integration/paged.py) live under the same slots and
block table: a layer may keep both, answer prompts and short histories exactly and long ones from
the compressed rows, or compare the two."""

from __future__ import annotations

from typing import Optional

import torch

from .. import ops
from .paged import PagedCompressedCache


class RequestPool:
    """Pages and requests of one paged cache: ``max_requests`` rows of up to ``max_blocks`` pages."""

    def __init__(self, num_blocks: int, block_size: int, max_requests: int, max_blocks: int,
                 device: torch.device | str = "cuda"):
        self.num_blocks, self.block_size = num_blocks, block_size
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_blocks, dtype=torch.int32, device=device)
        self.block_table = torch.zeros((max_requests, max_blocks), dtype=torch.int32, device=device)
        self.context = torch.zeros(max_requests, dtype=torch.int32, device=device)   # tokens held

    def step(self, query_lens: torch.Tensor, num_tokens: int,
             finished: Optional[torch.Tensor] = None) -> ops.StepTables:
        """Pages for ``query_lens [max_requests]`` new tokens (0: the row sits this step out) after the
        rows marked ``finished`` (bool or uint8) gave theirs back.  A row that is not admitted keeps what
        it holds.  The pool's tensors are updated in place, so that a step captured in a CUDA graph goes on
        where the last replay ended."""
        if finished is not None and finished.dtype is torch.uint8:
            finished = finished.bool()  # nothing may fail once the stack and the table are updated
        t = ops.step_tables(self.free_blocks, self.free_count, self.context, query_lens, self.block_table,
                            block_size=self.block_size, num_tokens=num_tokens, finished=finished)
        self.free_count.copy_(t.free_count)
        if finished is not None:
            self.context.masked_fill_(finished, 0)
        torch.where(t.admitted, t.seq_lens, self.context, out=self.context)
        return t


class ExactPagedCache:
    """Exact keys and values of one attention layer (module docstring)."""

    def __init__(self, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        self.kv = torch.zeros((2, num_blocks, block_size, num_kv_heads, head_dim), dtype=dtype, device=device)

    @property
    def keys(self) -> torch.Tensor:
        return self.kv[0]

    @property
    def values(self) -> torch.Tensor:
        return self.kv[1]

    def project(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tables: ops.StepTables,
                rope: torch.Tensor, *, q_weight: Optional[torch.Tensor] = None,
                k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                compressed: Optional[PagedCompressedCache] = None) -> torch.Tensor:
        """Norm and rotate the step's ``q [T, Hq, D]`` and ``k [T, Hkv, D]``, write keys and values to their
        slots and return the queries.  ``compressed``: the layer's compressed rows, written under the
        same slots."""
        out, _ = ops.norm_rope(q, k, tables.positions, rope, q_weight=q_weight, k_weight=k_weight, eps=eps,
                               interleaved=interleaved, v=v, k_cache=self.keys, v_cache=self.values,
                               slots=tables.slots)
        if compressed is not None:
            rows = self.kv.flatten(1, 2)[:, tables.slots.clamp(min=0)]
            compressed.write(rows[0], rows[1], tables.slots)
        return out

    def decode(self, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, **scores) -> torch.Tensor:
        """One new token per request, ``q [B, Hq, D]`` (keywords of ``ops.paged_decode``)."""
        return ops.paged_decode(q, self.keys, self.values, block_table, seq_lens, **scores)

    def prefill(self, q: torch.Tensor, block_table: torch.Tensor, tables: ops.StepTables, **scores) -> torch.Tensor:
        """The step's rows ``q [T, Hq, D]``, any number of new tokens per request (keywords of
        ``ops.paged_prefill``)."""
        return ops.paged_prefill(q, self.keys, self.values, block_table, tables.seq_lens, tables.cu_query, **scores)
