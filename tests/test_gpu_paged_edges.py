"""Decode and prefill attention over the exact paged cache where sizes, strides and values are at an edge."""

import pytest
import torch

from test_gpu_paged_attention import BF, HF, SF, decode, prefill

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
