"""Decode and prefill attention over the exact paged cache where sizes, strides and values are at an edge."""

import pytest
import torch

from test_gpu_paged_attention import BF, HF, SF, decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("D", [33, 65, 127, 201, 255])
@pytest.mark.parametrize("lens,Hq,Hkv", [([700, 1, 300, 64, 65], 4, 4), ([900, 0, 129], 8, 2), ([2000], 3, 1), ([513, 70], 5, 1)])
def test_odd_head_dims_join_their_parts(cuda, dtype, D, lens, Hq, Hkv):
    """A slot of an odd head_dim starts its maximum and sum at any float."""
    decode(cuda, lens, Hq, Hkv, D, 16, dtype)
