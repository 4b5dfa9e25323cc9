"""Serving operators of a ragged batch on the GPU at their edges: batches of short items, unusual values, other threads and streams."""
import numpy as np
import pytest

from fandhe_ai_b200 import BF16, F32, Backend, BackendError
from fandhe_ai_b200 import paged_kv as P

from serving_ref import Batch, bf16
from test_serving_gpu import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io_bf16", [False, True])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_many_items_of_one_tile(be, dh, io_bf16):
    """Sequences of one key tile, hundreds of items to a block's turn: one of the two slots has nothing to multiply in any of them."""
    check_attention(be, Batch([1] * 700, [1 + 13 * i % 128 for i in range(700)], heads=4, kv_heads=2, dh=dh, seed=31), io_bf16)
    new = [11 + 7 * i % 20 for i in range(200)]
    check_attention(be, Batch(new, [n + 5 * i % 97 for i, n in enumerate(new)], heads=4, kv_heads=4, dh=dh, seed=32), io_bf16)
    # one tile and several tiles in turn, more rows than the variant for few rows takes
    new = [12, 60, 12, 33] * 30
    check_attention(be, Batch(new, [n + [0, 200, 90, 600][i % 4] for i, n in enumerate(new)], heads=2, kv_heads=1, dh=dh, seed=33), io_bf16)
