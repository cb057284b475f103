"""The 8-bit key/value cache on the GPU at the edges of what its entry points allow: the largest blocks of
queries."""
import numpy as np
import pytest
import torch

from test_gpu_kv_cache import attention_case

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("group", [2048, 4096])
def test_blocks_of_more_rows_than_32_bits_count(device, group):
    """The largest query_block with large groups: a block has 2^31 and 2^32 rows, the call a few thousand."""
    print(f"block rows 2^20 x {group}", flush=True)
    blocks = np.array([[[0, 2, -1]]], np.int32)
    attention_case(device, BF16, group, 1, 64, [3], [170], True, seed=41, blocks=blocks, block=1 << 20)
