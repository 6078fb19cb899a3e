"""Adapters at ranks between the powers of two, and above 128 with more than 16 tokens a request: the shapes of the two kernels that
test_gpu_batch.py's sizes do not reach, against the same plain form and within the same bounds."""
import pytest

import test_gpu_batch as base

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2

# tokens of each request, adapters of each, K, M, rank
RANKS = [([1] * 9, [0, 3, -1, 2, 2, 1, 1, 0, 3], 512, 130, 24), ([70, 130], [2, 0], 516, 260, 24), ([40, 33], [1, 3], 300, 96, 17), ([50], [0], 96, 132, 32),
         ([60, 21], [1, -1], 333, 140, 200), ([45, 80], [3, 0], 640, 257, 256), ([90], [2], 100, 64, 129), ([20, 30], [0, 1], 128, 40, 65)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,adapter,K,M,r", RANKS)
def test_lora_ranks(gpu, dtype, new, adapter, K, M, r):
    base.test_lora_add(gpu, dtype, new, adapter, K, M, r)
