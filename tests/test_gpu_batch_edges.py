"""The batch calls on the GPU at the ends of their ranges. Tolerances as in test_gpu_batch.py."""
import pytest

import test_gpu_batch as base
from batch_ref import Batch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 30, 5])
@pytest.mark.parametrize("new,kv,Hq,Hk", [([40], [4], 2, 1), ([40, 1], [4, 3000], 2, 1), ([200], [8], 8, 8), ([200, 1], [8, 3000], 8, 8)])
def test_wide_windows_and_positions_before_the_first(gpu, new, kv, Hq, Hk, window):
    """More new tokens than positions: the first ones are before position 0 and get zeros, the rest see what is there."""
    b = Batch(gpu, new, kv, 16, Hk, 64, F16, seed=window % 7)
    base.check_attention(gpu, b, F32, Hq, 1, window)
