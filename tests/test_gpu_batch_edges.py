"""The batch calls on the GPU at the ends of their ranges. Tolerances as in test_gpu_batch.py."""
import pytest

import test_gpu_batch as base
from batch_ref import Batch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2

# Sequences (new tokens, cached positions), query heads, key/value heads: 16 rows a tile and 128, in one part and in several.
FEW_ONE = ([3, 9], [9, 100], 2, 1)
FEW_PARTS = ([40, 1], [1400, 2100], 4, 2)
TILES_ONE = ([90, 170], [90, 200], 8, 8)
TILES_PARTS = ([150, 130], [1700, 900], 8, 8)
FORMS = [FEW_ONE, FEW_PARTS, TILES_ONE, TILES_PARTS]


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 30, 5])
@pytest.mark.parametrize("new,kv,Hq,Hk", [([40], [4], 2, 1), ([40, 1], [4, 3000], 2, 1), ([200], [8], 8, 8), ([200, 1], [8, 3000], 8, 8)])
def test_wide_windows_and_positions_before_the_first(gpu, new, kv, Hq, Hk, window):
    """More new tokens than positions: the first ones are before position 0 and get zeros, the rest see what is there."""
    b = Batch(gpu, new, kv, 16, Hk, 64, F16, seed=window % 7)
    base.check_attention(gpu, b, F32, Hq, 1, window)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("scale,q_std", [(0.0, 1e-20), (1e-30, 1e-15), (0.0, 1e20)])
def test_scale_of_zero_and_tiny_queries(gpu, new, kv, Hq, Hk, scale, q_std):
    """Every weight is the same, whatever the size of the queries: rows are the mean of the values that they see."""
    b = Batch(gpu, new, kv, 16, Hk, 64, F16, seed=3)
    base.check_attention(gpu, b, F32, Hq, 1, 0, scale=scale, q_std=q_std)
