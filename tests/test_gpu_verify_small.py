"""Verification of drafts whose probabilities are fp64's smallest numbers: a draft of probability e^-700 to e^-738 stands as the rule has it, also where that
is below 2^-1022 and has fewer bits. The two sides of the comparison are a sixteenth apart, and at e^-738 = 2^-1064.7 a step is 2^-9 of a number; q, u q and p are
rounded to steps once or twice each."""
import numpy as np
import pytest

import test_gpu_verify as verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("u,count", [(0.75, 2), (0.85, 1)])
def test_drafts_of_the_smallest_probabilities(gpu, u, count):
    depth = np.linspace(700.0, 738.0, 153)
    c = verify.Case(gpu, [2] * len(depth), 5, verify.F32, True, seed=1)
    c.logits[:], c.draft[:] = [0.0, -20.0, 0.0, -90.0, -np.inf], [0.0, -40.0, 0.0, -95.0, -np.inf]
    c.logits[::2, 3], c.draft[::2, 3] = -depth, -(np.float32(depth) - np.log(1.25))
    c.tokens[1::2] = 3
    c.accept[:] = u
    out, counts = c.run()
    assert np.all(counts == count)
    assert np.all(out[::2] == (3 if count == 2 else 1))
