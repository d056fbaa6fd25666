"""styx_op_sample where the sum of the weights is near its largest, 2^63 - 2^44:
the longest rows, of one logit, with random numbers up to the last below 1."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_sample import check, gpu, params  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [2 ** 19 - 1, 523000, 522900])
@pytest.mark.parametrize("setting", [(1.0, 0, 1.0, 0.0), (1.0, 0, 0.9999, 0.0), (1.0, 2 ** 19 - 2, 1.0, 0.0),
                                     (1.0, 0, 1.0, 0.5)])
def test_random_numbers_near_1_meet_the_last_words(gpu, n, setting):  # noqa: F811
    u = np.array([0.5, 0.997, 0.9975, 0.998, 0.999, 0.9999, 1 - 2.0 ** -24], np.float32)
    got = check(gpu, np.full((len(u), n), -1.5, np.float32), params([setting]), u)
    if setting[2] == 1.0:
        assert np.array_equal(got[0], np.floor(u.astype(np.float64) * got[2]).astype(np.uint32))
