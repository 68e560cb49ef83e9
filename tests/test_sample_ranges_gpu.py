"""Filtered draws: parameters at the ends of their ranges, calls from several threads."""
import math

import numpy as np
import pytest
import torch

from test_sample_filtered_gpu import sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_p", [1.5, math.inf, float(np.nextafter(np.float32(1), np.float32(2))), -math.inf])
@pytest.mark.parametrize("V", [100, 40000])
def test_top_p_out_of_range(cuda, top_p, V):
    """A top_p beyond 1 is refused as one below 0 is, for its row alone."""
    x = torch.randn(3, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    ids, err = sample(x, [1.0] * 3, [5, 0, 5], [0.9, top_p, 1.0], [0.0] * 3, [0.5] * 3)
    good, code = sample(x, [1.0] * 3, [5, 0, 5], [0.9, 1.0, 1.0], [0.0] * 3, [0.5] * 3)
    assert code == 0 and err == 7 and ids == [good[0], -1, good[2]]
