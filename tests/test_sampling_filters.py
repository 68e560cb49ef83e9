"""Filters of a draw, as far as they go without a GPU."""
import math

import numpy as np
import pytest
import torch

import plain_sampling as P
from ferrum_b200.errors import InvalidRequest, KernelError


@pytest.mark.parametrize("kw,name", [(dict(top_k=-1), "top_k"), (dict(top_k=1.5), "top_k"), (dict(top_k=1 << 31), "top_k"), (dict(top_k=True), "top_k"),
                                     (dict(top_p=0.0), "top_p"), (dict(top_p=1.1), "top_p"), (dict(top_p=math.nan), "top_p"), (dict(top_p=1e-60), "top_p"),
                                     (dict(min_p=-0.1), "min_p"), (dict(min_p=1.2), "min_p"), (dict(min_p=math.nan), "min_p")])
def test_filters_out_of_range(kw, name):
    from ferrum_b200.sampling import Filters
    with pytest.raises(InvalidRequest, match=name):
        Filters(**kw)


@pytest.mark.parametrize("top_k", [math.inf, -math.inf, math.nan, None, "a"])
def test_top_k_that_is_no_whole_number(top_k):
    from ferrum_b200.sampling import Filters
    with pytest.raises(InvalidRequest, match="top_k"):
        Filters(top_k=top_k)


def test_filters_on():
    from ferrum_b200.sampling import Filters
    assert not Filters().on and Filters(3).on and Filters(0, 0.5).on and Filters(0, 1.0, 0.1).on


def test_random_numbers():
    """In [0, 1), a function of (seed, counter) alone, evenly spread."""
    from ferrum_b200.sampling.sampler import uniform
    u = np.array([[uniform(s, c) for c in range(400)] for s in (0, 1, 7, -5, 2 ** 64 - 1)])
    assert u.min() >= 0 and u.max() < 1 and len(np.unique(u)) == u.size
    assert uniform(-5, 3) == uniform(2 ** 64 - 5, 3)
    # the mean of 400 is off by 5 standard deviations (0.289 / 20 each) once in two million times
    assert np.abs(u.mean(1) - 0.5).max() < 5 * 0.289 / 20


def test_plain_filters():
    x = np.log(np.array([4.0, 1.0, 2.0, 2.0, 1.0]))
    assert np.allclose(P.kept(x, 1.0, 2, 1.0, 0.0), [1, 0, 0.5, 0, 0])
    assert np.allclose(P.kept(x, 1.0, 0, 0.59, 0.0), [1, 0, 0.5, 0, 0])         # 4 + 2 of 10 reach 0.59
    assert np.allclose(P.kept(x, 1.0, 0, 0.61, 0.0), [1, 0, 0.5, 0.5, 0])
    assert np.allclose(P.kept(x, 1.0, 0, 1.0, 0.4), [1, 0, 0.5, 0.5, 0])
    assert [P.draw(x, 1.0, 0, 1.0, 0.0, u)[0] for u in (0.0, 0.39, 0.41, 0.51, 0.95)] == [0, 0, 1, 2, 4]


def test_wrapper_refuses():
    from ferrum_b200.ops import lib as ops
    x, f, i = torch.zeros(2, 10), torch.zeros(2), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(KernelError, match="CUDA tensor"):
        ops.sample_filtered(x, 2, i, i, f, i, f, f, f.double())
    assert ops.lib().ferrum_sample_filtered(None, 5, 2, 2, 10, None, None, None, None, None, None, None, None, None, None) == 1
    assert b"bad sizes" in ops.lib().ferrum_last_error()
    assert ops.lib().ferrum_sample_filtered(None, 10, 2, 2, 10, None, None, None, None, None, None, None, None, None, None) == 1
    assert b"required" in ops.lib().ferrum_last_error()
