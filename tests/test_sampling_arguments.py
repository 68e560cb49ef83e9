"""Filters that are no numbers."""
import decimal

import numpy as np
import pytest
import torch

from ferrum_b200.errors import InvalidRequest


@pytest.mark.filterwarnings("error")
@pytest.mark.parametrize("name", ["top_p", "min_p"])
@pytest.mark.parametrize("value", ["a", "0.5", b"0.5", [0.5], object(), None, 0.5j, 1e39, -1e39])
def test_filters_that_are_no_numbers(name, value):
    from ferrum_b200.sampling import Filters
    with pytest.raises(InvalidRequest, match=name):
        Filters(**{name: value})


def test_numbers_of_other_types():
    from ferrum_b200.sampling import Filters
    for half in (0.5, np.float32(0.5), np.float64(0.5), decimal.Decimal("0.5"), torch.tensor(0.5)):
        assert Filters(0, half).on and Filters(0, 1.0, half).on
    assert Filters(np.int64(3)).on and Filters(2.0).on and not Filters(0, 1, 0).on
