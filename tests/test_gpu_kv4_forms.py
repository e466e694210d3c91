"""Attention over the 4-bit cache in every form that its plan can take, against
64-bit references (tolerances: test_gpu_kv4.py; run on an MI355X)."""
import pytest
import torch

import busfill as bf
from test_gpu_kv4 import Sequences

pytestmark = pytest.mark.gpu

NO_LIMIT = 2 ** 31 - 1


@pytest.mark.parametrize("nqs,lens", [([5, 1], [2, 100]), ([40, 3], [3, 7]), ([9, 9], [0, 1])])
@pytest.mark.parametrize("group", [1, 4])
def test_windows_that_hide_nothing(nqs, lens, group):
    """The largest window, also where queries stand before the first cached token."""
    s = Sequences(lens, 2, 64, max_kv=256)
    a = s.check(nqs, group, max_kv=256)
    for window in (256, NO_LIMIT - 1, NO_LIMIT):
        assert torch.equal(a, s.check(nqs, group, max_kv=256, window=window))


def test_prompt_under_the_largest_window():
    """A row tile whose first queries stand before the first cached token (128 rows of the prompt kernel)."""
    s = Sequences([40, 120], 64, 64)
    a = s.check([70, 120], 8)
    assert torch.equal(a, s.check([70, 120], 8, window=NO_LIMIT))
