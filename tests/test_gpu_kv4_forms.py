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


def mixed(long_, many, heads):
    """`many` lengths, a few of them long: each of those costs a second of reference."""
    return (long_ + [641, 640, 639, 33, 1, 0] + [100, 70] * many)[:many]


# Shapes whose plans test_kv4_forms_plan.py asserts: lengths, heads, group, queries, window, head sizes, cached tokens
# that the call allows for.
FORMS = {
    "16-wave join": ([9000], 1, 3, [1], 0, [64, 96, 128, 256], 9000),
    "16-wave join, shorter": ([8700, 70, 8449], 1, 2, [1, 1, 1], 0, [96, 256], 66000),
    "chunks of four waves": (mixed([8000, 4100], 20, 8), 8, 1, [1] * 20, 0, [64, 96], 8000),
    "chunks of four waves, wide heads": (mixed([4000], 20, 4), 4, 2, [1] * 20, 0, [256], 6000),
    "whole, eight waves": (mixed([1500, 1313], 24, 8), 8, 1, [1] * 24, 0, [64, 128], 8000),
    "chunks in a window": ([6000, 2100, 1999], 1, 4, [1, 1, 1], 2000, [64, 96], 6000),
    "chunks in a window, queries": ([6000, 2010, 33], 1, 8, [20, 20, 20], 2000, [64, 128], 6000),
    "chunks, queries": ([3000, 500], 1, 8, [20, 9], 0, [64, 256], 3000),
}


@pytest.mark.parametrize("form,dim", [(f, d) for f in FORMS for d in FORMS[f][5]])
def test_form(form, dim):
    lens, heads, group, nqs, window, _, most = FORMS[form]
    Sequences(lens, heads, dim, max_kv=most).check(nqs, group, max_kv=most, window=window, workspace=dim == 96)


@pytest.mark.parametrize("dim", [64, 96])
def test_chunks_without_a_page(dim):
    """Chunks of 8 records, four pages: all of a chunk's pages absent, the first one's, the last one's, and all."""
    s = Sequences([3000, 1500], 1, dim)
    s.check([1, 1], 4, absent=[(0, p) for p in (4, 5, 6, 7, 20)] + [(1, p) for p in range(0, 4)])
    s.check([9, 2], 4, absent=[(0, p) for p in range(40, 47)] + [(1, p) for p in range(24)])


def test_same_bits_whatever_the_workspace_held():
    s = Sequences([9000], 1, 96)
    a = s.check([1], 4).clone()
    assert torch.equal(a, s.check([1], 4, workspace=True))
