"""Engine.paged_plan's checks of its own, without a GPU."""

import types

import pytest

from fast_dllm_relax_b200.engine import Engine


def plan(*args, **kw):
    def reached(*a):
        raise AssertionError("handed to the library")

    return Engine.paged_plan(types.SimpleNamespace(lib=types.SimpleNamespace(fdllm_paged_plan_batch=reached), _h=None),
                             *args, **kw)


@pytest.mark.parametrize("args,kw", [
    (([2 ** 32 + 1], [0]), {}), (([1], [2 ** 32 + 5]), {}), (([1], [0], [2 ** 32]), {}), (([1], [2 ** 31]), {}),
    (([-2 ** 32 + 1], [0]), {}), (([1, 1], [0, 2 ** 40]), {}), (([1], [0]), dict(causal_block=2 ** 32)),
    (([1], [0]), dict(page_size=2 ** 32 + 32)),
])
def test_numbers_past_32_bits_are_refused_not_cut(args, kw):
    with pytest.raises(ValueError, match="32 bits"):
        plan(*args, **kw)


def test_unequal_lists_are_refused():
    for args in (([1], []), ([1], [0, 0]), ([1], [0], [])):
        with pytest.raises(ValueError, match="one start"):
            plan(*args)


def test_ordinary_numbers_reach_the_library():
    for args, kw in ((([1, 2], [0, 2 ** 30]), {}), (([], []), {}), (([3], [5], [9]), dict(causal_block=32, page_size=16))):
        with pytest.raises(AssertionError, match="handed"):
            plan(*args, **kw)
