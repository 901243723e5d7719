"""Refusals of mtc_orthogonalize: every malformed call is turned away on the host, before
any device work (no GPU needed)."""
import ctypes

import pytest
from test_lm_operators_cpu import P, desc, ints

from minitensor_cpp_b200 import abi

QUINTIC = [abi.QUINTIC] * 5


def call(tensors, outs=None, steps=QUINTIC, eps=1e-7, n=None, count=None):
    outs = tensors if outs is None else outs
    a = (abi.Desc * max(len(tensors), 1))(*tensors)
    b = (abi.Desc * max(len(outs), 1))(*outs)
    flat = [v for s in steps for v in s]
    table = (ctypes.c_float * max(len(flat), 1))(*flat)
    return abi.lib().mtc_orthogonalize(a, len(tensors) if n is None else n, table,
                                       len(steps) if count is None else count, eps, b, None)


@pytest.mark.parametrize("refused", [
    lambda: call([desc([3])]),                                       # a vector
    lambda: call([desc([])]),
    lambda: call([ints([3, 4])]),
    lambda: call([desc([3, 4])], [desc([4, 3])]),
    lambda: call([desc([3, 4])], [desc([1, 3, 4])]),
    lambda: call([desc([3, 4])], [ints([3, 4])]),
    lambda: call([desc([3, 4])], [desc([3, 4], [0, 1])]),            # a written view that repeats
    lambda: call([desc([2, 3, 4])], [desc([2, 3, 4], [0, 4, 1])]),
    lambda: call([desc([3, 4], [2, 1])]),                            # in place, rows that overlap
    lambda: call([desc([3, 4]), desc([3, 4])]),                      # one output twice
    lambda: call([desc([3, 4]), desc([3, 4])], [desc([3, 4]), desc([3, 4], offset=5)]),
    lambda: call([desc([3, 4])], n=-1),
    lambda: call([desc([3, 4])], eps=-1.0),
    lambda: call([desc([3, 4])], eps=float("nan")),
    lambda: call([desc([3, 4])], eps=float("inf")),
    lambda: call([desc([3, 4])], steps=[]),
    lambda: call([desc([3, 4])], count=-1),
    lambda: call([desc([3, 4])], steps=[(1.0, 0.0, 0.0)] * 33),
    lambda: call([desc([3, 4])], steps=[(float("nan"), 0.0, 0.0)]),
    lambda: call([desc([3, 4])], steps=[(1.0, 0.0, float("inf"))]),
    lambda: call([desc([3, 4])], steps=[(2.0 ** 21, 0.0, 0.0)]),     # values that grow out of their scale
    lambda: call([desc([3, 4])], steps=[(10.0, 10.0, 10.0)] * 3),
    lambda: call([desc([3, 4])], steps=[(0.0, 2.0 ** 41, -2.0 ** 41)]),
    lambda: abi.lib().mtc_orthogonalize(None, 1, (ctypes.c_float * 3)(1, 0, 0), 1, 0.0, None, None),
    lambda: abi.lib().mtc_orthogonalize(None, 0, None, 5, 0.0, None, None),
])
def test_refused(refused):
    assert refused() == abi.ERR_INVALID_ARGUMENT
    assert abi.lib().mtc_last_error()


def test_refused_views_outside_their_buffers_and_sizes_beyond_the_counters():
    assert call([desc([3, 4], capacity=11)]) == abi.ERR_OUT_OF_RANGE
    assert call([desc([3, 4])], [desc([3, 4], capacity=11)]) == abi.ERR_OUT_OF_RANGE
    assert call([desc([1, 2 ** 30 + 1])]) == abi.ERR_UNSUPPORTED
    assert call([desc([300, 2 ** 30])]) == abi.ERR_UNSUPPORTED


def test_nothing_is_a_call_without_work():
    assert call([]) == abi.OK
    assert call([desc([0, 4]), desc([4, 0], ptr=2 * P), desc([0, 3, 4], ptr=3 * P)]) == abi.OK


def test_python_wrapper():
    import torch

    v = lambda *s: abi.View.of(torch.zeros(*s))
    abi.orthogonalize([v(0, 3)], [v(0, 3)], stream=0)
    with pytest.raises(ValueError, match="outputs for"):
        abi.orthogonalize([v(0, 3)], [], stream=0)
    with pytest.raises(ValueError, match="three numbers"):
        abi.orthogonalize([v(0, 3)], coefficients=[(1.0, 2.0)], stream=0)
    with pytest.raises(ValueError, match="three numbers"):
        abi.orthogonalize([v(0, 3)], coefficients=[(1.0, 2.0), (1.0, 2.0, 3.0, 4.0)], stream=0)
    with pytest.raises(ValueError, match="no matrix"):
        abi.orthogonalize([v(3)], stream=0)
    with pytest.raises(ValueError, match="steps"):
        abi.orthogonalize([v(0, 3)], coefficients=[], stream=0)
    with pytest.raises(ValueError, match="eps"):
        abi.orthogonalize([v(0, 3)], eps=-1.0, stream=0)
    with pytest.raises(ValueError, match="differs in shape"):
        abi.orthogonalize([v(3, 3)], [v(3, 4)], stream=0)


SHRINK = [[(2.0 ** -50, 0.0, 0.0), (1.0, 2.0 ** 100, 0.0)], [(2.0 ** -100, 2.0 ** -100, 0.0)], [(2.0 ** -61, 0.0, 0.0)],
          [(2.0 ** -31, 0.0, 0.0), (1.0, 1.0, 0.0)], [(2.0 ** -31, 0.0, 0.0), (1.0, 0.0, 1.0)], [(0.0, 0.0, 2.0 ** -62)],
          [(2.0 ** -40, 0.0, 0.0), (2.0 ** -40, 0.0, 0.0), (2.0 ** 40, 0.0, 0.0)]]


@pytest.mark.parametrize("steps", SHRINK)
def test_refused_coefficients_that_leave_next_to_nothing(steps):
    """Their values would fall out of the scales of the packed operands, and lose digits."""
    assert call([desc([300, 200])], steps=steps) == abi.ERR_INVALID_ARGUMENT
    assert b"fall" in abi.lib().mtc_last_error()


def test_coefficients_up_to_there_are_taken():
    for steps in ([(2.0 ** -60, 0.0, 0.0)], [(2.0 ** -30, 0.0, 0.0), (1.0, 2.0 ** 60, 0.0)], [(0.0, 0.0, 0.0), (1.0, 1.0, 1.0)],
                  [(2.0 ** -40, 0.0, 0.0), (2.0 ** 40, 0.0, 0.0)], [(2.0 ** -10, 0.0, 2.0 ** -30)] * 4):
        assert call([desc([0, 200])], steps=steps) == abi.OK
