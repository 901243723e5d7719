"""Refusals of the log-probability entry points: every malformed call is turned away on
the host, before any device work (no GPU needed)."""
import pytest
from test_lm_operators_cpu import desc, ints, ref

from minitensor_cpp_b200 import abi

Z, T, L = desc([6, 9]), ints([6]), desc([6])


def log_probs(logits=Z, tokens=T, out=L, lse=None, entropy=None, top=None, best=None, scale=1.0):
    return abi.lib().mtc_token_log_probs(ref(logits), ref(tokens), scale, -100, ref(out), ref(lse), ref(entropy), ref(top),
                                         ref(best), None)


def grad(logits=Z, tokens=T, dlp=L, dent=None, dlogits=Z, scale=1.0):
    return abi.lib().mtc_token_log_probs_grad(ref(logits), ref(tokens), scale, -100, ref(dlp), ref(dent), ref(dlogits), None)


@pytest.mark.parametrize("call", [
    lambda: log_probs(logits=None),
    lambda: log_probs(logits=ints([6, 9])),
    lambda: log_probs(logits=desc([])),                             # no axis of classes
    lambda: log_probs(logits=desc([6, 0])),                         # no classes
    lambda: log_probs(tokens=ints([5])),
    lambda: log_probs(tokens=ints([6, 1])),
    lambda: log_probs(tokens=desc([6])),                            # float tokens
    lambda: log_probs(tokens=None),                                 # log probabilities of nothing
    lambda: log_probs(out=desc([7])),
    lambda: log_probs(out=ints([6])),
    lambda: log_probs(out=desc([6], [0])),                          # a written view that repeats
    lambda: log_probs(lse=desc([6, 9])),
    lambda: log_probs(entropy=desc([5])),
    lambda: log_probs(entropy=desc([6], [0])),
    lambda: log_probs(top=desc([6, 0])),
    lambda: log_probs(top=desc([6, 10])),                           # more alternatives than classes
    lambda: log_probs(logits=desc([6, 99]), top=desc([6, 33])),     # more than 32
    lambda: log_probs(top=desc([6, 4]), best=ints([6, 3])),
    lambda: log_probs(top=desc([5, 4])),
    lambda: log_probs(top=desc([6])),
    lambda: log_probs(best=desc([6, 4])),                           # float indices
    lambda: log_probs(top=desc([6, 4], [2, 1])),                    # rows that overlap
    lambda: log_probs(best=ints([6, 4], strides=[0, 1])),
    lambda: log_probs(scale=0.0),
    lambda: log_probs(scale=-1.0),
    lambda: log_probs(scale=float("nan")),
    lambda: log_probs(scale=float("inf")),
    lambda: log_probs(scale=2.0 ** 101),
    lambda: grad(logits=None),
    lambda: grad(dlogits=None),
    lambda: grad(dlogits=desc([6, 8])),
    lambda: grad(dlogits=desc([6, 9, 1])),
    lambda: grad(dlogits=ints([6, 9])),
    lambda: grad(dlogits=desc([6, 9], [0, 1])),
    lambda: grad(dlp=None),                                         # no gradient comes in
    lambda: grad(tokens=None),
    lambda: grad(dlp=desc([5])),
    lambda: grad(dent=desc([6, 1])),
    lambda: grad(dlp=ints([6])),
    lambda: grad(scale=0.0),
])
def test_log_probs_refuse(call):
    assert call() == abi.ERR_INVALID_ARGUMENT
    assert abi.lib().mtc_last_error()


def test_log_probs_refuse_views_outside_their_buffers():
    assert log_probs(logits=desc([6, 9], capacity=53)) == abi.ERR_OUT_OF_RANGE
    assert log_probs(tokens=ints([6], capacity=5)) == abi.ERR_OUT_OF_RANGE
    assert log_probs(top=desc([6, 4], capacity=23)) == abi.ERR_OUT_OF_RANGE
    assert grad(dlogits=desc([6, 9], capacity=53)) == abi.ERR_OUT_OF_RANGE


def test_log_probs_refuse_more_classes_than_they_count():
    many = desc([1, 2 ** 30 + 1])
    assert log_probs(logits=many, tokens=ints([1]), out=desc([1])) == abi.ERR_UNSUPPORTED


def test_log_probs_of_nothing_are_a_call_without_work():
    assert log_probs(desc([0, 9]), ints([0]), desc([0]), top=desc([0, 3])) == abi.OK
    assert log_probs(desc([4, 0, 9]), ints([4, 0]), desc([4, 0])) == abi.OK
    assert grad(desc([0, 9]), ints([0]), desc([0]), None, desc([0, 9])) == abi.OK
    assert grad(desc([0, 9]), None, None, desc([0]), desc([0, 9])) == abi.OK


def test_python_wrappers_hand_every_operand_over():
    import torch

    v = lambda *s: abi.View.of(torch.zeros(*s))
    t = lambda *s: abi.View.of(torch.zeros(*s, dtype=torch.int64))
    fine = {"tokens": t(0), "log_probs": v(0), "lse": v(0), "entropy": v(0), "top_log_probs": v(0, 3),
            "top_tokens": t(0, 3)}
    abi.token_log_probs(v(0, 7), stream=0, **fine)
    for name in fine:
        wrong = t(5, 5) if "tokens" in name else v(5, 5)
        with pytest.raises(ValueError, match=name):
            abi.token_log_probs(v(0, 7), stream=0, **{**fine, name: wrong})
    fine = {"tokens": t(0), "dlog_probs": v(0), "dentropy": v(0)}
    abi.token_log_probs_grad(v(0, 7), v(0, 7), stream=0, **fine)
    for name in fine:
        wrong = t(5, 5) if "tokens" in name else v(5, 5)
        with pytest.raises(ValueError, match=name):
            abi.token_log_probs_grad(v(0, 7), v(0, 7), stream=0, **{**fine, name: wrong})
    with pytest.raises(ValueError, match="scale"):
        abi.token_log_probs(v(0, 7), scale=-2.0, stream=0)


def test_log_probs_refuse_scales_that_float32_differences_do_not_bear():
    for scale in (1e-45, 2.0 ** -126, 2.0 ** -101):
        assert log_probs(scale=scale) == abi.ERR_INVALID_ARGUMENT
        assert grad(scale=scale) == abi.ERR_INVALID_ARGUMENT
    for scale in (2.0 ** -100, 2.0 ** 100):
        assert log_probs(desc([0, 9]), ints([0]), desc([0]), scale=scale) == abi.OK
        assert grad(desc([0, 9]), ints([0]), desc([0]), None, desc([0, 9]), scale=scale) == abi.OK
