"""Refusals of the embedding, linear cross entropy and clipping entry points: every
malformed call is turned away on the host, before any device work (no GPU needed)."""
import ctypes

import pytest

from minitensor_cpp_b200 import abi

P = 0x10000  # an address nothing reads: the calls below return before a launch


def desc(shape, strides=None, offset=0, capacity=None, dtype=abi.FLOAT32, ptr=P):
    strides = abi.contiguous_strides(shape) if strides is None else strides
    if capacity is None:
        capacity = offset + 1 + sum(abs(s) * (e - 1) for s, e in zip(strides, shape) if e > 0)
    return abi.make_desc(ptr, capacity, dtype, shape, strides, offset)


def ints(shape, **k):
    return desc(shape, dtype=abi.INT64, **k)


def ref(d):
    return None if d is None else ctypes.byref(d)


def embedding(table, tokens, out):
    return abi.lib().mtc_embedding(ref(table), ref(tokens), 1.0, abi.NO_TOKEN, ref(out), None)


def embedding_grad(dout, tokens, dtable):
    return abi.lib().mtc_embedding_grad(ref(dout), ref(tokens), 1.0, abi.NO_TOKEN, 0, ref(dtable), None)


@pytest.mark.parametrize("table, tokens, out, code", [
    (desc([4, 3]), ints([5]), desc([5, 4]), abi.ERR_INVALID_ARGUMENT),           # columns differ
    (desc([4, 3]), ints([5]), desc([6, 3]), abi.ERR_INVALID_ARGUMENT),           # positions differ
    (desc([4, 3]), ints([5]), desc([5, 1, 3]), abi.ERR_INVALID_ARGUMENT),        # rank
    (desc([4]), ints([5]), desc([5, 4]), abi.ERR_INVALID_ARGUMENT),              # the table is no matrix
    (desc([4, 3]), desc([5]), desc([5, 3]), abi.ERR_INVALID_ARGUMENT),           # float tokens
    (ints([4, 3]), ints([5]), desc([5, 3]), abi.ERR_INVALID_ARGUMENT),           # whole numbers in the table
    (desc([4, 3]), ints([5]), desc([5, 3], [0, 1]), abi.ERR_INVALID_ARGUMENT),   # a written view that repeats
    (desc([4, 3]), ints([5]), desc([5, 3], [2, 1]), abi.ERR_INVALID_ARGUMENT),   # rows that overlap
    (desc([4, 3], capacity=11), ints([5]), desc([5, 3]), abi.ERR_OUT_OF_RANGE),
    (desc([4, 3]), ints([5], capacity=4), desc([5, 3]), abi.ERR_OUT_OF_RANGE),
    (None, ints([5]), desc([5, 3]), abi.ERR_INVALID_ARGUMENT),
])
def test_embedding_refuses(table, tokens, out, code):
    assert embedding(table, tokens, out) == code


def test_embedding_grad_refuses_a_table_whose_rows_overlap():
    assert embedding_grad(desc([5, 3]), ints([5]), desc([4, 3], [0, 1])) == abi.ERR_INVALID_ARGUMENT
    assert b"share addresses" in abi.lib().mtc_last_error()
    assert embedding_grad(desc([5, 3]), ints([5]), desc([4, 4])) == abi.ERR_INVALID_ARGUMENT
    assert embedding_grad(desc([5, 3]), desc([5]), desc([4, 3])) == abi.ERR_INVALID_ARGUMENT


def test_embedding_of_nothing_is_a_call_without_work():
    assert embedding(desc([4, 3]), ints([0]), desc([0, 3])) == abi.OK
    assert embedding(desc([4, 0]), ints([5]), desc([5, 0])) == abi.OK
    assert embedding_grad(desc([5, 0]), ints([5]), desc([4, 0])) == abi.OK


def ce(x, w, t, loss, bias=None, lse=None):
    return abi.lib().mtc_linear_cross_entropy(ref(x), ref(w), ref(bias), ref(t), -100, ref(loss), ref(lse), None)


def ce_grad(x, w, t, dloss, dx=None, dw=None, bias=None, db=None, loss=None, lse=None):
    return abi.lib().mtc_linear_cross_entropy_grad(ref(x), ref(w), ref(bias), ref(t), -100, ref(dloss), ref(loss),
                                                   ref(lse), ref(dx), ref(dw), ref(db), None)


X, W, T, L = desc([6, 4]), desc([9, 4]), ints([6]), desc([6])


@pytest.mark.parametrize("call", [
    lambda: ce(desc([6, 5]), W, T, L),                 # columns of x and weight differ
    lambda: ce(desc([6, 4, 1]), W, T, L),
    lambda: ce(X, W, ints([5]), L),
    lambda: ce(X, W, desc([6]), L),                    # float targets
    lambda: ce(X, W, T, desc([5])),
    lambda: ce(X, W, T, desc([6, 1])),
    lambda: ce(X, W, T, desc([6], [0])),               # a written view that repeats
    lambda: ce(X, W, T, None),
    lambda: ce(X, W, T, L, bias=desc([8])),
    lambda: ce(X, W, T, L, bias=ints([9])),
    lambda: ce(X, W, T, L, lse=desc([7])),
    lambda: ce(X, desc([0, 4]), T, L),                 # no classes
    lambda: ce(None, W, T, L),
    lambda: ce(X, W, None, L),
    lambda: ce_grad(X, W, T, None),
    lambda: ce_grad(X, W, T, desc([5])),
    lambda: ce_grad(X, W, T, L, dx=desc([6, 5])),
    lambda: ce_grad(X, W, T, L, dx=desc([6, 4], [0, 1])),
    lambda: ce_grad(X, W, T, L, dw=desc([4, 9])),
    lambda: ce_grad(X, W, T, L, dw=desc([9, 4], [2, 1])),
    lambda: ce_grad(X, W, T, L, db=desc([4])),
])
def test_linear_cross_entropy_refuses(call):
    assert call() == abi.ERR_INVALID_ARGUMENT
    assert abi.lib().mtc_last_error()


def test_linear_cross_entropy_refuses_views_outside_their_buffers():
    assert ce(desc([6, 4], capacity=23), W, T, L) == abi.ERR_OUT_OF_RANGE
    assert ce(X, W, ints([6], capacity=5), L) == abi.ERR_OUT_OF_RANGE
    assert ce_grad(X, W, T, L, dx=desc([6, 4], capacity=20)) == abi.ERR_OUT_OF_RANGE


def norm(tensors, out):
    arr = (abi.Desc * max(len(tensors), 1))(*tensors)
    return abi.lib().mtc_global_norm(arr, len(tensors), ref(out), None)


def clip(tensors, outs, max_norm=1.0, n=None):
    a = (abi.Desc * max(len(tensors), 1))(*tensors)
    b = (abi.Desc * max(len(outs), 1))(*outs)
    return abi.lib().mtc_clip_global_norm(a, len(tensors) if n is None else n, max_norm, b, None, None)


@pytest.mark.parametrize("call", [
    lambda: norm([desc([3])], None),
    lambda: norm([desc([3])], desc([2])),                                # the norm is one number
    lambda: norm([ints([3])], desc([])),
    lambda: clip([desc([3])], [desc([4])]),
    lambda: clip([desc([3])], [desc([3, 1])]),
    lambda: clip([desc([3])], [ints([3])]),
    lambda: clip([desc([3])], [desc([3])], max_norm=-1.0),
    lambda: clip([desc([3])], [desc([3])], max_norm=float("nan")),
    lambda: clip([desc([3])], [desc([3], [0])]),                         # a written view that repeats
    lambda: clip([desc([3]), desc([3])], [desc([3]), desc([3])]),        # one output twice: scaled twice in place
    lambda: clip([desc([3]), desc([3])], [desc([3]), desc([3], offset=2)]),
    lambda: clip([desc([3])], [desc([3])], n=-1),
])
def test_clipping_refuses(call):
    assert call() == abi.ERR_INVALID_ARGUMENT


def test_clipping_refuses_more_elements_than_its_counters_hold():
    huge = desc([2 ** 41])
    assert norm([huge] * 5, desc([])) == abi.ERR_UNSUPPORTED
    assert norm([desc([2 ** 43])], desc([])) == abi.ERR_UNSUPPORTED
    assert clip([huge] * 5, [desc([2 ** 41], ptr=P * (i + 1) * 2 ** 32) for i in range(5)]) == abi.ERR_UNSUPPORTED


def test_clipping_nothing_is_a_call_without_work():
    assert clip([], []) == abi.OK
    assert clip([desc([0, 5])], [desc([0, 5])]) == abi.OK


def test_python_wrapper_turns_refusals_into_exceptions():
    import torch

    v = lambda *s: abi.View.of(torch.zeros(*s))
    t = lambda *s: abi.View.of(torch.zeros(*s, dtype=torch.int64))
    with pytest.raises(ValueError, match="columns"):
        abi.embedding(v(4, 3), t(5), v(5, 4), stream=0)
    with pytest.raises(ValueError, match="columns"):
        abi.linear_cross_entropy(v(6, 5), v(9, 4), t(6), v(6), stream=0)
    with pytest.raises(ValueError, match="outputs for"):
        abi.clip_global_norm([v(3)], 1.0, outs=[], stream=0)
    with pytest.raises(ValueError, match="max_norm"):
        abi.clip_global_norm([v(3)], -1.0, stream=0)


def test_views_of_tensors_keep_their_fields():
    """A view made of a tensor has the fields of one made of a storage, which can be set."""
    import torch

    t = torch.arange(12.0).reshape(3, 4)[1:, ::2]
    v = abi.View.of(t)
    bound = v.packed()
    assert (v.shape, v.strides, v.offset) == ((2, 2), (4, 2), 4) and v.storage.numel() == 12
    assert v.packed() == bound and bytes(v.desc()) == bound
    assert torch.equal(v.tensor(), t)
    v.offset = 1
    assert v.tensor().tolist() == [[1.0, 3.0], [5.0, 7.0]]
    s = torch.zeros(6)
    assert abi.View(s, (2, 3), (3, 1)) == abi.View.contiguous(s, (2, 3))
    assert abi.View.of(torch.ones(2, requires_grad=True)).tensor().requires_grad is False
    words = abi.View.of(torch.zeros(3, dtype=torch.int32))  # 4-byte words, as the bitwise copies take them
    assert words.desc().dtype == abi.FLOAT32
    with pytest.raises(ValueError, match="int32"):
        words.packed()


def test_views_of_tensors_are_made_when_they_are_made():
    """What is done to the tensor afterwards is not done to the view: its shape, strides and
    offset are the tensor's at the time, and it holds the memory but no autograd graph."""
    import dataclasses
    import gc
    import weakref

    import torch

    def fields(v):
        return v.offset, v.shape, v.strides, v.storage.data_ptr(), v.storage.numel()

    t = torch.arange(12.0).reshape(3, 4)[1:, 1:]
    want = (5, (2, 3), (4, 1), t.data_ptr() - 20, 12)
    first, v = abi.View.of(t), abi.View.of(t)
    before = first.packed()
    assert abi.View.of(t).offset == 5  # the first field that is asked for
    t.t_()
    assert v.packed() == before and fields(v) == want
    t.resize_(2)
    assert first.packed() == before and fields(first) == want
    other = abi.View.of(t)
    t.set_(torch.zeros(7))
    assert other.shape == (2,) and other.storage.numel() == 12
    moved = torch.zeros(3)
    held = abi.View.of(moved)
    moved.resize_(100)  # the same storage, elsewhere by now: the view goes with it
    assert held.packed() == bytes(held.desc()) and held.storage.data_ptr() == moved.data_ptr()
    x = torch.ones(4, requires_grad=True)
    y = x * 2
    graph = weakref.ref(y)
    v = abi.View.of(y)
    del y
    gc.collect()
    assert graph() is None and v.tensor().tolist() == [2.0] * 4
    assert dataclasses.is_dataclass(v) and [f.name for f in dataclasses.fields(v)] == ["storage", "shape", "strides", "offset"]
    assert dataclasses.replace(v, offset=1, shape=(3,)).tensor().tolist() == [2.0] * 3
    v.note = "as any object"
    assert v.note == "as any object" and v.packed() == bytes(v.desc())
    with pytest.raises(AttributeError, match="stride"):
        v.stride


def test_python_wrappers_hand_every_operand_over():
    """Calls without work: each wrapper's operands arrive in their places."""
    import torch

    v = lambda *s: abi.View.of(torch.zeros(*s))
    t = lambda *s: abi.View.of(torch.zeros(*s, dtype=torch.int64))
    abi.embedding(v(4, 3), t(0), v(0, 3), stream=0)
    abi.embedding_grad(v(5, 0), t(5), v(4, 0), stream=0)
    abi.linear_cross_entropy(v(0, 3), v(4, 3), t(0), v(0), bias=v(4), lse=v(0), stream=0)
    abi.linear_cross_entropy_grad(v(0, 3), v(0, 3), t(0), v(0), dx=v(0, 3), dweight=v(0, 3), bias=v(0), dbias=v(0),
                                  loss=v(0), lse=v(0), stream=0)
    abi.clip_global_norm([v(0)], 1.0, stream=0)
    for bad in ({"bias": v(3)}, {"lse": v(1)}):
        with pytest.raises(ValueError, match=next(iter(bad))):
            abi.linear_cross_entropy(v(0, 3), v(4, 3), t(0), v(0), stream=0, **bad)
    for name in ("dx", "dweight", "dbias", "bias", "loss", "lse"):
        with pytest.raises(ValueError, match=name):
            abi.linear_cross_entropy_grad(v(0, 3), v(4, 3), t(0), v(0), stream=0, **{name: v(7)})
    with pytest.raises(ValueError, match="dloss"):
        abi.linear_cross_entropy_grad(v(0, 3), v(4, 3), t(0), v(1), stream=0)
    with pytest.raises(ValueError, match="norm"):
        abi.global_norm([v(3)], v(2), stream=0)
    with pytest.raises(ValueError, match="null"):
        abi.embedding_grad(None, t(5), v(4, 3), stream=0)
