"""weights_laid_out with several callers, without a GPU: the layout is replaced by a counter."""
import copy
import pickle
import threading

import torch

from test_dense8_cpu import field


def counted():
    """A field whose weights laid out are numbers, in the order in which they are asked for."""
    m = field(dense_inference="int8")
    made = []

    def make():
        made.append(len(made) + 1)
        return made[-1]

    m._make_weights8 = make
    return m, made


def test_one_caller():
    m, made = counted()
    assert m._weights8 is None
    with m.weights_laid_out() as same:
        assert same is m and m._weights8 == 1
        with m.weights_laid_out():
            assert m._weights8 == 2
        assert m._weights8 == 1
    assert m._weights8 is None and made == [1, 2]
    try:
        with m.weights_laid_out():
            raise KeyError
    except KeyError:
        pass
    assert m._weights8 is None


def test_two_threads():
    """A enters, B enters, A leaves, B leaves: each has its own, and nothing is left behind."""
    m, _ = counted()
    seen = {}
    steps = [threading.Event() for _ in range(4)]

    def a():
        with m.weights_laid_out():
            seen["a"] = m._weights8
            steps[0].set()
            assert steps[1].wait(20)
            seen["a, b inside"] = m._weights8
        seen["a left"] = m._weights8
        steps[2].set()

    def b():
        assert steps[0].wait(20)
        seen["b before"] = m._weights8
        with m.weights_laid_out():
            seen["b"] = m._weights8
            steps[1].set()
            assert steps[2].wait(20)
            seen["b, a left"] = m._weights8
        seen["b left"] = m._weights8

    threads = [threading.Thread(target=f) for f in (a, b)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert seen == {"a": 1, "a, b inside": 1, "a left": None, "b before": None, "b": 2, "b, a left": 2, "b left": None}
    assert m._weights8 is None


def test_left_in_another_order_and_another_thread():
    m, _ = counted()
    first, second = m.weights_laid_out(), m.weights_laid_out()
    first.__enter__()
    second.__enter__()
    first.__exit__(None, None, None)
    assert m._weights8 == 2
    t = threading.Thread(target=second.__exit__, args=(None, None, None))
    t.start()
    t.join(30)
    assert m._weights8 is None


def test_another_model_and_copies():
    m, _ = counted()
    other, _ = counted()
    plain = field()
    with m.weights_laid_out():
        assert other._weights8 is None and plain._weights8 is None
        with plain.weights_laid_out():  # nothing to lay out
            assert plain._weights8 is None and m._weights8 == 1
    real = field(dense_inference="int8")
    with torch.no_grad():
        for c in (copy.deepcopy(real), pickle.loads(pickle.dumps(real))):
            assert c._weights8 is None and c.dense_inference == "int8"
