"""The Python entry points of drafted tokens on the CPU: what they make of their arguments before the library sees them."""
import numpy as np
import pytest

import sllm_qmm as sq


class Closed(sq.PageBatch):
    """A batch without a handle: the library refuses it (a null pointer) before anything else."""

    def __init__(self):
        self.handle = None


def message(f, *args):
    with pytest.raises(sq.SllmError) as e:
        f(*args)
    assert e.value.status == 1
    return str(e.value)


@pytest.mark.parametrize("kind", [np.uint8, np.int8, np.uint16, np.int16, np.int32, np.int64])
@pytest.mark.filterwarnings("error")
def test_rows_of_any_integers_are_added_up_whole(kind):
    """The sum of the rows says how many parents are read: it does not wrap in the array's type."""
    most = min(np.iinfo(kind).max, 40000)
    rows = np.array([most, most, 5], kind)
    n = 2 * most + 5
    wrapped = int(np.array(n).astype(kind))
    for wrong in {n - 1, n + 1, max(wrapped, 0)} - {n}:
        assert "parents" in message(Closed().begin_tree, [0, 1, 2], rows, [-1] * wrong)
    assert "null pointer" in message(Closed().begin_tree, [0, 1, 2], rows, [-1] * n)


def test_a_closed_batch_is_not_no_batch():
    """logits_rules_dev without a batch is another call: rows are requests then."""
    assert "closed" in message(sq.logits_rules_dev, 64, 1, 4, sq.LogitsParams(), 0, 64, Closed())


def test_arrays_that_hold_pythons_integers():
    assert sq._ints(np.array([3, 4, 5], object))[:3] == [3, 4, 5]
    assert len(sq._ints(np.array([], object))) == 0
    for wrong in (np.array([3, 4.5], object), np.array([[1, 2]], object), np.array([3, "a"], object)):
        with pytest.raises(TypeError):
            sq._ints(wrong)
