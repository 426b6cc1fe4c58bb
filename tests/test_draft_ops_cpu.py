"""The entry points of drafted tokens on the CPU: bad arguments are refused with status codes before a GPU is touched."""
import ctypes as C
import os

import numpy as np
import pytest

import sllm_qmm as sq


def test_bad_arguments_need_no_device():
    lib = sq.lib()
    i = (C.c_int * 4)(1, 1, 1, 1)
    p = C.addressof(i)
    none = sq.LogitsParams()
    rules = lambda x, rows, vocab, params, dst, chosen: lib.sllm_logits_rules_dev(x, rows, vocab, params, dst, chosen, None, None)  # noqa: E731
    assert lib.sllm_page_batch_begin_tree(None, i, i, 1, i, None) == 1
    assert lib.sllm_page_accept_dev(None, p, p, p, p, p, None) == 1 and lib.sllm_page_keep_dev(None, p, None) == 1
    assert rules(None, 1, 1, C.byref(none), p, p) == 1 and rules(p, 1, 1, None, p, p) == 1
    assert rules(p, 1, 1, C.byref(none), None, None) == 1
    assert rules(p, -1, 1, C.byref(none), p, p) == 1 and rules(p, 1, 0, C.byref(none), p, p) == 1
    assert rules(p, 65536, 1, C.byref(none), p, p) == 3 and rules(p, 1, (1 << 28) + 1, C.byref(none), p, p) == 3
    for count, first in (("n_rules", "rules"), ("n_history", "history"), ("n_biases", "bias_tokens"), ("n_masks", "masks")):
        for n, more in ((-1, {}), (1, {})) + (((1, {first: p}),) if first in ("bias_tokens", "masks") else ()):
            assert rules(p, 1, 1, C.byref(sq.LogitsParams(**{count: n}, **more)), p, p) == 1
    for name in ("rules", "history", "bias_tokens", "bias_values", "masks", "mask_ids", "tokens"):
        assert rules(p, 1, 1, C.byref(sq.LogitsParams(**{name: p + 2})), p, p) == 1
    assert rules(p + 1, 1, 1, C.byref(none), p, p) == 1 and rules(p, 1, 1, C.byref(none), p + 2, p) == 1
    assert rules(p, 1, 1, C.byref(none), p, p + 3) == 1


def test_parents_are_counted():
    class Batch(sq.PageBatch):
        def __init__(self):
            self.handle = None

    for seqs, rows, parents in (([0], [1, 2], [0]), ([0], [2], [-1]), ([0, 1], [1, 1], [-1, -1, -1])):
        with pytest.raises(sq.SllmError) as e:
            Batch().begin_tree(seqs, rows, parents)
        assert e.value.status == 1


@pytest.mark.parametrize("parents", [np.array([-1.0, 0.5]), np.zeros((2, 2), np.int32), np.zeros((2, 0), np.int32)])
def test_arrays_of_other_kinds_are_refused(parents):
    with pytest.raises(TypeError):
        sq._ints(parents)


@pytest.mark.parametrize("kind", [np.int32, np.int64, np.uint8])
def test_arrays_of_integers(kind):
    assert sq._ints(np.arange(12, dtype=kind)[::3])[:4] == [0, 3, 6, 9]
    assert len(sq._ints(list(np.arange(3, dtype=kind)))) == 3
    sq._ints(np.array([]))


def test_a_rule_has_the_headers_layout():
    assert sq.LOGITS_RULE.itemsize == 32 and sq.LOGITS_RULE.isalignedstruct is False
    assert [sq.LOGITS_RULE.fields[n][1] for n in sq.LOGITS_RULE.names] == list(range(0, 32, 4))
    assert np.zeros(1, sq.LOGITS_RULE).view(np.int32).size == 8


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="checks the no-GPU error path")
def test_no_gpu_is_a_device_error():
    i = (C.c_int * 4)()
    with pytest.raises(sq.SllmError) as e:
        sq.logits_rules_dev(C.addressof(i), 1, 4, sq.LogitsParams(), 0, C.addressof(i))
    assert e.value.status == 4
