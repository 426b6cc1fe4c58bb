"""The entry points of batches of sequences on the CPU: bad arguments are refused with status codes before a GPU
is touched."""
import ctypes as C
import os

import pytest

import sllm_qmm as sq


def test_bad_arguments_need_no_device():
    lib, h, n = sq.lib(), C.c_void_p(), C.c_int()
    create = lambda *a: lib.sllm_page_cache_create(*a, C.byref(h))  # noqa: E731
    assert lib.sllm_page_cache_create(1, 1, 64, 16, 4, 0, None) == 1
    assert create(0, 1, 64, 16, 4, 0) == 1 and create(1, 0, 64, 16, 4, 0) == 1 and create(1, 1, 64, 16, 0, 0) == 1
    assert create(1, 1, 60, 16, 4, 0) == 3     # d_k % 8
    assert create(1, 1, 264, 16, 4, 0) == 3    # d_k > 256
    for rows in (0, 8, 24, 512):
        assert create(1, 1, 64, rows, 4, 0) == 3
    assert create(1, 1, 64, 16, 4, 2) == 1     # no such type
    assert create(32768, 1, 64, 16, 4, 0) == 3 and create(1, 65536, 64, 16, 4, 0) == 3
    assert create(32767, 65535, 256, 256, 2 ** 31 - 1, 0) == 5 and not h
    i = (C.c_int * 1)()
    for call in (lambda: lib.sllm_page_cache_data(None, C.byref(h), C.byref(h)),
                 lambda: lib.sllm_page_cache_vacant(None, C.byref(n)), lambda: lib.sllm_page_seq_add(None, C.byref(n)),
                 lambda: lib.sllm_page_seq_fork(None, 0, 0, 1, i), lambda: lib.sllm_page_seq_copy(None, 0, 0, 1, i, None),
                 lambda: lib.sllm_page_seq_extend(None, 0, 1, None), lambda: lib.sllm_page_seq_truncate(None, 0, 0),
                 lambda: lib.sllm_page_seq_free(None, i, 1), lambda: lib.sllm_page_seq_length(None, 0, C.byref(n)),
                 lambda: lib.sllm_page_seq_tables(None, i, 1, i, 1, None),
                 lambda: lib.sllm_page_cache_compact(None, None, None),
                 lambda: lib.sllm_page_batch_create(None, 8, 1, 1, C.byref(h)),
                 lambda: lib.sllm_page_batch_begin(None, i, i, 1, None),
                 lambda: lib.sllm_page_attention_dev(None, 0, C.byref(sq.AttnParams()), i, i, i, i, None)):
        assert call() == 1
    lib.sllm_page_cache_destroy(None)
    lib.sllm_page_batch_destroy(None)
    make = lambda *a: lib.sllm_lora_set_create(*a, C.byref(h))  # noqa: E731
    assert make(0, 32, 1, 1, 0) == 1 and make(1, 0, 1, 1, 0) == 1 and make(1, 32, 0, 1, 0) == 1 and make(1, 32, 1, 0, 0) == 1
    assert make(1, 33, 1, 1, 0) == 3 and make(1, 32, 1, 257, 0) == 3 and make(1, 32, 1, 1, 3) == 1
    assert make(2 ** 24, 32, 1, 256, 0) == 3
    assert lib.sllm_lora_set_create(1, 32, 1, 1, 0, None) == 1
    assert lib.sllm_lora_set_load(None, 0, 1, i, i, C.c_float(1)) == 1
    assert lib.sllm_lora_add_dev(None, i, 1, i, i, i, None) == 1
    lib.sllm_lora_set_destroy(None)


def test_unknown_types_are_refused():
    for make in (lambda: sq.PageCache(1, 1, 64, 16, 4, "bf16"), lambda: sq.LoraSet(64, 64, 1, 1, "f64")):
        with pytest.raises(sq.SllmError) as e:
            make()
        assert e.value.status == 1


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="checks the no-GPU error path")
def test_no_gpu_is_a_device_error():
    for make in (lambda: sq.PageCache(1, 1, 64, 16, 4), lambda: sq.LoraSet(64, 64, 1, 1)):
        with pytest.raises(sq.SllmError) as e:
            make()
        assert e.value.status == 4
