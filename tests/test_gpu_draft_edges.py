"""GPU tests of the operators of drafted tokens where calls are refused, or are captured and meet other steps."""
from __future__ import annotations

import pytest
import torch

import sllm_qmm as sq

pytestmark = pytest.mark.gpu


def test_captured_calls_of_too_many_sequences():
    """Captured paths and moves launch for max_seqs: refused where a launch has too few threads, taken below."""
    cache = sq.PageCache(1, 1, 8, 16, 4)
    s = cache.add()
    x = torch.zeros(64, dtype=torch.int32, device="cuda")
    p = x.data_ptr()
    for most, status in ((1 << 24, 3), (64, 0)):
        batch = sq.PageBatch(cache, 1, most, 16)
        batch.begin_tree([s], [2], [-1, 0])
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            y = x * 2
            for f in (lambda: sq.page_accept_dev(batch, p, p, p, p, p, st.cuda_stream),
                      lambda: sq.page_keep_dev(batch, p, st.cuda_stream)):
                try:
                    f()
                    got = 0
                except sq.SllmError as e:
                    got = e.status
                assert got == status
        torch.cuda.synchronize()
        del g, y
        # eager calls are of the step's sequences
        t = torch.zeros(2, dtype=torch.int32, device="cuda")
        kept, counts, after = (torch.full((2,), -7, dtype=torch.int32, device="cuda") for _ in range(3))
        sq.page_accept_dev(batch, t.data_ptr(), t.data_ptr(), kept.data_ptr(), counts.data_ptr(), after.data_ptr())
        sq.page_keep_dev(batch, kept.data_ptr())
        torch.cuda.synchronize()
        assert kept.tolist() == [0, 1] and counts.tolist() == [2, -7] and after.tolist() == [0, -7]
        cache.truncate(s, 0)


def test_a_refused_capture_leaves_the_batch_free_to_grow():
    """Rules whose candidates need more workspace than may be had record nothing: the batch's steps may grow afterwards."""
    rows, v = 60000, 9001  # (three chunks of 8 bytes a row: 1.4 MB)
    cache = sq.PageCache(1, 1, 8, 16, 60000)
    batch = sq.PageBatch(cache, 1, 1, rows)
    s = cache.add()
    batch.begin_tree([s], [1], [-1])
    x = torch.zeros(64, dtype=torch.int32, device="cuda")
    p = x.data_ptr()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    sq.set_param("workspace_max_mb", 1)
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            y = x * 2
            try:
                sq.logits_rules_dev(p, rows, v, sq.LogitsParams(), 0, p, batch, st.cuda_stream)
                status = 0
            except sq.SllmError as e:
                status = e.status
    finally:
        sq.set_param("workspace_max_mb", 0)
    torch.cuda.synchronize()
    assert status == 5
    del g, y
    cache.extend(s, 16 * 59000)
    batch.begin_tree([s], [1], [-1])
