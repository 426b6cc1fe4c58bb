"""GPU tests of a batch's steps where calls are refused, inputs are lopsided or launches take many pieces: against the
formulas in 64 bits, with the bounds of test_gpu_pages.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import sllm_qmm as sq
from test_gpu_pages import Model, Pools, batch_of, check_step

pytestmark = pytest.mark.gpu


def inputs(m, n, rng):
    q, k, v = (rng.normal(size=(n, h * m.dk)).astype(np.float32) for h in (m.H, m.KV, m.KV))
    return (q, k, v), [torch.from_numpy(a).cuda() for a in (q, k, v)]


def attend(batch, m, d, n, stream=0):
    out = torch.full((n + 1, m.H * m.dk), float("nan"), device="cuda")
    torch.cuda.synchronize()
    sq.page_attention_dev(batch, 0, m.params, *(t.data_ptr() for t in d), out.data_ptr(), stream)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def test_a_refused_step_leaves_the_one_before_it():
    """Refused for pages, and of so many rows that the batch would have needed more room for it."""
    rng = np.random.default_rng(1)
    m = Model(8, 2, 64, 32, rng)
    cache = sq.PageCache(1, 2, 64, 16, 60, "f32")
    pools = Pools(cache)
    seqs = batch_of(cache, pools, 200, [3, 90], rng)
    batch = sq.PageBatch(cache, 8, 2, 4000)
    batch.begin(seqs, [2, 5])
    before, vacant = pools.host(), cache.vacant()
    for _ in range(2):
        with pytest.raises(sq.SllmError) as e:
            batch.begin(seqs, [3500, 1])
        assert e.value.status == 5
        assert cache.vacant() == vacant and [cache.length(s) for s in seqs] == [205, 295]
    host, d = inputs(m, 7, rng)
    out = attend(batch, m, d, 7)
    check_step(cache, pools, m, seqs, [2, 5], *host, out, before, 0)
