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


def test_a_sequence_next_to_the_longest():
    """2^31 - 1000 rows, a page table of 8 million entries: every score is 0, so each output is the mean of V. V is 1, and 2
    in the last 3 million rows (a part of the last piece): the waves' sums are whole numbers below 2^24 and exact; the
    merge of 205 pieces rounds twice for each, the sums of values and of weights, and a few times behind it."""
    rows, more = 2 ** 31 - 1000, 3_000_000
    cache = sq.PageCache(1, 1, 8, 256, (2 ** 31 - 512) // 256 + 1, "f16")
    pools = Pools(cache, fill=0.0)
    s = cache.add()
    cache.extend(s, rows)
    v = pools.t[1].view(-1, 8)
    v.fill_(1.0)
    v[rows - more:rows] = 2.0
    m = Model(2, 1, 8, 0, np.random.default_rng(0))
    batch = sq.PageBatch(cache, 2, 1, 3)
    batch.begin([s], [3])
    d = [torch.zeros(3, 16, device="cuda"), torch.zeros(3, 8, device="cuda"), torch.full((3, 8), 2.0, device="cuda")]
    out = attend(batch, m, d, 3)
    for r in range(3):
        n = rows + r + 1
        want = (n + more + r + 1) / n
        assert (np.abs(out[r] - want) <= want * (2 * 205 + 16) * 2.0 ** -24).all(), (r, out[r] - want)
