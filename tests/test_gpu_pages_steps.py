"""GPU tests of a batch's steps where calls are refused, inputs are lopsided or launches take many pieces: against the
formulas in 64 bits, with the bounds of test_gpu_pages.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import sllm_qmm as sq
from test_gpu_pages import NP, Model, Pools, attention64, batch_of, check_step

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


@pytest.mark.parametrize("gap", [8, 11, 14, 17])
@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("prefix,owns,news", [(0, [450, 300], [1, 1]), (330, [3] * 20, [1] * 20), (200, [1, 30], [70, 20])])
def test_small_weights_behind_a_large_one(prefix, owns, news, dt, gap):
    """Position 0's score is `gap` nats above hundreds of others, and its V is small: what those add is most of the
    output, or a share of it that fp32 holds. Few rows (a workgroup's waves have tiles of their own), rows of 20
    sequences on a prefix and rows of prompts (tiles for all waves). The values' weights of f16 caches are within 2^-23 of
    themselves or 2^-38 of the largest: the latter, times |v|, is added to the bounds of test_gpu_pages."""
    rng = np.random.default_rng(gap)
    H, KV, dk = 8, 2, 64
    m = Model(H, KV, dk, 0, rng)
    cache = sq.PageCache(1, KV, dk, 16, 300, dt)
    pools = Pools(cache)
    base = cache.add()
    seqs = []

    def more(s, n):
        at = cache.length(s)
        cache.extend(s, n)
        K, V = rng.normal(size=(1, n, KV, dk)) * 0.3, np.abs(rng.normal(size=(1, n, KV, dk))) + 0.5
        K[..., 0] = 0
        if at == 0 and n:
            K[0, 0], V[0, 0] = 0, 1e-3 * V[0, 0]
            K[0, 0, :, 0] = gap
        if n:
            pools.write(s, at, K.astype(NP[dt]), V.astype(NP[dt]))

    more(base, prefix)
    for o in owns:
        seqs += cache.fork(base, prefix, 1)
        more(seqs[-1], o)
    n = sum(news)
    batch = sq.PageBatch(cache, H, len(seqs), n)
    batch.begin(seqs, news)
    (q, k, v), _ = inputs(m, n, rng)
    q, k, v = 0.5 * q, 0.3 * k, np.abs(v) + np.float32(0.5)
    q[:, ::dk], k[:, ::dk] = dk ** 0.5, 0
    out = attend(batch, m, [torch.from_numpy(a).cuda() for a in (q, k, v)], n)
    host, at = pools.host(), 0
    for s, c in zip(seqs, news):
        pos = np.arange(cache.length(s) - c, cache.length(s))
        K, V = (a[0].astype(np.float64) for a in pools.read(s, host))
        qr, qs = m.row(q[at:at + c], H, None, None, pos)
        for h in range(H):
            o, b = attention64(qr[:, h], qs[:, h], K[:, h // 4], V[:, h // 4], pos, dk ** -0.5)
            floor = np.stack([2.0 ** -38 * V[:p + 1, h // 4].sum(0) for p in pos])
            got = out[at:at + c, h * dk:(h + 1) * dk]
            worst = (np.abs(got - o) / (b + floor)).max()
            assert worst <= 1, (s, h, worst, np.abs(got / o - 1).max())
        at += c


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("dk", [64, 192])
def test_workgroups_that_take_several_pieces(dk, dt):
    """A captured launch has 1024 workgroups whatever the step: steps of more pieces, of blocks of one row, of up to 32
    and of more, in one replay; each replayed twice, with the same bits."""
    rng = np.random.default_rng(dk)
    H = KV = 32
    m = Model(H, KV, dk, dk // 2, rng)
    cache = sq.PageCache(1, KV, dk, 16, 260, dt)
    pools = Pools(cache)
    seqs = batch_of(cache, pools, 150, [3, 40, 9, 170] * 8, rng)
    batch = sq.PageBatch(cache, H, 32, 500)
    st = torch.cuda.Stream()
    d = [torch.zeros(500, h * dk, device="cuda") for h in (H, KV, KV)]
    out = torch.zeros(500, H * dk, device="cuda")
    batch.begin(seqs, [1] * 31 + [400], st.cuda_stream)  # (the buffer's size)
    batch.begin(seqs[:1], [1], st.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        sq.page_attention_dev(batch, 0, m.params, *(t.data_ptr() for t in d), out.data_ptr(), st.cuda_stream)
    for i, s in enumerate(seqs):  # (rows that no attention call wrote)
        cache.truncate(s, 150 + [3, 40, 9, 170][i % 4])
    for rows in ([1, 20, 1, 70, 2, 33, 1, 40] + [1] * 24, [1] * 32, [1, 1, 65, 1] * 4 + [1, 17, 1, 1] * 4):
        n = sum(rows)
        batch.begin(seqs, rows, st.cuda_stream)
        before = pools.host()
        host, dev = inputs(m, n, rng)
        for t, a in zip(d, dev):
            t[:n] = a
        bits = []
        for _ in range(2):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            bits.append(out.cpu().numpy())
        check_step(cache, pools, m, seqs, rows, *host, bits[0], before, 0)
        assert np.array_equal(bits[0].view(np.int32), bits[1].view(np.int32))
