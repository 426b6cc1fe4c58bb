"""GPU tests of the page cache (sllm_page_cache_*, sllm_page_seq_*) and of the attention section of a batch
over it (sllm_page_attention_dev), against plain implementations: the bookkeeping against a small model of its
rules, the attention against the formulas in 64 bits.

Attention, what must agree and how closely (u = 2^-24):
* the appended v rows: the bias add (one rounding) and the rounding to the cache's type; the appended k rows:
  bias, norm and rotation in float32 take at most 12 roundings of values no larger than the element's rotated
  pair, then the rounding to the cache's type (2^-11 of the value for f16; below its normal range 2^-25);
* the output, given the rows as the pages hold them: a score is scale * q . k with q off by at most 12 u of its
  pair and d_k products and sums, each rounded once: ds = (d_k + 40) u scale sum_d |pair(q)_d k_d| (splitting q into
  two f16 parts loses 4 u of it, counted in the 40). A weight e = exp(s - m) is then off by
  ds + (4 + 4 |s - m|) u relatively (the argument's and the function's roundings, two f16 parts), the sum of the
  weights by the weights' mean of that, and adding up kv of them, and kv products with v, by 2 kv u:
  |out - exact| <= sum_j p_j |v_j| (delta_j + sum_i p_i delta_i + (2 kv + 64) u).
Rows and pages that a call does not name keep their bits; they hold NaN here, so that any use of them shows.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import sllm_qmm as sq

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NP = {"f32": np.float32, "f16": np.float16}
BITS = {"f32": np.uint32, "f16": np.uint16}


class Pools:
    """A cache's pools as tensors and arrays."""

    def __init__(self, cache: sq.PageCache, fill=float("nan")):
        self.cache, self.dt = cache, cache.dtype
        shape = (cache.n_layers, cache.n_pages, cache.n_kv_heads, cache.page_rows, cache.d_k)
        self.t = []
        for p in cache.data():
            class _Mem:
                pass
            m = _Mem()
            m.__cuda_array_interface__ = {"shape": shape, "typestr": "<f4" if self.dt == "f32" else "<f2",
                                          "data": (p, False), "version": 2}
            self.t.append(torch.as_tensor(m, device="cuda"))
            self.t[-1].fill_(fill)

    def host(self):
        torch.cuda.synchronize()
        return [t.cpu().numpy() for t in self.t]

    def where(self, seq, rows):
        """Page and slot of a sequence's rows."""
        tab = self.cache.tables([seq])[0]
        r = np.asarray(rows)
        return tab[r // self.cache.page_rows], r % self.cache.page_rows

    def write(self, seq, first, K, V):
        """K, V: (layers, rows, heads, d_k) into rows first .. of the sequence."""
        pg, sl = (torch.from_numpy(a.astype(np.int64)).cuda() for a in self.where(seq, np.arange(first, first + K.shape[1])))
        for t, x in zip(self.t, (K, V)):
            x = torch.from_numpy(x).cuda()
            for layer in range(t.shape[0]):
                t[layer][pg, :, sl] = x[layer]

    def read(self, seq, host=None):
        """The sequence's K and V: (layers, rows, heads, d_k)."""
        n = self.cache.length(seq)
        pg, sl = self.where(seq, np.arange(n))
        return [h[:, pg, :, sl].swapaxes(0, 1) if n else h[:, :0, :, 0] for h in (host or self.host())]


class Model:
    def __init__(self, H, KV, dk, half, rng, bias=False, qk=False):
        self.H, self.KV, self.dk, self.half, self.eps = H, KV, dk, half, 1e-5
        self.freqs = np.array([1.0 / math.pow(10000.0, 2.0 * i / max(2 * half, 1)) for i in range(half)], np.float32)
        f = lambda *s: rng.normal(size=s).astype(np.float32)  # noqa: E731
        self.qb, self.kb, self.vb = (f(H * dk - 5), f(KV * dk + 3), f(KV * dk)) if bias else (None,) * 3
        self.qn, self.kn = (1 + 0.2 * f(dk), 1 + 0.2 * f(dk)) if qk else (None, None)
        self.keep = {n: torch.from_numpy(a).cuda() for n, a in
                     (("f", self.freqs), ("qb", self.qb), ("kb", self.kb), ("vb", self.vb), ("qn", self.qn),
                      ("kn", self.kn)) if a is not None and a.size}
        p = lambda n: self.keep[n].data_ptr() if n in self.keep else None  # noqa: E731
        n = lambda a: 0 if a is None else a.size  # noqa: E731
        self.params = sq.AttnParams(n_heads=H, n_kv_heads=KV, d_k=dk, rope_half_dim=half, rope_freqs=p("f"),
                                    q_bias=p("qb"), q_bias_len=n(self.qb), k_bias=p("kb"), k_bias_len=n(self.kb),
                                    v_bias=p("vb"), v_bias_len=n(self.vb), q_norm_w=p("qn"), k_norm_w=p("kn"),
                                    norm_eps=self.eps)

    def row(self, x, heads, bias, nw, pos):
        """(rows, heads * d_k) -> rotated rows in 64 bits and, per element, its pair's size."""
        x = x.astype(np.float64).copy()
        if bias is not None:
            n = min(len(bias), x.shape[1])
            x[:, :n] += bias[:n]
        x = x.reshape(len(x), heads, self.dk)
        if nw is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + self.eps) * nw
        ang = (self.freqs[None] * np.asarray(pos, np.float32)[:, None]).astype(np.float64)[:, None]
        y, h = x.copy(), 2 * self.half
        a, b = x[..., 0:h:2], x[..., 1:h:2]
        y[..., 0:h:2], y[..., 1:h:2] = a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)
        size = np.abs(y)
        size[..., 0:h:2] = size[..., 1:h:2] = np.hypot(a, b)
        return y, size


def attention64(q, qs, K, V, last, scale):
    """One head: q, qs (rows, dk), K, V (kv, dk); row r sees positions 0 .. last[r]. Output and its bound."""
    dk = q.shape[1]
    s = q @ K.T * scale
    ds = (dk + 40) * U * scale * (qs @ np.abs(K).T)
    out, bound = np.empty_like(q), np.empty_like(q)
    for r in range(len(q)):
        n = last[r] + 1
        m = s[r, :n].max()
        p = np.exp(s[r, :n] - m)
        p /= p.sum()
        d = ds[r, :n] + (4 + 4 * np.abs(s[r, :n] - m)) * U
        out[r] = p @ V[:n]
        bound[r] = (p * (d + p @ d + (2 * n + 64) * U)) @ np.abs(V[:n])
    return out, bound + 1e-30


def run_step(cache, pools, m, batch, seqs, rows, rng, layer=0, stream=0, scale_q=1.5):
    """begin + one attention call, checked whole."""
    before_len = [cache.length(s) for s in seqs]
    batch.begin(seqs, rows, stream)
    assert [cache.length(s) for s in seqs] == [a + b for a, b in zip(before_len, rows)]
    before = pools.host()
    R = sum(rows)
    q = (rng.normal(size=(R, m.H * m.dk)) * scale_q).astype(np.float32)
    k = rng.normal(size=(R, m.KV * m.dk)).astype(np.float32)
    v = rng.normal(size=(R, m.KV * m.dk)).astype(np.float32)
    d = [torch.from_numpy(a).cuda() for a in (q, k, v)]
    out = torch.full((R + 1, m.H * m.dk), float("nan"), device="cuda")
    torch.cuda.synchronize()
    sq.page_attention_dev(batch, layer, m.params, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), out.data_ptr(), stream)
    torch.cuda.synchronize()
    check_step(cache, pools, m, seqs, rows, q, k, v, out.cpu().numpy(), before, layer)
    for t, a in zip(d, (q, k, v)):
        assert np.array_equal(t.cpu().numpy(), a)
    return out


def check_step(cache, pools, m, seqs, rows, q, k, v, out, before, layer):
    after = pools.host()
    R, rep, dt = sum(rows), m.H // m.KV, cache.dtype
    assert np.isnan(out[R:]).all()
    want = [b.copy() for b in before]
    half = 2.0 ** -11 if dt == "f16" else 0.0
    at = 0
    for s, n in zip(seqs, rows):
        if not n:
            continue
        total = cache.length(s)
        pos = np.arange(total - n, total)
        pg, sl = pools.where(s, pos)
        kr, ks = m.row(k[at:at + n], m.KV, m.kb, m.kn, pos)
        vr = v[at:at + n].reshape(n, m.KV, m.dk).astype(np.float64)
        if m.vb is not None:
            vr = vr + m.vb.reshape(m.KV, m.dk)
        for i, (x, size) in enumerate(((kr, 12 * U * ks), (vr, U * np.abs(vr)))):
            got = after[i][layer][pg, :, sl].astype(np.float64)
            assert (np.abs(got - x) <= size + half * (np.abs(x) + size) + (2.0 ** -25 if half else 0)).all()
            want[i][layer][pg, :, sl] = after[i][layer][pg, :, sl]
        K, V = (a[layer].astype(np.float64) for a in pools.read(s, after))
        qr, qs = m.row(q[at:at + n], m.H, m.qb, m.qn, pos)
        for h in range(m.H):
            o, b = attention64(qr[:, h], qs[:, h], K[:, h // rep], V[:, h // rep], pos, 1 / math.sqrt(m.dk))
            got = out[at:at + n, h * m.dk:(h + 1) * m.dk].astype(np.float64)
            bad = ~(np.abs(got - o) <= b)
            assert not bad.any(), (s, h, np.argwhere(bad)[:3], got[bad][:3], o[bad][:3], b[bad][:3])
        at += n
    # nothing else moved
    for w, a in zip(want, after):
        assert np.array_equal(w.view(BITS[dt]), a.view(BITS[dt]))


def fill(cache, pools, seq, first, n, rng):
    """n more rows with contents."""
    cache.extend(seq, n)
    shape = (cache.n_layers, n, cache.n_kv_heads, cache.d_k)
    if n:
        pools.write(seq, first, *(rng.normal(size=shape).astype(NP[cache.dtype]) for _ in range(2)))


def batch_of(cache, pools, prefix, owns, rng, tree=False):
    """Sequences behind a shared prefix (tree: every second one forks off the one before it)."""
    base = cache.add()
    fill(cache, pools, base, 0, prefix, rng)
    seqs = []
    for i, o in enumerate(owns):
        if tree and i % 2:
            parent = seqs[-1]
            seqs += cache.fork(parent, cache.length(parent), 1)
        else:
            seqs += cache.fork(base, prefix, 1)
        fill(cache, pools, seqs[-1], cache.length(seqs[-1]), o, rng)
    cache.free([base])
    return seqs


CASES = [
    # H, KV, dk, half, type, page rows, prefix, own rows, new rows
    (9, 3, 64, 32, "f32", 16, 0, [0], [1]),                    # the first token of a sequence
    (9, 3, 64, 32, "f32", 16, 0, [130, 0, 15, 16, 17], [1] * 5),
    (4, 4, 64, 32, "f16", 16, 0, [1, 63], [1, 1]),
    (32, 8, 128, 64, "f32", 32, 0, [300, 5, 64, 127, 128, 129], [1] * 6),
    (32, 8, 128, 64, "f16", 64, 200, [3, 0, 70, 1, 64], [1] * 5),  # a tail page shared and copied
    (32, 8, 128, 64, "f16", 64, 1024, [1] * 20, [1] * 20),
    (32, 4, 128, 64, "f32", 64, 640, [33] * 9, [1] * 9),         # 8 q heads per kv head
    (8, 1, 256, 128, "f32", 16, 100, [40, 1, 0], [1, 1, 1]),
    (8, 1, 256, 128, "f16", 256, 700, [40, 1, 0], [1, 2, 3]),
    (16, 16, 80, 40, "f16", 32, 257, [5, 9], [1, 1]),           # head sizes between the kernel's blocks
    (10, 2, 72, 20, "f32", 16, 99, [5, 9, 31], [1, 7, 0]),      # partly rotated; a sequence without rows
    (6, 2, 8, 4, "f16", 16, 40, [0, 3], [2, 1]),                # the smallest head
    (6, 2, 8, 0, "f32", 128, 300, [0, 3], [5, 1]),              # no rotation
    (6, 2, 200, 100, "f32", 16, 65, [2, 40], [3, 1]),
    (32, 8, 128, 64, "f16", 64, 130, [0, 1, 7], [65, 1, 130]),   # prompts of several lengths behind a prefix
    (32, 8, 128, 64, "f32", 16, 0, [0, 0], [100, 33]),
    (12, 12, 64, 32, "f16", 128, 300, [10], [70]),
    (7, 1, 96, 48, "f32", 64, 200, [9, 80], [19, 1]),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("extras", [False, True])
def test_step_matches_the_formulas(case, extras):
    H, KV, dk, half, dt, page, prefix, owns, news = CASES[case]
    rng = np.random.default_rng(100 * case + extras)
    m = Model(H, KV, dk, half, rng, bias=extras, qk=extras)
    pages = -(-prefix // page) + sum(-(-(o + n) // page) + 2 for o, n in zip(owns, news)) + 1
    cache = sq.PageCache(2, KV, dk, page, pages, dt)
    pools = Pools(cache)
    seqs = batch_of(cache, pools, prefix, owns, rng)
    batch = sq.PageBatch(cache, H, len(seqs) + 1, sum(news) + 2)
    run_step(cache, pools, m, batch, seqs, news, rng, layer=1)
    # a second step of the same batch: one row each, in another order
    order = list(rng.permutation(len(seqs)))
    run_step(cache, pools, m, batch, [seqs[i] for i in order], [1] * len(order) if sum(news) + 2 >= len(order) else news, rng,
             layer=1)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_two_levels_of_sharing_and_a_fork_in_mid_page(dt):
    rng = np.random.default_rng(5)
    m = Model(32, 8, 128, 64, rng)
    cache = sq.PageCache(1, 8, 128, 32, 120, dt)
    pools = Pools(cache)
    seqs = batch_of(cache, pools, 333, [200, 3, 170, 0, 1, 40], rng, tree=True)
    other = batch_of(cache, pools, 65, [1, 2], rng)  # a second prefix in the same batch
    batch = sq.PageBatch(cache, 32, 8, 40)
    for step in range(3):
        run_step(cache, pools, m, batch, seqs[:3] + other + seqs[3:], [1, 1, 2 * step, 1, 3, 1, 0, 1], rng)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_long_context(dt):
    # more positions than one workgroup takes, for few and for many rows
    rng = np.random.default_rng(6)
    m = Model(8, 2, 128, 64, rng)
    cache = sq.PageCache(1, 2, 128, 64, 330, dt)
    pools = Pools(cache)
    seqs = batch_of(cache, pools, 9000, [2500] + [7] * 3, rng)
    batch = sq.PageBatch(cache, 8, 4, 64)
    run_step(cache, pools, m, batch, seqs, [1, 1, 1, 1], rng)
    run_step(cache, pools, m, batch, seqs, [1, 40, 3, 1], rng)


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), -float("inf")])
def test_values_that_a_row_does_not_see(dt, bad):
    # position 70's V holds a non-finite element: rows before it are untouched, rows from it on hold it there;
    # everything behind the sequence's end is NaN anyway
    rng = np.random.default_rng(8)
    H, KV, dk = 8, 2, 128
    m = Model(H, KV, dk, 64, rng)
    cache = sq.PageCache(1, KV, dk, 16, 12, dt)
    pools = Pools(cache)
    s = cache.add()
    fill(cache, pools, s, 0, 50, rng)
    batch = sq.PageBatch(cache, H, 1, 64)
    batch.begin([s], [40])
    q, k, v = (rng.normal(size=(40, n * dk)).astype(np.float32) for n in (H, KV, KV))
    v[20, 5] = bad  # position 70, kv head 0, element 5
    d = [torch.from_numpy(a).cuda() for a in (q, k, v)]
    out = torch.empty(40, H * dk, device="cuda")
    sq.page_attention_dev(batch, 0, m.params, *(t.data_ptr() for t in d), out.data_ptr())
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(40, H, dk)
    v[20, 5] = 0.0
    K, V = (a[0].astype(np.float64) for a in pools.read(s))
    V[70, 0, 5] = 0.0
    qr, qs = m.row(q, H, None, None, np.arange(50, 90))
    for h in range(H):
        o, b = attention64(qr[:, h], qs[:, h], K[:, h // 4], V[:, h // 4], np.arange(50, 90), 1 / math.sqrt(dk))
        g = got[:, h].copy()
        if h < 4:
            hit = g[20:, 5].copy()
            assert np.isnan(hit).all() if math.isnan(bad) else (hit == np.float32(bad)).all()
            g[20:, 5] = o[20:, 5]
        assert (np.abs(g - o) <= b).all(), h


def test_scores_of_minus_infinity_and_large_values():
    # k of -inf against a positive q: those positions weigh nothing; a row that sees only such has no weights (NaN),
    # as the softmax's formula says; q far beyond f16's range is computed all the same
    rng = np.random.default_rng(9)
    H, KV, dk = 4, 1, 64
    m = Model(H, KV, dk, 0, rng)
    for dt in ("f32", "f16"):
        cache = sq.PageCache(1, KV, dk, 16, 40, dt)
        pools = Pools(cache)
        s = cache.add()
        K = np.zeros((1, 500, KV, dk), NP[dt])
        K[..., 1:] = rng.normal(size=(1, 500, KV, dk - 1))
        K[0, 100:400, 0, 0] = -np.inf
        V = rng.normal(size=K.shape).astype(NP[dt])
        cache.extend(s, 500)
        pools.write(s, 0, K, V)
        none = cache.add()
        cache.extend(none, 20)
        pools.write(none, 0, np.full((1, 20, KV, dk), -np.inf, NP[dt]), V[:, :20])
        batch = sq.PageBatch(cache, H, 2, 2)
        batch.begin([s, none], [1, 1])
        q = np.abs(rng.normal(size=(2, H * dk))).astype(np.float32)
        q[0] *= 1e-3 * 2.0 ** rng.integers(-4, 4, size=H).repeat(dk)
        q[0, :dk] = q[0, :dk] * 1e9
        k = np.full((2, KV * dk), -np.inf, np.float32)
        k[0] = rng.normal(size=dk) * 1e-3
        v = rng.normal(size=(2, KV * dk)).astype(np.float32)
        d = [torch.from_numpy(a).cuda() for a in (q, k, v)]
        out = torch.zeros(2, H * dk, device="cuda")
        sq.page_attention_dev(batch, 0, m.params, *(t.data_ptr() for t in d), out.data_ptr())
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        assert np.isnan(got[1]).all()
        Kd, Vd = (a[0, :, 0].astype(np.float64) for a in pools.read(s))
        see = np.r_[0:100, 400:501]
        for h in range(H):
            qh = q[0, h * dk:(h + 1) * dk].astype(np.float64)[None]
            o, b = attention64(qh, np.abs(qh), Kd[see], Vd[see], [len(see) - 1], 1 / math.sqrt(dk))
            assert (np.abs(got[0, h * dk:(h + 1) * dk] - o[0]) <= b[0] * (501 / len(see))).all()


def test_on_another_stream_and_in_a_graph():
    rng = np.random.default_rng(10)
    H, KV, dk = 32, 8, 128
    m = Model(H, KV, dk, 64, rng)
    cache = sq.PageCache(1, KV, dk, 64, 60, "f16")
    pools = Pools(cache)
    seqs = batch_of(cache, pools, 500, [3, 60, 100, 1], rng)
    batch = sq.PageBatch(cache, H, 4, 12)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    run_step(cache, pools, m, batch, seqs, [1, 1, 1, 1], rng, stream=st.cuda_stream)
    bufs = [torch.zeros(12, n * dk, device="cuda") for n in (H, KV, KV)]
    out = torch.full((12, H * dk), float("nan"), device="cuda")
    torch.cuda.synchronize()
    batch.begin(seqs, [1, 1, 1, 1], st.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        sq.page_attention_dev(batch, 0, m.params, *(t.data_ptr() for t in bufs), out.data_ptr(), st.cuda_stream)
    g.replay()  # the step that was begun for the capture
    # replays follow the batch's steps: other rows, other sequences, none at all
    for who, rows in ((seqs, [1, 1, 1, 1]), (seqs[1:3], [2, 5]), (seqs[::-1], [1, 0, 3, 1]), (seqs[:1], [12])):
        batch.begin(who, rows, st.cuda_stream)
        before = pools.host()
        q, k, v = (rng.normal(size=(sum(rows), n * dk)).astype(np.float32) for n in (H, KV, KV))
        for t, a in zip(bufs, (q, k, v)):
            t[:sum(rows)] = torch.from_numpy(a).cuda()
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check_step(cache, pools, m, who, rows, q, k, v, out.cpu().numpy(), before, 0)
    before = pools.host()
    batch.begin(seqs, [0] * 4, st.cuda_stream)
    out.fill_(float("nan"))
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert torch.isnan(out).all()
    for a, b in zip(before, pools.host()):
        assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


def test_two_batches_of_one_cache():
    # a prompt's batch and a decode batch, their steps interleaved
    rng = np.random.default_rng(11)
    m = Model(8, 2, 64, 32, rng)
    cache = sq.PageCache(2, 2, 64, 16, 60, "f32")
    pools = Pools(cache)
    seqs = batch_of(cache, pools, 100, [1, 20], rng)
    new = cache.add()
    a, b = sq.PageBatch(cache, 8, 4, 8), sq.PageBatch(cache, 8, 1, 64)
    run_step(cache, pools, m, a, seqs, [1, 1], rng)
    run_step(cache, pools, m, b, [new], [50], rng)
    run_step(cache, pools, m, a, seqs + [new], [1, 2, 1], rng)
    cache.close()  # lives on with its batches
    b.close()
    a.close()


class Rules:
    """The cache's bookkeeping as its documentation states it."""

    def __init__(self, page, pages):
        self.page, self.held, self.seqs, self.ids = page, {}, {}, set()
        self.pages = pages

    def take(self):
        p = next(i for i in range(self.pages) if i not in self.held)
        self.held[p] = 1
        return p

    def drop(self, p):
        self.held[p] -= 1
        if not self.held[p]:
            del self.held[p]

    def add(self, tab=(), data=()):
        s = next(i for i in range(10 ** 6) if i not in self.seqs)
        self.seqs[s] = [list(tab), list(data)]
        return s

    def fork(self, s, rows):
        tab = self.seqs[s][0][:-(-rows // self.page)]
        for p in tab:
            self.held[p] += 1
        return self.add(tab, self.seqs[s][1][:rows])

    def copy(self, s, rows):
        return self.add([self.take() for _ in range(-(-rows // self.page))], self.seqs[s][1][:rows])

    def extend(self, s, marks):
        tab, data = self.seqs[s]
        if marks and len(data) % self.page and self.held[tab[-1]] > 1:
            p = self.take()
            self.drop(tab[-1])
            tab[-1] = p
        data += marks
        while len(tab) < -(-len(data) // self.page):
            tab.append(self.take())

    def truncate(self, s, rows):
        tab, data = self.seqs[s]
        del data[rows:]
        while len(tab) > -(-rows // self.page):
            self.drop(tab.pop())

    def free(self, s):
        for p in self.seqs.pop(s)[0]:
            self.drop(p)

    def compact(self):
        n = len(self.held)
        high, gaps = sorted(p for p in self.held if p >= n), (p for p in range(n) if p not in self.held)
        to = dict(zip(high, gaps))
        self.held = {to.get(p, p): c for p, c in self.held.items()}
        for q in self.seqs.values():
            q[0] = [to.get(p, p) for p in q[0]]
        return n


@pytest.mark.parametrize("page,dt,seed", [(16, "f32", 0), (16, "f16", 1), (32, "f32", 2), (64, "f16", 3)])
def test_bookkeeping_follows_its_rules(page, dt, seed):
    rng = np.random.default_rng(seed)
    pages, layers, KV, dk = 40, 3, 2, 8
    cache, r = sq.PageCache(layers, KV, dk, page, pages, dt), Rules(page, pages)
    pools, mark = Pools(cache), 0
    batch = sq.PageBatch(cache, 2 * KV, 8, 1000)
    for step in range(220):
        live = sorted(r.seqs)
        op = rng.choice(["add", "fork", "copy", "extend", "extend", "begin", "truncate", "free", "compact"])
        s = int(rng.choice(live)) if live else None
        room = pages - len(r.held)
        if op == "add" or s is None:
            if len(live) < 12:
                assert cache.add() == r.add()
        elif op in ("fork", "copy"):
            n = int(rng.integers(0, len(r.seqs[s][1]) + 1))
            count = int(rng.integers(0, 4))
            if len(live) < 12 and (op == "fork" or count * -(-n // page) <= room):
                got = getattr(cache, op)(s, n, count)
                assert got == [getattr(r, op)(s, n) for _ in range(count)]
        elif op in ("extend", "begin"):
            who = [s] if op == "extend" else [int(x) for x in rng.permutation(live)[:4]]
            n = [int(rng.integers(0, 3 * page)) for _ in who]
            if sum(-(-x // page) + 1 for x in n) <= room:
                at = [len(r.seqs[x][1]) for x in who]
                if op == "extend":
                    cache.extend(s, n[0])
                else:
                    batch.begin(who, n)
                for x, c in zip(who, n):
                    r.extend(x, list(range(mark, mark + c)))
                    mark += c
                for x, a, c in zip(who, at, n):
                    if c:
                        m = np.array(r.seqs[x][1][a:], np.float32) % 1999
                        K = np.broadcast_to(m[None, :, None, None], (layers, c, KV, dk)).astype(NP[dt])
                        pools.write(x, a, K, K + 1)
        elif op == "truncate":
            n = int(rng.integers(0, len(r.seqs[s][1]) + 1))
            cache.truncate(s, n)
            r.truncate(s, n)
        elif op == "free":
            cache.free([s])
            r.free(s)
        else:
            assert cache.compact() == r.compact()
        assert cache.vacant() == pages - len(r.held)
        live = sorted(r.seqs)
        if live:
            tab = cache.tables(live)
            assert [[p for p in t if p >= 0] for t in tab.tolist()] == [r.seqs[x][0] for x in live]
            assert [cache.length(x) for x in live] == [len(r.seqs[x][1]) for x in live]
        if step % 5 == 0:
            host = pools.host()
            for x in live:
                m = (np.array(r.seqs[x][1], np.float32) % 1999)[None, :, None, None]
                K, V = pools.read(x, host)
                assert (K == m).all() and (V == m + 1).all()


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_steps_one_after_the_other_without_waiting(dt):
    """Steps of one row and of hundreds in turn (more than the batch has staging memory for), nothing waited for between
    them: the same bits as step by step."""
    outs = []
    for wait in (True, False):
        rng = np.random.default_rng(3)
        m = Model(8, 2, 64, 32, rng)
        cache = sq.PageCache(1, 2, 64, 16, 400, dt)
        batch = sq.PageBatch(cache, 8, 40, 400)
        st = torch.cuda.Stream()
        seqs = [cache.add() for _ in range(40)]
        got, keep = [], []
        torch.cuda.synchronize()
        for i in range(14):
            rows = [1] if i % 3 == 0 else [1] * 40 if i % 3 == 1 else [9 + j % 3 for j in range(30)]
            n = sum(rows)
            d = [torch.from_numpy(rng.normal(size=(n, k * 64)).astype(np.float32)).cuda() for k in (8, 2, 2)]
            out = torch.empty(n, 8 * 64, device="cuda")
            if wait:
                torch.cuda.synchronize()
            else:
                st.wait_stream(torch.cuda.current_stream())
            batch.begin(seqs[:len(rows)], rows, st.cuda_stream)
            sq.page_attention_dev(batch, 0, m.params, *(t.data_ptr() for t in d), out.data_ptr(), st.cuda_stream)
            got.append(out)
            keep.append(d)
        torch.cuda.synchronize()
        outs.append([o.cpu().numpy() for o in got])
        assert all(np.isfinite(o).all() for o in outs[-1])
    for a, b in zip(*outs):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_refused_steps_change_nothing():
    cache = sq.PageCache(1, 2, 64, 16, 4, "f32")
    a, b = cache.add(), cache.add()
    cache.extend(a, 40)
    batch = sq.PageBatch(cache, 4, 2, 64)
    m = Model(4, 2, 64, 32, np.random.default_rng(0))
    x = torch.zeros(64, 256, device="cuda")
    p = x.data_ptr()

    def refused(status, f, *args):
        with pytest.raises(sq.SllmError) as e:
            f(*args)
        assert e.value.status == status, e.value
        assert cache.vacant() == 1 and cache.length(a) == 40 and cache.length(b) == 0

    refused(5, batch.begin, [a, b], [8, 17])   # one page is vacant, two are needed
    refused(5, cache.extend, b, 33)
    refused(5, cache.copy, a, 40, 1)
    refused(1, batch.begin, [a, a], [1, 1])    # a sequence twice
    refused(1, batch.begin, [a, 7], [1, 1])
    refused(1, batch.begin, [a, b], [1, -1])
    refused(1, batch.begin, [a, b, a], [1, 1, 1])
    refused(3, batch.begin, [a, b], [1, 64])   # more than max_rows
    refused(1, cache.fork, a, 41, 1)
    refused(1, cache.fork, 9, 0, 1)
    refused(1, cache.truncate, a, 41)
    refused(1, cache.truncate, a, -1)
    refused(1, cache.free, [a, a])
    refused(1, cache.free, [b, 5])
    refused(1, cache.length, 5)
    refused(1, cache.tables, [0, 5])
    refused(1, sq.page_attention_dev, batch, 0, m.params, p, p, p, p)  # no step yet
    batch.begin([a], [1])
    sq.page_attention_dev(batch, 0, m.params, p, p, p, p)
    with pytest.raises(sq.SllmError):
        sq.page_attention_dev(batch, 1, m.params, p, p, p, p)          # no such layer
    with pytest.raises(sq.SllmError):
        sq.page_attention_dev(batch, 0, m.params, p + 4, p, p, p)      # alignment
    wrong = Model(8, 2, 64, 32, np.random.default_rng(0))
    with pytest.raises(sq.SllmError):
        sq.page_attention_dev(batch, 0, wrong.params, p, p, p, p)      # another model
    for end in (lambda: cache.truncate(a, 3), lambda: cache.free([a])):
        end()
        with pytest.raises(sq.SllmError) as e:
            sq.page_attention_dev(batch, 0, m.params, p, p, p, p)      # the step has ended
        assert e.value.status == 1
        if cache.vacant() < 4:
            batch.begin([a], [1])
            sq.page_attention_dev(batch, 0, m.params, p, p, p, p)
    st = torch.cuda.Stream()
    b2 = cache.add()
    batch.begin([b2], [1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        y = x * 2
        for f, args in ((batch.begin, ([b2], [1], st.cuda_stream)), (cache.extend, (b2, 1, st.cuda_stream)),
                        (cache.copy, (b2, 1, 1, st.cuda_stream)), (cache.compact, (st.cuda_stream,))):
            with pytest.raises(sq.SllmError) as e:
                f(*args)
            assert e.value.status == 1
        sq.page_attention_dev(batch, 0, m.params, p, p, p, p, st.cuda_stream)
    with pytest.raises(sq.SllmError) as e:  # the captured call's buffers stay as they are
        big = sq.PageCache(1, 2, 64, 16, 60000, "f32")
        bb = sq.PageBatch(big, 4, 2, 64)
        s = big.add()
        bb.begin([s], [1])
        g2 = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g2, stream=st):
            sq.page_attention_dev(bb, 0, m.params, p, p, p, p, st.cuda_stream)
        big.extend(s, 16 * 59000)
        bb.begin([s], [1])
    assert e.value.status == 3
    torch.cuda.synchronize()
