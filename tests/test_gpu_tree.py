"""GPU tests of drafted trees over a page cache: the attention of a step begun with parents (sllm_page_batch_begin_tree),
the accepted paths (sllm_page_accept_dev) and the kept rows (sllm_page_keep_dev), against plain implementations.

The attention has the bound of test_gpu_pages (u = 2^-24), with the rows that a node sees in place of all up to its own:
masked scores are -inf, their weights exactly 0, so sums have no further terms. Accepted paths are whole numbers and
kept rows copies: both are exact, and rows that a call does not name keep their bits.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import sllm_qmm as sq
from test_gpu_pages import BITS, U, Model, Pools, attention64, batch_of, fill

pytestmark = pytest.mark.gpu


def tree(n, kind, rng):
    """Parents: chain, binary, random, random with several roots, wide."""
    r = np.arange(n)
    if kind == "chain":
        return (r - 1).tolist()
    if kind == "binary":
        return np.where(r == 0, -1, (r - 1) // 2).tolist()
    if kind == "wide":
        return np.where(r == 0, -1, np.maximum(0, r - max(1, n // 3))).tolist()
    return [-1 if i == 0 else int(rng.integers(-1 if kind == "forest" else 0, i)) for i in range(n)]


def path_of(parents, r):
    """Row r and its ancestors, the first last."""
    p = []
    while r >= 0:
        p.append(r)
        r = parents[r]
    return p


def attend(cache, m, batch, q, k, v, layer=0, stream=0):
    d = [torch.from_numpy(a).cuda() for a in (q, k, v)]
    out = torch.full((len(q) + 1, m.H * m.dk), float("nan"), device="cuda")
    torch.cuda.synchronize()
    sq.page_attention_dev(batch, layer, m.params, *(t.data_ptr() for t in d), out.data_ptr(), stream)
    torch.cuda.synchronize()
    assert torch.isnan(out[len(q):]).all()
    return out[:len(q)].cpu().numpy()


def check(cache, pools, m, seqs, parents, q, k, v, out, before, layer=0, see=None):
    """The step's rows in the pools, and every output against the formula. see: rows whose outputs are looked at."""
    after = pools.host()
    want = [b.copy() for b in before]
    half = 2.0 ** -11 if cache.dtype == "f16" else 0.0
    at, rep = 0, m.H // m.KV
    for s, par in zip(seqs, parents):
        n = len(par)
        if not n:
            continue
        total = cache.length(s)
        base = total - n
        paths = [path_of(par, r) for r in range(n)]
        pos = np.array([base + len(p) - 1 for p in paths])
        pg, sl = pools.where(s, np.arange(base, total))
        kr, ks = m.row(k[at:at + n], m.KV, m.kb, m.kn, pos)
        vr = v[at:at + n].reshape(n, m.KV, m.dk).astype(np.float64)
        if m.vb is not None:
            vr = vr + m.vb.reshape(m.KV, m.dk)
        for i, (x, size) in enumerate(((kr, 12 * U * ks), (vr, U * np.abs(vr)))):
            got = after[i][layer][pg, :, sl].astype(np.float64)
            fine = np.isfinite(x)
            near = np.abs(got - x) <= size + half * (np.abs(x) + size) + (2.0 ** -25 if half else 0)
            assert (near | ~fine).all()
            want[i][layer][pg, :, sl] = after[i][layer][pg, :, sl]
        K, V = (a[layer].astype(np.float64) for a in pools.read(s, after))
        qr, qs = m.row(q[at:at + n], m.H, m.qb, m.qn, pos)
        for r in range(n):
            if see is not None and at + r not in see:
                continue
            rows = np.append(np.arange(base), base + np.array(paths[r][::-1]))
            for h in range(m.H):
                o, b = attention64(qr[r:r + 1, h], qs[r:r + 1, h], K[rows, h // rep], V[rows, h // rep], [len(rows) - 1],
                                   1 / math.sqrt(m.dk))
                got = out[at + r, h * m.dk:(h + 1) * m.dk].astype(np.float64)
                assert (np.abs(got - o[0]) <= b[0]).all(), (s, r, h, np.abs(got - o[0]).max(), b[0].max())
        at += n
    for w, a in zip(want, after):
        assert np.array_equal(w.view(BITS[cache.dtype]), a.view(BITS[cache.dtype]))


def rows_of(m, n, rng, std=1.5):
    return ((rng.normal(size=(n, m.H * m.dk)) * std).astype(np.float32),
            *(rng.normal(size=(n, m.KV * m.dk)).astype(np.float32) for _ in range(2)))


def run_tree(cache, pools, m, batch, seqs, parents, rng, layer=0, stream=0, see=None):
    batch.begin_tree(seqs, [len(p) for p in parents], [x for p in parents for x in p], stream)
    before = pools.host()
    x = rows_of(m, sum(len(p) for p in parents), rng)
    out = attend(cache, m, batch, *x, layer, stream)
    check(cache, pools, m, seqs, parents, *x, out, before, layer, see)
    return out


SHAPES = [
    # heads, kv heads, d_k, page rows, type, prefix, rows of their own, (nodes, kind) of each sequence
    (4, 2, 64, 16, "f32", 0, [1], [(2, "forest")]),
    (9, 3, 64, 16, "f32", 0, [130], [(8, "binary")]),
    (8, 1, 64, 16, "f16", 0, [31, 16, 1], [(17, "random"), (33, "wide"), (1, "chain")]),
    (8, 8, 80, 32, "f16", 0, [15, 47], [(19, "random"), (40, "forest")]),
    (4, 4, 256, 16, "f32", 20, [3, 40], [(21, "random"), (5, "wide")]),
    (4, 1, 200, 64, "f16", 0, [70, 5], [(23, "binary"), (64, "random")]),
    (8, 2, 128, 64, "f16", 190, [5, 77, 300], [(16, "random"), (61, "wide"), (9, "chain")]),
    (8, 2, 128, 32, "f32", 140, [33, 0, 9], [(13, "forest"), (30, "random"), (50, "binary")]),
    (5, 1, 8, 256, "f32", 0, [255, 600], [(3, "wide"), (130, "random")]),
    (6, 2, 136, 16, "f16", 333, [1, 2, 3, 4], [(7, "random"), (1, "chain"), (12, "wide"), (2, "forest")]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("extras", [False, True])
def test_trees(shape, extras):
    H, KV, dk, page, dt, prefix, owns, trees = shape
    rng = np.random.default_rng(H * dk + page)
    cache = sq.PageCache(2, KV, dk, page, 60 + (prefix + sum(owns) + 1200) // page, dt)
    pools = Pools(cache)
    m = Model(H, KV, dk, dk // 2 - 2 if extras else dk // 2, rng, bias=extras, qk=extras)
    seqs = batch_of(cache, pools, prefix, owns, rng)
    batch = sq.PageBatch(cache, H, len(seqs), 300)
    parents = [tree(n, kind, rng) for n, kind in trees]
    run_tree(cache, pools, m, batch, seqs, parents, rng, layer=1)
    # the step again behind the first two rows of each tree, one sequence without rows, on another stream
    for s, p in zip(seqs, parents):
        cache.truncate(s, cache.length(s) - len(p) + min(2, len(p)))
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    parents = parents[1:] + [[] if len(parents) > 1 else parents[0]]
    for s in seqs:
        fill(cache, pools, s, cache.length(s), 1, rng)
    run_tree(cache, pools, m, batch, seqs, parents, rng, layer=1, stream=st.cuda_stream)


def test_tree_beside_prompt_and_large_tree():
    """A prompt, a tree of 1024 rows cut into several pieces, of which rows see little, and small trees."""
    rng = np.random.default_rng(3)
    for dt in ("f16", "f32"):
        cache = sq.PageCache(1, 2, 64, 32, 200, dt)
        pools = Pools(cache)
        m = Model(8, 2, 64, 32, rng)
        seqs = batch_of(cache, pools, 100, [7, 40, 3], rng)
        batch = sq.PageBatch(cache, 8, 3, 1500)
        big = [-1] + [0] * 300 + list(range(1, 724))
        run_tree(cache, pools, m, batch, seqs, [big, tree(200, "chain", rng), tree(30, "random", rng)], rng,
                 see=set(range(0, 1024, 37)) | {1023} | set(range(1024, 1254, 11)))


def test_rows_without_cached_ones():
    """Trees at the very start of their sequences: a node sees its path alone."""
    rng = np.random.default_rng(5)
    for dt in ("f16", "f32"):
        cache = sq.PageCache(1, 2, 128, 16, 60, dt)
        pools = Pools(cache)
        m = Model(8, 2, 128, 64, rng)
        seqs = [cache.add() for _ in range(3)]
        batch = sq.PageBatch(cache, 8, 3, 200)
        run_tree(cache, pools, m, batch, seqs, [tree(40, "forest", rng), tree(70, "wide", rng), [-1, -1, -1]], rng)


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("what", ["inf", "nan", "lowest"])
def test_what_a_node_does_not_see_does_not_reach_it(dt, what):
    """A node whose k and v rows are not finite (or the type's lowest value): its siblings' outputs are the formula's."""
    rng = np.random.default_rng(11)
    bad = {"inf": math.inf, "nan": math.nan, "lowest": -65504.0 if dt == "f16" else -3e38}[what]
    for nodes, H in ((6, 2), (20, 8), (40, 8)):
        cache = sq.PageCache(1, 1, 64, 16, 60, dt)
        pools = Pools(cache)
        m = Model(H, 1, 64, 0, rng)
        seqs = batch_of(cache, pools, 0, [150], rng)
        batch = sq.PageBatch(cache, H, 1, nodes)
        par = tree(nodes, "binary", rng)
        batch.begin_tree(seqs, [nodes], par)
        before = pools.host()
        q, k, v = rows_of(m, nodes, rng)
        k[2], v[2] = bad, bad
        out = attend(cache, m, batch, q, k, v)
        clean = {r for r in range(nodes) if 2 not in path_of(par, r)}
        assert np.isfinite(out[sorted(clean)]).all()
        if what == "nan":
            assert np.isnan(out[[r for r in range(nodes) if r not in clean]]).all()
        check(cache, pools, m, seqs, [par], q, k, v, out, before, see=clean)


def accept(starts, parents, tokens, chosen):
    """Paths by the rule, in Python."""
    kept, counts, after = np.full(len(tokens), -1, np.int32), [], []
    for at, par in zip(starts, parents):
        if not par:
            counts.append(0)
            after.append(-1)
            continue
        path = [0]
        while True:
            more = [r for r in range(len(par)) if par[r] == path[-1] and tokens[at + r] == chosen[at + path[-1]]]
            if not more:
                break
            path.append(more[0])
        kept[at:at + len(path)] = at + np.array(path)
        counts.append(len(path))
        after.append(chosen[at + path[-1]])
    return kept, np.array(counts, np.int32), np.array(after, np.int32)


def draw_choices(starts, parents, rng, hit=0.75, vocab=6):
    n = sum(len(p) for p in parents)
    tokens, chosen = (rng.integers(0, vocab, n).astype(np.int32) for _ in range(2))
    for at, par in zip(starts, parents):
        for r, p in enumerate(par):
            if p >= 0 and rng.random() < hit:
                chosen[at + p] = tokens[at + r]
    return tokens, chosen


def accept_dev(batch, tokens, chosen, n_seqs, stream=0):
    t, c = torch.from_numpy(tokens).cuda(), torch.from_numpy(chosen).cuda()
    kept = torch.full((len(tokens) + 3,), -7, dtype=torch.int32, device="cuda")
    counts, after = (torch.full((n_seqs + 2,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    sq.page_accept_dev(batch, t.data_ptr(), c.data_ptr(), kept.data_ptr(), counts.data_ptr(), after.data_ptr(), stream)
    torch.cuda.synchronize()
    assert (kept[len(tokens):] == -7).all() and (counts[n_seqs:] == -7).all() and (after[n_seqs:] == -7).all()
    return kept[:len(tokens)].cpu().numpy(), counts[:n_seqs].cpu().numpy(), after[:n_seqs].cpu().numpy()


def starts_of(parents):
    return np.cumsum([0] + [len(p) for p in parents])[:-1]


@pytest.mark.parametrize("seed", range(6))
def test_accepted_paths(seed):
    rng = np.random.default_rng(seed)
    cache = sq.PageCache(1, 1, 8, 16, 2000)
    kinds = ["chain", "binary", "random", "forest", "wide"]
    sizes = [[1], [2, 0, 5], [64, 17, 33, 1, 0, 16], [1024, 3], [300, 700, 7], [8] * 40][seed]
    parents = [tree(n, kinds[(i + seed) % 5], rng) for i, n in enumerate(sizes)]
    batch = sq.PageBatch(cache, 1, 64, 2200)
    seqs = [cache.add() for _ in sizes]
    for i, s in enumerate(seqs):
        cache.extend(s, (i * 7 + seed) % 40)
    batch.begin_tree(seqs, sizes, [x for p in parents for x in p])
    starts = starts_of(parents)
    for hit in (0.0, 0.75, 1.0):
        tokens, chosen = draw_choices(starts, parents, rng, hit, 2 if seed == 3 else 6)
        for a, b in zip(accept_dev(batch, tokens, chosen, len(seqs)), accept(starts, parents, tokens, chosen)):
            assert np.array_equal(a, b)
    # any integers are allowed
    tokens = rng.choice(np.array([-1, 2 ** 31 - 1, -2 ** 31], np.int32), sum(sizes))
    chosen = rng.choice(np.array([-1, 2 ** 31 - 1, -2 ** 31], np.int32), sum(sizes))
    for a, b in zip(accept_dev(batch, tokens, chosen, len(seqs)), accept(starts, parents, tokens, chosen)):
        assert np.array_equal(a, b)


def test_accepted_paths_of_a_step_without_trees():
    rng = np.random.default_rng(9)
    cache = sq.PageCache(1, 1, 8, 16, 2000)
    batch = sq.PageBatch(cache, 1, 8, 3000)
    seqs, rows = [cache.add() for _ in range(4)], [5, 1, 0, 2500]
    batch.begin(seqs, rows)
    parents = [tree(n, "chain", rng) for n in rows]
    starts = starts_of(parents)
    for hit in (0.5, 1.0):
        tokens, chosen = draw_choices(starts, parents, rng, hit)
        if hit == 1.0:
            chosen[starts[3] + 2000] = 99
        for a, b in zip(accept_dev(batch, tokens, chosen, 4), accept(starts, parents, tokens, chosen)):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("dt,page,dk,kv", [("f32", 16, 64, 3), ("f16", 32, 128, 8), ("f16", 16, 8, 1), ("f32", 64, 256, 2),
                                           ("f16", 16, 200, 5)])
def test_kept_rows(dt, page, dk, kv):
    rng = np.random.default_rng(dk)
    cache = sq.PageCache(3, kv, dk, page, 120, dt)
    pools = Pools(cache, 0.0)
    for t in pools.t:
        t.copy_(torch.randn(t.shape, device="cuda").to(t.dtype))
    sizes = [40, 1, 7, 0, 33, 300, 20]
    seqs = [cache.add() for _ in sizes]
    for i, s in enumerate(seqs):
        cache.extend(s, 5 * i)
    parents = [tree(n, "wide", rng) for n in sizes[:-1]] + [tree(20, "chain", rng)]
    batch = sq.PageBatch(cache, kv, len(sizes), sum(sizes))
    batch.begin_tree(seqs, sizes, [x for p in parents for x in p])
    starts = starts_of(parents)
    kept = np.full(sum(sizes), -1, np.int32)
    for i, (at, n) in enumerate(zip(starts, sizes)):
        path = np.sort(rng.permutation(n)[:(0, 1, 3, 0, 12, 290, 20)[i]])
        kept[at:at + len(path)] = at + path
    before = pools.host()
    want = [b.copy() for b in before]
    for s, at, n in zip(seqs, starts, sizes):
        m = int((kept[at:at + n] >= 0).sum())
        base = cache.length(s) - n
        (dp, ds), (sp, ss) = pools.where(s, base + np.arange(m)), pools.where(s, base + kept[at:at + m] - at)
        for w, b in zip(want, before):
            w[:, dp, :, ds] = b[:, sp, :, ss]
    d = torch.from_numpy(kept).cuda()
    torch.cuda.synchronize()
    sq.page_keep_dev(batch, d.data_ptr())
    for w, a in zip(want, pools.host()):
        assert np.array_equal(w.view(BITS[dt]), a.view(BITS[dt]))


def test_entries_that_name_no_row_end_the_path():
    cache = sq.PageCache(2, 2, 64, 16, 20)
    pools = Pools(cache, 0.0)
    for t in pools.t:
        t.copy_(torch.randn(t.shape, device="cuda"))
    seqs = [cache.add(), cache.add()]
    batch = sq.PageBatch(cache, 2, 2, 16)
    batch.begin_tree(seqs, [8, 8], ([-1] + [0] * 7) * 2)
    for bad in (-5, 3, 8, 15, 16, 2 ** 31 - 1, -2 ** 31):  # rows before its place, of the other sequence, of nobody
        kept = np.full(16, -1, np.int32)
        kept[0:4] = [0, 2, 4, bad]  # (3 is the place itself)
        kept[4:8] = [5, 6, 7, 7]
        before = pools.host()
        d = torch.from_numpy(kept).cuda()
        torch.cuda.synchronize()
        sq.page_keep_dev(batch, d.data_ptr())
        pg, sl = pools.where(seqs[0], np.arange(8))
        want = [b.copy() for b in before]
        rows = [0, 2, 4, 3, 5, 6, 7, 7] if bad == 3 else [0, 2, 4, 3, 4, 5, 6, 7]
        for w, b in zip(want, before):
            w[:, pg, :, sl] = b[:, pg[rows], :, sl[rows]]
        for w, a in zip(want, pools.host()):
            assert np.array_equal(w.view(np.uint32), a.view(np.uint32))


def test_refusals():
    cache = sq.PageCache(1, 1, 64, 16, 20)
    batch = sq.PageBatch(cache, 2, 2, 16)
    s = cache.add()
    x = torch.zeros(64, dtype=torch.int32, device="cuda")
    p = x.data_ptr()

    def status(f):
        with pytest.raises(sq.SllmError) as e:
            f()
        return e.value.status

    keep = lambda: sq.page_keep_dev(batch, p)  # noqa: E731
    acc = lambda: sq.page_accept_dev(batch, p, p, p, p, p)  # noqa: E731
    rules = lambda n=3: sq.logits_rules_dev(p, n, 4, sq.LogitsParams(), 0, p, batch)  # noqa: E731
    for f in (keep, acc, rules):
        assert status(f) == 1  # no step yet
    assert status(lambda: batch.begin_tree([s], [2], [-1])) == 1
    assert status(lambda: batch.begin_tree([s], [2], [0, 0])) == 1
    assert cache.length(s) == 0
    cache.extend(s, 4)
    batch.begin_tree([s], [3], [-1, 0, 0])
    assert status(lambda: rules(2)) == 3 and status(lambda: rules(4)) == 3
    other = cache.fork(s, 6)  # holds the page of the step's rows
    assert status(keep) == 1
    cache.free(other)
    keep()
    cache.truncate(s, 6)
    for f in (keep, acc, rules):
        assert status(f) == 1  # the step has ended
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        assert status(lambda: batch.begin_tree([s], [1], [-1], st.cuda_stream)) == 1
    torch.cuda.synchronize()
    # a captured call with a batch is for all rows that it may have
    batch.begin_tree([s], [3], [-1, 0, 0])
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        assert status(lambda: sq.logits_rules_dev(p, 3, 4, sq.LogitsParams(), 0, p, batch, st.cuda_stream)) == 3
    torch.cuda.synchronize()
