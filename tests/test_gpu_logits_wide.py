"""GPU tests of the rules for logits in large launches, which take chunks of 4096 tokens: rows x ceil((vocab + 3) / 1024) above
2048, asserted for each call. Values bit for bit, chosen tokens equal, as in test_gpu_logits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import sllm_qmm as sq
from test_gpu_logits import Case, draw
from test_gpu_tree import path_of, starts_of, tree

pytestmark = pytest.mark.gpu
F = np.float32


def large(rows, vocab):
    assert rows * -(-(vocab + 3) // 1024) > 2048
    return rows, vocab


@pytest.mark.parametrize("rows,vocab", [(24, 128256), (17, 128257), (70, 32003), (300, 9001), (530, 4093), (530, 4095), (530, 4096),
                                        (530, 4097), (530, 4099), (300, 8189), (300, 8192), (300, 8195), (2100, 7)])
def test_vocabularies(rows, vocab):
    large(rows, vocab)
    rng = np.random.default_rng(vocab)
    for i, allowed in enumerate((None, 0.5, 0.03, 0.0)):
        c, x = draw(vocab, rows, rng, 200, 20, allowed)
        c.run(x, off=(i, 0))
        c.run(x, dst="in", off=(3 - i, 0))
        c.run(x, dst="none", off=(i, 0))
        c.run(x, chosen=False, off=(i, (i + 1) % 4))
        c.run(x, off=(3, 3))


def test_values_that_are_not_numbers():
    rng = np.random.default_rng(1)
    rows, v = large(230, 9001)
    c, x = draw(v, rows, rng, 300, 30, 0.4)
    for r in range(0, rows, 8):
        x[r, ::2] = np.nan
        x[r + 1, 100:8400] = np.inf
        x[r + 2, :] = -np.inf
        x[r + 3, :] = np.nan
        x[r + 4, :] = np.finfo(F).min
        x[r + 5, 0], x[r + 5, v - 1] = np.nan, np.inf
    c.run(x)
    c.run(x, dst="in", off=(1, 0))
    c.run(x, dst="none", off=(2, 0))
    some = [(0.0, 1.0, 0.0, [1, 1, 2], []), (1e-38, -3e38, 3e38, [5000] * 100, [(5000, np.inf)]),
            (-2.0, 0.0, 0.0, range(8190, 8250), [(8195, np.nan)])]
    masks = [None, None, [8195, 60]]
    Case(v, some * 77, masks * 77).run((rng.normal(size=(231, v)) * 5).astype(F))


def test_ties_take_the_first_token():
    rows, v = large(260, 9001)
    x = np.full((rows, v), 1.0, F)
    for r in range(rows):
        if r % 4 == 1:  # zeros of either sign are equal: the first
            x[r, :8000] = -0.0
            x[r, 8000:] = 0.0
        elif r % 4 == 2:  # across chunks, and within a thread's elements
            x[r, [4096 + r % 3, 8192 + r % 5, 8999]] = 3.0
        elif r % 4 == 3:
            x[r, :] = np.nan
            x[r, 8990 + r % 10:] = -5.0
    for off in range(4):
        Case(v, []).run(x, off=(off, 0))
    masks = [None if r % 3 else [8000 + r, 7000 + r, 4095, 4096] for r in range(rows)]
    Case(v, [], masks).run(x)


def test_a_token_biased_twice_takes_the_later():
    rng = np.random.default_rng(0)
    rows, v = large(420, 5000)
    x = np.zeros((rows, v), F)
    rules = [(1.0, 0.0, 0.0, [], [(7, 1.0), (4999, 2.0), (4096, 5.0), (7, 3.0), (4999, -1.0), (7, 2.5), (4096, 0.5)])] * 3
    rules += [(1.0, 0.0, 0.0, [], [(int(t), float(i)) for i, t in enumerate(4080 + rng.integers(0, 40, 2000))])] * 2
    Case(v, rules).run(x)
    Case(v, rules).run(x, dst="in", off=(1, 0))


def test_long_histories():
    rng = np.random.default_rng(4)
    rows, v = large(350, 6000)
    c = Case(v, [(1.25, 0.001, 0.5, rng.integers(0, v, 40000), []), (1.0, 0.5, 0.0, np.full(30000, 4097), []),
                 (1.5, 0.25, 0.0, np.arange(4090, 4100), [(4095, 1.0), (4096, -1.0)])])
    c.run((rng.normal(size=(rows, v)) * 3).astype(F), off=(2, 0))


def trees_of(sizes, rng):
    return [tree(n, ("random", "chain", "forest", "wide", "binary")[i % 5], rng) for i, n in enumerate(sizes)]


def opened(max_rows, max_seqs=6):
    cache = sq.PageCache(1, 1, 8, 16, 400)
    batch = sq.PageBatch(cache, 1, max_seqs, max_rows)
    seqs = [cache.add() for _ in range(max_seqs)]
    for i, s in enumerate(seqs):
        cache.extend(s, 11 * i)
    return cache, batch, seqs


def paths(parents, tokens):
    return [tokens[[at + y for y in path_of(p, r)]] for at, p in zip(starts_of(parents), parents) for r in range(len(p))]


def test_trees():
    rng = np.random.default_rng(3)
    cache, batch, seqs = opened(400)
    sizes = [17, 0, 1, 120, 100, 62]
    rows, v = large(sum(sizes), 9001)
    parents = trees_of(sizes, rng)
    batch.begin_tree(seqs, sizes, [x for p in parents for x in p])
    tokens = rng.choice(np.array([5, 6, 4095, 4096, 4097, 8999, -1], np.int32), rows)
    of = np.repeat(np.arange(len(sizes)), sizes)
    some, _ = draw(v, 5, rng, 30, 4)  # (the last sequence has no rule)
    masks = [None if r % 4 else rng.permutation(v)[:9] for r in range(rows)]
    x = (rng.normal(size=(rows, v)) * 3).astype(F)
    c = Case(v, some.rules, masks, tokens)
    c.run(x, batch=batch, of=of, extra=paths(parents, tokens))
    c.run(x, dst="none", off=(1, 0), batch=batch, of=of, extra=paths(parents, tokens))
    Case(v, some.rules, masks).run(x, dst="in", batch=batch, of=of)


@pytest.mark.parametrize("most", [40, 300])
def test_captured_calls_follow_the_steps(most):
    """A call recorded for max_rows rows, replayed over steps of fewer, of none and of as many: rows behind the step's keep
    what they hold. (Chunks of 1024 and of 4096.)"""
    rng = np.random.default_rng(most)
    v = 9001
    assert (most * -(-(v + 3) // 1024) > 2048) == (most == 300)
    cache, batch, seqs = opened(most)
    st = torch.cuda.Stream()
    sq.workspace_reserve(st.cuda_stream, 1 << 20)
    first = [3, 2, 1, 4, 5, 6]
    batch.begin_tree(seqs, [most - 5, 1, 1, 1, 1, 1], [x for p in trees_of([most - 5, 1, 1, 1, 1, 1], rng) for x in p], st.cuda_stream)
    some, _ = draw(v, 5, rng, 40, 6)
    c = Case(v, some.rules, [np.nonzero(rng.random(v) < 0.2)[0] if r % 3 == 0 else None for r in range(most)],
             np.zeros(most, np.int32))
    src = torch.zeros(most, v, device="cuda")
    dst = torch.zeros(most, v, device="cuda")
    chosen = torch.zeros(most, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        sq.logits_rules_dev(src.data_ptr(), most, v, c.params, dst.data_ptr(), chosen.data_ptr(), batch, st.cuda_stream)
    for i, s in enumerate(seqs):
        cache.truncate(s, 11 * i)
    full = [most - 25, 5, 5, 5, 5, 5]
    for sizes in (first, [0] * 6, [0, 0, 7, 0, 1, 0], full, [1] * 6, full[::-1]):
        n = sum(sizes)
        parents = trees_of(sizes, rng)
        batch.begin_tree(seqs, sizes, [x for p in parents for x in p], st.cuda_stream)
        tokens = rng.choice(np.array([1, 2, 4095, 4096, 8999], np.int32), most)
        x = (rng.normal(size=(most, v)) * 3).astype(F)
        src.copy_(torch.from_numpy(x))
        c.keep["tokens"].copy_(torch.from_numpy(tokens))
        of, extra = np.repeat(np.arange(6), sizes), paths(parents, tokens[:n])
        for _ in range(2):
            dst.fill_(77.0)
            chosen.fill_(-9)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got, picked = dst.cpu().numpy(), chosen.tolist()
            for r in range(n):
                y, best = c.row(x[r], of[r], extra[r], c.masks[r])
                assert picked[r] == best and np.array_equal(got[r], y, equal_nan=True), (sizes, r)
            assert (got[n:] == 77.0).all() and picked[n:] == [-9] * (most - n)
        if n:  # an eager call between replays
            c.tokens = tokens
            masks, c.masks = c.masks, c.masks[:n]
            c.run(x[:n], batch=batch, stream=st.cuda_stream, of=of, extra=extra)
            c.masks = masks
        for i, s in enumerate(seqs):
            cache.truncate(s, 11 * i)
