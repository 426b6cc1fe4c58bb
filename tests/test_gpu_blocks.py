"""GPU tests of every kind of block that the batch attention cuts a step's rows into (_blocks.py; the plans are checked in
test_block_plans_cpu.py): rows of prompts and of trees, against the formulas in 64 bits with the bounds of test_gpu_pages.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import _blocks
import sllm_qmm as sq
from test_gpu_pages import NP, Model, Pools, attention64, batch_of, check_step
from test_gpu_tree import attend, check, path_of, rows_of

pytestmark = pytest.mark.gpu
STEPS = {s.name: s for s in _blocks.steps()}


def opened(step, rng, extras=False, fill=float("nan")):
    rows = sum(step.owns) + sum(step.rows)
    pages = step.prefix // step.page + rows // step.page + 3 * len(step.owns) + 2
    cache = sq.PageCache(1, step.kv, step.dk, step.page, pages, step.dtype)
    pools = Pools(cache, fill)
    m = Model(step.heads, step.kv, step.dk, step.dk // 2, rng, bias=extras, qk=extras)
    seqs = batch_of(cache, pools, step.prefix, step.owns, rng)
    return cache, pools, m, seqs, sq.PageBatch(cache, step.heads, len(seqs), sum(step.rows))


def some(step):
    """Rows whose outputs are looked at: some of each tree, fewer where they are long."""
    n = sum(step.rows)
    return set(range(0, n, max(1, n * max(1, (step.prefix + step.owns[0]) // 500) // 50))) | {n - 1}


@pytest.mark.parametrize("name", STEPS)
def test_blocks(name):
    step = STEPS[name]
    rng = np.random.default_rng(step.dk + len(name))
    cache, pools, m, seqs, batch = opened(step, rng, extras="128" not in name)
    n = sum(step.rows)
    parents = _blocks.parents(step) if step.trees else None
    if parents:
        batch.begin_tree(seqs, step.rows, [x for p in parents for x in p])
    else:
        batch.begin(seqs, step.rows)
    before = pools.host()
    q, k, v = rows_of(m, n, rng)
    out = attend(cache, m, batch, q, k, v)
    if parents:
        check(cache, pools, m, seqs, parents, q, k, v, out, before, see=some(step))
    else:
        check_step(cache, pools, m, seqs, step.rows, q, k, v, np.concatenate([out, np.full((1, out.shape[1]), np.nan, np.float32)]),
                   before, 0)


@pytest.mark.parametrize("bad", ["inf", "nan"])
@pytest.mark.parametrize("name", [f"{s}_{t}" for s in ("trees61", "trees12") for t in ("f32_128", "f16_128")] +
                         ["trees61_f16_96", "trees61_f32_192", "wide_far_f16", "wide_far_f32"])
def test_nodes_that_are_not_finite(name, bad):
    """A node of two trees whose k and v rows are not finite: rows that do not see it have the formula's outputs, also
    those of its own block (computed again, row by row)."""
    step = STEPS[name]
    rng = np.random.default_rng(7)
    cache, pools, m, seqs, batch = opened(step, rng)
    parents = _blocks.parents(step)
    batch.begin_tree(seqs, step.rows, [x for p in parents for x in p])
    before = pools.host()
    n = sum(step.rows)
    q, k, v = rows_of(m, n, rng)
    starts = np.cumsum([0] + step.rows)
    hit = set()
    for i in {0, len(seqs) - 1}:
        k[starts[i] + 2] = v[starts[i] + 2] = float(bad)
        hit |= {int(starts[i]) + r for r, p in enumerate(parents[i]) if 2 in path_of(parents[i], r)}
    out = attend(cache, m, batch, q, k, v)
    clean = set(range(n)) - hit
    assert hit and np.isfinite(out[sorted(clean)]).all()
    if bad == "nan":
        assert np.isnan(out[sorted(hit)]).all()
    near = {r for r in clean if r < step.rows[0] or r >= n - step.rows[-1]}
    see = set(sorted(near)[::7]) if "far" not in name else set(sorted(near)[::19])
    check(cache, pools, m, seqs, parents, q, k, v, out, before, see=see | (some(step) & clean if "far" not in name else set()))


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("name", ["prompts_f32_128", "prompts_f16_128", "prompts_f32_96", "prompts_f16_96", "prompts_f32_256",
                                  "short_prompts_f32_128", "short_prompts_f16_72"])
def test_rows_that_are_not_finite(name, bad):
    """An element of a prompt's v row: rows before it have the formula's outputs, rows from it on that value there."""
    step = STEPS[name]
    rng = np.random.default_rng(8)
    cache, pools, m, seqs, batch = opened(step, rng)
    H, dk, rep, c = step.heads, step.dk, step.heads // step.kv, step.rows[2]
    batch.begin(seqs, step.rows)
    q, k, v = rows_of(m, sum(step.rows), rng)
    at, x = 2 * c, c // 2  # (all prompts have as many rows: the third one's middle)
    v[at + x, dk + 5] = bad  # kv head 1
    out = attend(cache, m, batch, q, k, v).reshape(-1, H, dk)
    assert np.isfinite(np.delete(out, np.s_[at:at + c], 0)).all()
    K, V = (a[0].astype(np.float64) for a in pools.read(seqs[2]))
    base = cache.length(seqs[2]) - c
    assert not np.isfinite(V[base + x, 1, 5])
    V[base + x, 1, 5] = 0.0
    pos = np.arange(base, base + c)
    qr, qs = m.row(q[at:at + c], H, None, None, pos)
    for h in range(H):
        o, b = attention64(qr[:, h], qs[:, h], K[:, h // rep], V[:, h // rep], pos, 1 / math.sqrt(dk))
        got = out[at:at + c, h].copy()
        if h // rep == 1:
            seen = got[x:, 5].copy()
            assert np.isnan(seen).all() if math.isnan(bad) else (seen == np.float32(bad)).all()
            got[x:, 5] = o[x:, 5]
        assert (np.abs(got - o) <= b).all(), h


@pytest.mark.parametrize("gap", [8, 14, 17])
@pytest.mark.parametrize("name", ["prompts_f32_128", "prompts_f16_128", "prompts_f16_96", "prompts_f16_192",
                                  "short_prompts_f16_128", "short_prompts_f32_72"])
def test_small_weights_behind_a_large_one(name, gap):
    """Position 0's score is `gap` nats above the others', and its V is small. Weights of f16 caches are within 2^-23 of
    themselves or 2^-38 of the largest: the latter, times |v|, is added to the bounds of test_gpu_pages."""
    step = STEPS[name]
    rng = np.random.default_rng(gap)
    H, KV, dk, rep = step.heads, step.kv, step.dk, step.heads // step.kv
    owns = [o + 120 for o in step.owns]  # (hundreds of others)
    cache, pools, m, seqs, batch = opened(step._replace(owns=owns), rng)
    m = Model(H, KV, dk, 0, rng)
    for s, o in zip(seqs, owns):
        K, V = rng.normal(size=(1, o, KV, dk)) * 0.3, np.abs(rng.normal(size=(1, o, KV, dk))) + 0.5
        K[..., 0] = 0
        K[0, 0], V[0, 0] = 0, 1e-3 * V[0, 0]
        K[0, 0, :, 0] = gap
        pools.write(s, 0, K.astype(NP[step.dtype]), V.astype(NP[step.dtype]))
    batch.begin(seqs, step.rows)
    q, k, v = rows_of(m, sum(step.rows), rng, 0.5)
    k, v = 0.3 * k, np.abs(v) + np.float32(0.5)
    q[:, ::dk], k[:, ::dk] = dk ** 0.5, 0
    out = attend(cache, m, batch, q, k, v)
    host, at = pools.host(), 0
    for i, (s, c) in enumerate(zip(seqs, step.rows)):
        if i % 3 == 0:
            pos = np.arange(cache.length(s) - c, cache.length(s))
            K, V = (a[0].astype(np.float64) for a in pools.read(s, host))
            qr, qs = m.row(q[at:at + c], H, None, None, pos)
            for h in range(H):
                o, b = attention64(qr[:, h], qs[:, h], K[:, h // rep], V[:, h // rep], pos, dk ** -0.5)
                floor = np.stack([2.0 ** -38 * V[:p + 1, h // rep].sum(0) for p in pos])
                got = out[at:at + c, h * dk:(h + 1) * dk]
                assert (np.abs(got - o) <= b + floor).all(), (s, h)
        at += c
