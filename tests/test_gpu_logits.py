"""GPU tests of the rules for logits (sllm_logits_rules_dev) against the formula: each operation rounds once to float32 in
the documented order, so values agree bit for bit (zeros in value), and the chosen tokens are equal."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import sllm_qmm as sq
from test_gpu_tree import path_of, starts_of, tree

pytestmark = pytest.mark.gpu
F = np.float32


class Case:
    """rules: per request (repeat, frequency, presence, history, {or list of} biases); masks: per row an array of allowed
    tokens or None."""

    def __init__(self, vocab, rules, masks=None, tokens=None):
        self.vocab, self.rules, self.tokens = vocab, rules, tokens
        r = np.zeros(len(rules), sq.LOGITS_RULE)
        hist, bt, bv = [7], [3], [9.0]  # (entries that no rule names)
        for i, (rep, fr, pr, h, b) in enumerate(rules):
            r[i] = (rep, fr, pr, len(hist), len(h), len(bt), len(b), 0)
            hist += list(h)
            bt += [t for t, _ in b]
            bv += [x for _, x in b]
        self.host = r
        self.keep = {"rules": torch.from_numpy(r.view(np.int32).copy()).cuda(),
                     "history": torch.tensor(hist, dtype=torch.int32, device="cuda"),
                     "bt": torch.tensor(bt, dtype=torch.int32, device="cuda"),
                     "bv": torch.tensor(bv, dtype=torch.float32, device="cuda")}
        kw = {}
        self.masks = masks
        if masks is not None:
            words = -(-vocab // 32)
            table, ids = [], []
            for k in masks:
                if k is None:
                    ids.append(-1)
                    continue
                bits = np.zeros(words * 32, np.uint8)
                bits[vocab:] = 1  # (bits behind the vocabulary say nothing)
                bits[np.asarray(k, int)] = 1
                ids.append(len(table))
                table.append(np.packbits(bits, bitorder="little").view(np.int32))
            self.keep["masks"] = torch.from_numpy(np.array(table)).cuda() if table else torch.zeros(1, dtype=torch.int32, device="cuda")
            self.keep["ids"] = torch.tensor(ids, dtype=torch.int32, device="cuda")
            kw = {"masks": self.keep["masks"].data_ptr(), "n_masks": len(table), "mask_ids": self.keep["ids"].data_ptr()}
        if tokens is not None:
            self.keep["tokens"] = torch.from_numpy(tokens).cuda()
            kw["tokens"] = self.keep["tokens"].data_ptr()
        self.params = sq.LogitsParams(rules=self.keep["rules"].data_ptr(), n_rules=len(rules),
                                      history=self.keep["history"].data_ptr(), n_history=len(hist),
                                      bias_tokens=self.keep["bt"].data_ptr(), bias_values=self.keep["bv"].data_ptr(),
                                      n_biases=len(bt), **kw)

    def row(self, x, i, extra=(), mask=None):
        """The formula for one row of request i (extra: tokens of its path)."""
        y = x.copy()
        with np.errstate(all="ignore"):
            if i < len(self.rules):
                rep, fr, pr, h, b = self.rules[i]
                t = np.concatenate([np.asarray(h, np.int64).reshape(-1), np.asarray(extra, np.int64).reshape(-1)])
                n = np.bincount(t[(t >= 0) & (t < self.vocab)].astype(int), minlength=self.vocab)
                s = n > 0
                l = np.where(y[s] > 0, y[s] / F(rep), y[s] * F(rep)).astype(F)
                y[s] = l - (F(fr) * n[s].astype(F) + F(pr))
                for t, v in dict(b).items():
                    if 0 <= t < self.vocab:
                        y[t] = y[t] + F(v)
            elif len(extra):
                pass  # (no rule: counts change nothing)
            if mask is not None:
                off = np.ones(self.vocab, bool)
                off[np.asarray(mask, int)] = False
                y[off] = -np.inf
        z = np.where(np.isnan(y), F(-np.inf), y)
        return y, int(np.argmax(z)) if z.max() > -np.inf else -1

    def run(self, x, dst="out", chosen=True, off=(0, 0), batch=None, stream=0, want=None, extra=None, of=None):
        """One call on rows x, checked. off: floats by which the buffers' starts are moved from 16-byte boundaries."""
        rows = len(x)
        src = torch.full((x.size + 8,), float("nan"), device="cuda")
        src[off[0]:off[0] + x.size] = torch.from_numpy(x.reshape(-1)).cuda()
        held = src.clone()
        out = src if dst == "in" else torch.full((x.size + 8,), 77.0, device="cuda")
        o = off[0] if dst == "in" else off[1]
        c = torch.full((rows + 1,), -9, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        sq.logits_rules_dev(src.data_ptr() + 4 * off[0], rows, self.vocab, self.params,
                            out.data_ptr() + 4 * o if dst != "none" else 0, c.data_ptr() if chosen else 0, batch, stream)
        torch.cuda.synchronize()
        got = out[o:o + x.size].cpu().numpy().reshape(x.shape)
        for r in range(rows):
            i = r if of is None else of[r]
            y, best = self.row(x[r], i, () if extra is None else extra[r], None if self.masks is None else self.masks[r])
            if chosen:
                assert int(c[r]) == best, (r, int(c[r]), best)
            if dst != "none":
                assert np.array_equal(got[r], y, equal_nan=True), (r, np.argwhere(got[r] != y)[:4])
        edge = torch.cat([out[:o], out[o + x.size:]])
        assert torch.isnan(edge).all() if dst == "in" else (edge == 77.0).all()
        if dst != "in":
            assert torch.equal(src.view(torch.int32), held.view(torch.int32))
        assert int(c[rows]) == -9 and (chosen or (c == -9).all())


def draw(vocab, rows, rng, history=50, biases=5, allowed=None):
    some = lambda: (1 + rng.random(), rng.random() * 2, rng.random(), rng.integers(0, vocab, rng.integers(0, history + 1)),  # noqa: E731
                    [(int(t), float(F(rng.normal() * 5))) for t in rng.integers(0, vocab, rng.integers(0, biases + 1))])
    masks = None
    if allowed is not None:
        masks = [None if i % 3 == 2 else np.nonzero(rng.random(vocab) < allowed)[0] for i in range(rows)]
    rules = [(float(F(a)), float(F(b)), float(F(c)), h, list(dict(bb).items())) for a, b, c, h, bb in (some() for _ in range(rows))]
    return Case(vocab, rules, masks), (rng.normal(size=(rows, vocab)) * 3).astype(F)


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 32, 33, 100, 4093, 4095, 4096, 4097, 4099, 8191, 8192, 12289, 32003, 128256])
def test_vocabularies(vocab):
    rng = np.random.default_rng(vocab)
    for rows, allowed in ((1, None), (3, 0.5), (6, 0.03), (2, 0.0)):
        c, x = draw(vocab, rows, rng, 200, 20, allowed)
        c.run(x)
        c.run(x, dst="in", off=(rows % 4, 0))
        c.run(x, dst="none", off=(1, 0))
        c.run(x, chosen=False, off=(2, 3))
        c.run(x, off=(3, 3))


def test_values_that_are_not_numbers():
    rng = np.random.default_rng(1)
    c, x = draw(5000, 7, rng, 300, 30, 0.4)
    x[0, ::2] = np.nan
    x[1, 100:4000] = np.inf
    x[2, :] = -np.inf
    x[3, :] = np.nan
    x[4, :] = np.finfo(F).min
    x[5, 0], x[5, 4999] = np.nan, np.inf
    x[6, :] = 2.0  # ties: the first
    c.run(x)
    c.run(x, dst="in")
    c.run(x, dst="none")
    # values whose rules leave the range, a penalty of 0 (division by it), negative ones
    rules = [(0.0, 1.0, 0.0, [1, 1, 2], []), (1e-38, -3e38, 3e38, [5] * 100, [(5, np.inf)]), (-2.0, 0.0, 0.0, range(60), [(3, np.nan)])]
    Case(64, rules, [None, None, [3, 60]]).run((rng.normal(size=(3, 64)) * 5).astype(F))


def test_ties_take_the_first_token():
    x = np.full((4, 9000), 1.0, F)
    x[1, :8000] = -0.0
    x[1, 8000:] = 0.0
    x[1, 5] = 0.0
    x[2, [4100, 8999]] = 3.0
    x[3, :] = np.nan
    x[3, 8998:] = -5.0
    Case(9000, []).run(x)
    Case(9000, [], [None, [8000, 7000], [8999], [8999]]).run(x)


def test_what_lies_outside_is_not_there():
    rng = np.random.default_rng(2)
    v = 300
    c = Case(v, [(1.5, 0.5, 0.25, [5, -1, v, 2 ** 31 - 1, -2 ** 31, 6, 6], [(-1, 4.0), (v, 4.0), (2 ** 31 - 1, 9.0), (8, 2.0)])] * 2)
    x = rng.normal(size=(4, v)).astype(F)  # (rows 2 and 3 have no rule)
    c.run(x)
    # ranges that leave their arrays; the later of two biases of a token counts
    n = int(c.keep["history"].numel())
    r = c.host.copy()
    r["history_at"], r["history"] = [n - 1, -3], [2 ** 31 - 1, 10]
    r["bias_at"], r["biases"] = [2 ** 31 - 1, 0], [5, 3]
    c.keep["rules"].copy_(torch.from_numpy(r.view(np.int32)))
    hist, bt, bv = (c.keep[k].cpu().tolist() for k in ("history", "bt", "bv"))
    c.rules = [(1.5, 0.5, 0.25, hist[n - 1:], []), (1.5, 0.5, 0.25, hist[:7], list(zip(bt, bv))[:3])]
    c.run(x)
    r["history"], r["biases"] = -4, -1  # (negative counts: none)
    c.keep["rules"].copy_(torch.from_numpy(r.view(np.int32)))
    c.rules = [(1.5, 0.5, 0.25, [], [])] * 2
    c.run(x)
    # a mask's number that there is not
    c = Case(v, [], [[1, 2], [3], None, [4]])
    c.keep["ids"].copy_(torch.tensor([0, 3, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32))
    c.masks = [[1, 2], None, None, None]
    c.run(x)


def test_a_token_biased_twice_takes_the_later():
    x = np.zeros((1, 5000), F)
    c = Case(5000, [(1.0, 0.0, 0.0, [], [(7, 1.0), (4999, 2.0), (7, 3.0), (4999, -1.0), (7, 2.5)])])
    c.run(x)
    # many names of few tokens
    rng = np.random.default_rng(0)
    b = [(int(t), float(i)) for i, t in enumerate(rng.integers(0, 40, 3000))]
    Case(5000, [(1.0, 0.0, 0.0, [], b)]).run(x)


def test_long_histories():
    rng = np.random.default_rng(4)
    c = Case(6000, [(1.25, 0.001, 0.5, rng.integers(0, 6000, 40000), []), (1.0, 0.5, 0.0, np.full(100000, 4097), [])])
    c.run((rng.normal(size=(2, 6000)) * 3).astype(F))


def test_many_rows_and_streams():
    rng = np.random.default_rng(6)
    c, x = draw(1003, 700, rng, 30, 3, 0.2)
    c.run(x)
    a, xa = draw(40001, 5, rng, 500, 9, 0.1)
    st = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for s in st:
        a.run(xa, stream=s.cuda_stream)


@pytest.mark.parametrize("vocab", [70, 9001])
def test_trees(vocab):
    """Rows of a step: penalties count the tokens of a row's path too."""
    rng = np.random.default_rng(vocab)
    cache = sq.PageCache(1, 1, 8, 16, 200)
    sizes, kinds = [17, 0, 1, 40, 100, 6], ["random", "chain", "chain", "forest", "wide", "chain"]
    parents = [tree(n, k, rng) for n, k in zip(sizes, kinds)]
    batch = sq.PageBatch(cache, 1, 8, 400)
    seqs = [cache.add() for _ in sizes]
    for i, s in enumerate(seqs):
        cache.extend(s, 11 * i)
    batch.begin_tree(seqs, sizes, [x for p in parents for x in p])
    starts, rows = starts_of(parents), sum(sizes)
    tokens = rng.integers(0, 12, rows).astype(np.int32)
    tokens[::9] = -1
    of = np.repeat(np.arange(len(sizes)), sizes)
    extra = [tokens[[at + y for y in path_of(p, r)]] for at, p in zip(starts, parents) for r in range(len(p))]
    some, _ = draw(vocab, 5, rng, 30, 4)  # (the last sequence has no rule)
    masks = [None if r % 4 else rng.permutation(vocab)[:9] for r in range(rows)]
    c = Case(vocab, some.rules, masks, tokens)
    x = (rng.normal(size=(rows, vocab)) * 3).astype(F)
    c.run(x, batch=batch, of=of, extra=extra)
    c.run(x, dst="none", batch=batch, of=of, extra=extra)
    # without tokens: the histories alone
    Case(vocab, some.rules, masks).run(x, batch=batch, of=of)
    # a step without trees
    batch.begin(seqs[:2], [30, 3])
    tokens = rng.integers(0, 12, 33).astype(np.int32)
    Case(vocab, some.rules, None, tokens).run(x[:33], batch=batch, of=[0] * 30 + [1] * 3,
                                              extra=[tokens[:r + 1] for r in range(30)] + [tokens[30:31 + r] for r in range(3)])


def test_refusals():
    x = torch.zeros(16, device="cuda")
    p = x.data_ptr()

    def status(*a, **k):
        with pytest.raises(sq.SllmError) as e:
            sq.logits_rules_dev(*a, **k)
        return e.value.status

    none = sq.LogitsParams()
    assert status(0, 1, 4, none, p, p) == 1 and status(p, 1, 4, none, 0, 0) == 1
    assert status(p, -1, 4, none, p, p) == 1 and status(p, 1, 0, none, p, p) == 1
    assert status(p + 2, 1, 4, none, p, p) == 1 and status(p, 1, 4, none, p + 1, p) == 1
    for f in ("n_rules", "n_history", "n_biases", "n_masks"):
        assert status(p, 1, 4, sq.LogitsParams(**{f: 1}), p, p) == 1
        assert status(p, 1, 4, sq.LogitsParams(**{f: -1}), p, p) == 1
    assert status(p, 65536, 4, none, p, p) == 3 and status(p, 1, (1 << 28) + 1, none, p, p) == 3
    sq.logits_rules_dev(p, 0, 4, none, p, p)
    torch.cuda.synchronize()


def test_captured_calls_read_what_is_there():
    """A graph replayed over other logits, rules and masks, with eager calls on the same stream between."""
    rng = np.random.default_rng(8)
    v, rows = 9001, 6
    c, x = draw(v, rows, rng, 300, 10, 0.3)
    st = torch.cuda.Stream()
    sq.workspace_reserve(st.cuda_stream, 1 << 20)
    src, dst = torch.zeros(rows, v, device="cuda"), torch.zeros(rows, v, device="cuda")
    chosen = torch.zeros(rows, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        sq.logits_rules_dev(src.data_ptr(), rows, v, c.params, dst.data_ptr(), chosen.data_ptr(), None, st.cuda_stream)
    for i in range(4):
        x = (rng.normal(size=(rows, v)) * 3).astype(F)
        src.copy_(torch.from_numpy(x))
        r = c.host.copy()
        r["frequency"] = i / 4
        c.keep["rules"].copy_(torch.from_numpy(r.view(np.int32)))
        c.rules = [(a, i / 4, p, h, b) for a, _, p, h, b in c.rules]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for k in range(rows):
            y, best = c.row(x[k], k, (), c.masks[k])
            assert np.array_equal(dst[k].cpu().numpy(), y) and int(chosen[k]) == best
        c.run(x[::-1].copy(), stream=st.cuda_stream)


def test_two_threads():
    """Calls of two threads, a stream each."""
    import threading
    rng = np.random.default_rng(12)
    jobs = [(draw(30011, 9, rng, 700, 8, 0.2), torch.cuda.Stream()) for _ in range(2)]
    torch.cuda.synchronize()
    out = [[torch.zeros(9, dtype=torch.int32, device="cuda") for _ in range(20)] for _ in jobs]
    src = [torch.from_numpy(x).cuda() for (_, x), _ in jobs]
    torch.cuda.synchronize()

    def work(i):
        (c, x), st = jobs[i]
        for o in out[i]:
            sq.logits_rules_dev(src[i].data_ptr(), 9, 30011, c.params, 0, o.data_ptr(), None, st.cuda_stream)

    t = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [a.start() for a in t]
    [a.join() for a in t]
    torch.cuda.synchronize()
    for i, ((c, x), _) in enumerate(jobs):
        want = [c.row(x[r], r, (), c.masks[r])[1] for r in range(9)]
        assert all(o.tolist() == want for o in out[i])
