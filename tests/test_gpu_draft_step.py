"""GPU test of drafted tokens as a server uses them: a model of two attention layers and an output head whose queries,
keys and values are those of a row's token, decoded greedily with penalties, biases and masks. Sequences that draft trees
(begin_tree, attention of both layers, head, rules, accepted path, kept rows, cut) have to write the same tokens as sequences
that take one token at a time, and to hold the same rows: a row's k and v depend on its token and position alone, so the
pages agree bit for bit, as do an eager step's and a replayed one's whole numbers.

Tokens agree unless a row's two largest logits are nearly equal: sums of 2 x 128 products of sizes around 3, off by at
most 256 x 2^-24 of the sum of their sizes (about 1e-2 x 2^-6 < 1e-3) in any order; the single steps check that they differ by more.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import sllm_qmm as sq
from test_gpu_pages import Model, Pools

pytestmark = pytest.mark.gpu
H, KV, DK, LAYERS, VOCAB, PAGE, SEQS, ROWS = 4, 2, 32, 2, 96, 16, 3, 36
D = H * DK


class Server:
    def __init__(self, dt, seed):
        rng = np.random.default_rng(seed)
        self.rng, f = rng, lambda *s: rng.normal(size=s).astype(np.float32)  # noqa: E731
        self.table = [[torch.from_numpy(f(VOCAB, n)).cuda() for n in (D, KV * DK, KV * DK)] for _ in range(LAYERS)]
        self.head = sq.quantize_q8_rows_f32((f(VOCAB * D) * 2).astype(np.float32), VOCAB, D)
        self.m = Model(H, KV, DK, DK // 2, rng)
        self.dt = dt
        self.prompts = [rng.integers(0, VOCAB, n).tolist() for n in (21, 5, 40)]
        rules = np.zeros(SEQS, sq.LOGITS_RULE)
        rules["repeat"], rules["frequency"], rules["presence"] = [1.0, 1.3, 1.1], [0.0, 0.25, 0.5], [0.0, 0.125, 0.0]
        rules["history_at"] = np.arange(SEQS) * 1000
        rules["bias_at"], rules["biases"] = [0, 0, 2], [0, 2, 1]
        self.rules = rules
        self.history = torch.zeros(SEQS * 1000, dtype=torch.int32, device="cuda")
        self.bias = torch.tensor([3, 90, 7], dtype=torch.int32, device="cuda"), torch.tensor([2.0, -50.0, 1.5], device="cuda")
        # of the last sequence's rows a third of the tokens is allowed, by the token before
        bits = rng.random((VOCAB, VOCAB)) < 1 / 3
        self.masks = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).cuda()

    def open(self, max_rows):
        """A cache with the prompts but for their last tokens, which are the first step's."""
        self.cache = sq.PageCache(LAYERS, KV, DK, PAGE, 60, self.dt)
        self.pools = Pools(self.cache, 0.0)
        self.batch = sq.PageBatch(self.cache, H, SEQS, max_rows)
        z = lambda n, t=torch.float32: torch.zeros(max_rows * n, dtype=t, device="cuda")  # noqa: E731
        self.qkv = [[z(D), z(KV * DK), z(KV * DK)] for _ in range(LAYERS)]
        self.out, self.sum, self.logits = [z(D) for _ in range(LAYERS)], z(D), z(VOCAB)
        self.tokens, self.chosen, self.kept, self.ids = (z(1, torch.int32) for _ in range(4))
        self.counts, self.after = (torch.zeros(SEQS, dtype=torch.int32, device="cuda") for _ in range(2))
        self.dev_rules = torch.zeros(SEQS * 8, dtype=torch.int32, device="cuda")
        self.params = sq.LogitsParams(
            rules=self.dev_rules.data_ptr(), n_rules=SEQS, history=self.history.data_ptr(), n_history=self.history.numel(),
            bias_tokens=self.bias[0].data_ptr(), bias_values=self.bias[1].data_ptr(), n_biases=3, masks=self.masks.data_ptr(),
            n_masks=VOCAB, mask_ids=self.ids.data_ptr(), tokens=self.tokens.data_ptr())
        self.seqs = [self.cache.add() for _ in range(SEQS)]
        fill = sq.PageBatch(self.cache, H, SEQS, 80)
        fill.begin(self.seqs, [len(p) - 1 for p in self.prompts])
        t = torch.tensor(sum((p[:-1] for p in self.prompts), []), device="cuda")
        for layer in range(LAYERS):
            x = [a[t].contiguous() for a in self.table[layer]]
            out = torch.empty_like(x[0])
            torch.cuda.synchronize()
            sq.page_attention_dev(fill, layer, self.m.params, *(a.data_ptr() for a in x), out.data_ptr())
            torch.cuda.synchronize()
        self.written = [list(p) for p in self.prompts]

    def calls(self, rows, st, keep):
        p = lambda t: t.data_ptr()  # noqa: E731
        for layer in range(LAYERS):
            sq.page_attention_dev(self.batch, layer, self.m.params, *(p(a) for a in self.qkv[layer]), p(self.out[layer]), st)
        sq.matmul_dev(self.head, p(self.out[0]), rows, D, p(self.logits), st)
        sq.matmul_add_dev(self.head, p(self.out[1]), rows, D, p(self.logits), st)
        sq.logits_rules_dev(p(self.logits), rows, VOCAB, self.params, 0 if keep else p(self.logits), p(self.chosen), self.batch, st)
        if keep:
            sq.page_accept_dev(self.batch, p(self.tokens), p(self.chosen), p(self.kept), p(self.counts), p(self.after), st)
            sq.page_keep_dev(self.batch, p(self.kept), st)

    def inputs(self, tokens):
        """The step's rows: what a program would put up before the calls."""
        n = len(tokens)
        t = torch.tensor(tokens, device="cuda")
        self.tokens[:n] = t.int()
        for layer in range(LAYERS):
            for buf, a in zip(self.qkv[layer], self.table[layer]):
                buf.view(-1, a.shape[1])[:n] = a[t]
        rules = self.rules.copy()
        for i, w in enumerate(self.written):
            self.history[1000 * i:1000 * i + len(w) - 1] = torch.tensor(w[:-1], dtype=torch.int32)
            rules["history"][i] = len(w) - 1  # (the last one is the step's first)
        self.dev_rules.copy_(torch.from_numpy(rules.view(np.int32)))

    def plain(self, steps):
        self.open(SEQS)
        for _ in range(steps):
            self.batch.begin(self.seqs, [1] * SEQS)
            self.inputs([w[-1] for w in self.written])
            self.ids[:SEQS] = torch.tensor([-1, -1, self.written[2][-1]], dtype=torch.int32)
            torch.cuda.synchronize()
            self.calls(SEQS, 0, False)
            torch.cuda.synchronize()
            two = self.logits.view(SEQS, VOCAB).topk(2).values
            assert (two[:, 0] - two[:, 1] > 1e-3).all()  # (any order of the sums chooses the same)
            for w, c in zip(self.written, self.chosen[:SEQS].tolist()):
                w.append(c)
        return self.written, [self.pools.read(s) for s in self.seqs]

    def draft(self, w, truth, wide):
        """A tree behind a sequence's last token: the tokens that it will write, some of them, and others beside them."""
        n = int(self.rng.integers(1, ROWS // SEQS + 1))
        tokens, parents = [w[-1]], [-1]
        on, at = 0, len(w)  # the node that has been right so far
        while len(tokens) < n:
            right = at < len(truth) and self.rng.random() < 0.7
            parents.append(on if right else int(self.rng.integers(0, len(tokens))) if wide else len(tokens) - 1)
            tokens.append(truth[at] if right else int(self.rng.integers(0, VOCAB)))
            if right:
                on, at = len(tokens) - 1, at + 1
        return tokens, parents

    def drafted(self, truth, wide, graph):
        self.open(ROWS)
        st = torch.cuda.Stream()
        s = st.cuda_stream
        sq.workspace_reserve(s, 1 << 24)
        rec, steps, kept_rows = None, 0, 0
        while min(len(w) for w in self.written) < min(len(t) for t in truth):
            trees = [self.draft(w, t, wide) for w, t in zip(self.written, truth)]
            base = [self.cache.length(q) for q in self.seqs]
            rows = [len(t) for t, _ in trees]
            self.batch.begin_tree(self.seqs, rows, sum((p for _, p in trees), []), s)
            if graph and rec is None:
                torch.cuda.synchronize()
                rec = torch.cuda.CUDAGraph()
                with torch.cuda.graph(rec, stream=st):
                    self.calls(ROWS, s, True)
                torch.cuda.synchronize()
            tokens = sum((t for t, _ in trees), [])
            self.inputs(tokens)
            last = rows[0] + rows[1]
            self.ids[:last] = -1
            self.ids[last:last + rows[2]] = torch.tensor(tokens[last:], dtype=torch.int32)
            torch.cuda.synchronize()
            if rec is not None:
                rec.replay()
            else:
                self.calls(sum(rows), s, True)
            torch.cuda.synchronize()
            kept, counts, after = (t.tolist() for t in (self.kept, self.counts, self.after))
            at = 0
            for i, q in enumerate(self.seqs):
                path = kept[at:at + counts[i]]
                assert path[0] == at and kept[at + counts[i]:at + rows[i]] == [-1] * (rows[i] - counts[i])
                self.written[i] += [tokens[r] for r in path[1:]] + [after[i]]
                self.cache.truncate(q, base[i] + counts[i])
                at += rows[i]
                kept_rows += counts[i]
            steps += 1
        return kept_rows / steps / SEQS


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("wide", [True, False], ids=["trees", "chains"])
@pytest.mark.parametrize("graph", [False, True], ids=["eager", "replayed"])
def test_drafted_tokens_are_those_of_single_steps(dt, wide, graph):
    srv = Server(dt, 5)
    truth, held = srv.plain(60)
    truth = [list(w) for w in truth]
    per_step = srv.drafted(truth, wide, graph)
    assert per_step > 1.5  # (drafts were accepted)
    for i, (w, t) in enumerate(zip(srv.written, truth)):
        n = min(len(w), len(t))
        assert w[:n] == t[:n], i
        rows = min(srv.cache.length(srv.seqs[i]), held[i][0].shape[1])
        assert rows >= n - 1
        for a, b in zip(srv.pools.read(srv.seqs[i]), held[i]):
            assert np.array_equal(a[:, :rows].view(np.uint8), b[:, :rows].view(np.uint8)), i
