"""GPU test of a batch's layer as a server runs it: projections of all rows, each request's adapter beside them, the
attention section over the shared pages, the output projection into the residual with its adapter; a prompt, its
forks, eager steps and steps of a captured graph whose begin calls stay outside.

Each stage is checked given the stage before it: projections bit for bit against single calls, adapters with the bound
of products and sums in float32 (u = 2^-24, test_gpu_lora), the attention with that of test_gpu_pages, and the
residual add with one rounding.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import sllm_qmm as sq
from test_gpu_lora import check as check_lora
from test_gpu_lora import make
from test_gpu_pages import Model, Pools, check_step

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
H, KV, DK, PROMPT, FORKS = 4, 2, 64, 45, 4
D = H * DK


class Layer:
    def __init__(self, rng, dt):
        w = lambda n: sq.quantize_q8_rows_f32((rng.normal(size=n * D) / 16).astype(np.float32), n, D)  # noqa: E731
        self.wq, self.wk, self.wv, self.wo = w(D), w(KV * DK), w(KV * DK), w(D)
        self.m = Model(H, KV, DK, 32, rng)
        self.cache = sq.PageCache(1, KV, DK, 16, 40, dt)
        self.pools = Pools(self.cache)
        self.batch = sq.PageBatch(self.cache, H, FORKS, PROMPT)
        self.lora = [make(n, D, [16, 5, 0, 30], "bf16", i) for i, n in enumerate((D, KV * DK, D))]
        f = lambda n: torch.zeros(PROMPT, n, device="cuda")  # noqa: E731
        self.x, self.res, self.att = f(D), f(D), f(D)
        self.q0, self.k, self.v0, self.q, self.v, self.res1 = f(D), f(KV * DK), f(KV * DK), f(D), f(KV * DK), f(D)
        self.ids = torch.zeros(PROMPT, dtype=torch.int32, device="cuda")

    def calls(self, n, st):
        p = lambda t: t.data_ptr()  # noqa: E731
        sq.matmul_multi_dev([self.wq, self.wk, self.wv], p(self.x), n, D, [p(self.q0), p(self.k), p(self.v0)], st)
        sq.lora_add_dev(self.lora[0][0], p(self.x), n, p(self.ids), p(self.q0), p(self.q), st)
        sq.lora_add_dev(self.lora[1][0], p(self.x), n, p(self.ids), p(self.v0), p(self.v), st)
        sq.page_attention_dev(self.batch, 0, self.m.params, p(self.q), p(self.k), p(self.v), p(self.att), st)
        sq.matmul_add_dev(self.wo, p(self.att), n, D, p(self.res), st)
        sq.lora_add_dev(self.lora[2][0], p(self.att), n, p(self.ids), p(self.res), p(self.res1), st)

    def step(self, seqs, rows, ids, rng, st, graph=None):
        n = sum(rows)
        self.batch.begin(seqs, rows, st.cuda_stream)
        st.synchronize()
        before = self.pools.host()
        x, res = (rng.normal(size=(n, D)).astype(np.float32) for _ in range(2))
        self.x[:n], self.res[:n] = torch.from_numpy(x).cuda(), torch.from_numpy(res).cuda()
        self.ids[:n] = torch.tensor(ids, dtype=torch.int32)
        self.att[n:] = float("nan")
        torch.cuda.synchronize()
        if graph is not None:
            graph.replay()
        else:
            self.calls(n, st.cuda_stream)
        torch.cuda.synchronize()
        one = torch.empty(n, D, device="cuda")
        for w, got in ((self.wq, self.q0), (self.wk, self.k), (self.wv, self.v0)):
            sq.matmul_dev(w, self.x.data_ptr(), n, D, one.data_ptr())
            torch.cuda.synchronize()
            assert torch.equal(one.flatten()[:n * w.rows].view(n, w.rows), got[:n])
        check_lora(self.lora[0][1], self.x[:n], self.q0[:n], ids, self.q[:n])
        check_lora(self.lora[1][1], self.x[:n], self.v0[:n], ids, self.v[:n])
        check_step(self.cache, self.pools, self.m, seqs, rows, self.q[:n].cpu().numpy(), self.k[:n].cpu().numpy(),
                   self.v[:n].cpu().numpy(), self.att.cpu().numpy(), before, 0)
        sq.matmul_dev(self.wo, self.att.data_ptr(), n, D, one.data_ptr())
        torch.cuda.synchronize()
        want = res.astype(np.float64) + one.cpu().numpy()
        assert (np.abs(self.res[:n].cpu().numpy() - want) <= U * np.abs(want)).all()
        check_lora(self.lora[2][1], self.att[:n], self.res[:n], ids, self.res1[:n])


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prompt_forks_and_captured_steps(dt):
    rng = np.random.default_rng(7)
    lay = Layer(rng, dt)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    base = lay.cache.add()
    lay.step([base], [PROMPT], [1] * PROMPT, rng, st)
    seqs = lay.cache.fork(base, PROMPT, FORKS)
    lay.cache.free([base])
    for i in range(2):
        lay.step(seqs, [1] * FORKS, [0, 3, -1, 1], rng, st)
    sq.workspace_reserve(st.cuda_stream, 1 << 24)
    lay.batch.begin(seqs, [1] * FORKS, st.cuda_stream)
    for s in seqs:  # (the step of the capture itself is not run)
        lay.cache.truncate(s, PROMPT + 2)
    lay.batch.begin(seqs, [1] * FORKS, st.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        lay.calls(FORKS, st.cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    for i in range(3):
        lay.step(seqs, [1] * FORKS, [i, 3, 3, -1], rng, st, graph)
    lay.cache.free(seqs[1:3])
    lay.cache.compact(st.cuda_stream)
    torch.cuda.synchronize()
    more = lay.cache.fork(seqs[0], 20, 2)
    now = [seqs[0], more[1], seqs[3], more[0]]
    lay.step(now, [1] * FORKS, [0, 1, 2, 3], rng, st, graph)
    lay.step(now, [3, 1, 2, 9], [1] * 3 + [0] + [3] * 2 + [-1] * 9, rng, st)
