"""GPU tests of the adapters beside a shared projection (sllm_lora_add_dev), against the formula in 64 bits.

dst = y + scale B (A x), products and sums in float32 (u = 2^-24): with T = |A| |x| the inner sums are off by at
most (cols + 2) u T (a product and an addition of each of cols terms, the scale), and the outer ones by rank + 2
roundings of |B| T more, so |dst - exact| <= u (|dst| + scale |B| T (cols + rank + 8)). Rows without an adapter keep
y's bits.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import sllm_qmm as sq

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(rows, cols, ranks, dt, seed, slots=None):
    g = torch.Generator().manual_seed(seed)
    s = sq.LoraSet(rows, cols, slots or len(ranks), max(ranks), dt)
    ad = []
    for i, r in enumerate(ranks):
        if not r:
            ad.append(None)
            continue
        a = (torch.randn(r, cols, generator=g) * cols ** -0.5).to(TORCH[dt])
        b = (torch.randn(rows, r, generator=g) * 0.3).to(TORCH[dt])
        scale = 0.25 + i
        s.load(i, a, b, scale)
        ad.append((a.double().numpy(), b.double().numpy(), scale))
    return s, ad


def check(ad, x, y, ids, got):
    x, y, got = (t.cpu().numpy() for t in (x, y, got))
    for r, i in enumerate(ids):
        if i < 0 or i >= len(ad) or ad[i] is None:
            assert np.array_equal(got[r].view(np.int32), y[r].view(np.int32)), r
            continue
        a, b, scale = ad[i]
        want = y[r] + scale * (b @ (a @ x[r].astype(np.float64)))
        size = scale * (np.abs(b) @ (np.abs(a) @ np.abs(x[r].astype(np.float64))))
        bound = U * (np.abs(want) + np.abs(y[r]) + size * (a.shape[1] + a.shape[0] + 8))
        assert (np.abs(got[r] - want) <= bound).all(), (r, i)


def run(s, ad, ids, seed, in_place=False, stream=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(len(ids), s.cols, generator=g).cuda()
    y = torch.randn(len(ids) + 1, s.rows, generator=g).cuda()
    y0 = y.clone()
    dst = y if in_place else torch.full_like(y, float("nan"))
    di = torch.tensor(ids, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    sq.lora_add_dev(s, x.data_ptr(), len(ids), di.data_ptr(), y.data_ptr(), dst.data_ptr(), stream)
    torch.cuda.synchronize()
    check(ad, x, y0[:-1], ids, dst[:-1])
    assert torch.equal(y0[-1], y[-1]) and (in_place or torch.isnan(dst[-1]).all())  # the row behind the last
    assert in_place or torch.equal(y, y0)
    return x, y0, dst


SHAPES = [
    # rows, cols, ranks
    (576, 576, [8]),
    (1, 32, [1]),
    (3, 64, [1, 2, 3]),
    (65, 96, [5, 17, 16, 15, 0, 31]),
    (257, 4128, [64, 33]),
    (1000, 2048, [7, 20, 13]),
    (4096, 4096, [16] * 8),
    (300, 14336, [128, 100]),
    (129, 160, [256, 250]),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_rows_of_a_decode_batch(shape, dt):
    rows, cols, ranks = SHAPES[shape]
    s, ad = make(rows, cols, ranks, dt, shape)
    n = len(ranks)
    rng = np.random.default_rng(shape)
    for m in (1, 2, 5, 17):
        ids = [int(i) for i in rng.integers(-1, n, size=m)]
        run(s, ad, ids, m, in_place=m == 5)
    run(s, ad, [n - 1] * 9, 3)                                    # one adapter for all
    run(s, ad, [-1, -5, n, 2 ** 31 - 1, -2 ** 31, 0], 4)          # ids that name none


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,cols,ranks", [(1000, 2048, [7, 20, 13]), (333, 544, [64, 1, 40]), (64, 4096, [200, 16])])
def test_rows_of_prompts(rows, cols, ranks, dt):
    s, ad = make(rows, cols, ranks, dt, 11)
    n = len(ranks)
    rng = np.random.default_rng(rows)
    for m in (31, 64, 65, 100, 300):
        ids = np.sort(rng.integers(-1, n, size=m))                 # rows of a request together
        run(s, ad, [int(i) for i in ids], m, in_place=m == 100)
    run(s, ad, [int(i) for i in rng.integers(-1, n, size=150)], 5)  # in any order


def test_non_finite_rows_stay_by_themselves():
    s, ad = make(200, 256, [16, 8], "f16", 3)
    for m in (4, 90):
        ids = [i % 2 for i in range(m)]
        g = torch.Generator().manual_seed(m)
        x = torch.randn(m, 256, generator=g).cuda()
        y = torch.randn(m, 200, generator=g).cuda()
        x[1, 7], x[3, 0] = float("nan"), float("inf")
        y[0, 5] = float("-inf")
        dst = torch.empty_like(y)
        di = torch.tensor(ids, dtype=torch.int32, device="cuda")
        sq.lora_add_dev(s, x.data_ptr(), m, di.data_ptr(), y.data_ptr(), dst.data_ptr())
        torch.cuda.synchronize()
        assert not torch.isfinite(dst[1]).any() and not torch.isfinite(dst[3]).any()
        assert dst[0, 5] == float("-inf") and torch.isfinite(dst[0, 6:]).all()
        rest = [r for r in range(m) if r not in (0, 1, 3)]
        check(ad, x[rest], y[rest], [ids[r] for r in rest], dst[rest])


def test_a_slot_is_loaded_again_and_emptied():
    s, ad = make(64, 128, [4, 9], "f32", 1, slots=5)
    run(s, ad + [None] * 3, [0, 1, 2, 4, -1], 1)
    a, b = np.ones((2, 128), np.float32), np.full((64, 2), 0.5, np.float32)
    s.load(1, a, b, 2.0)
    ad[1] = (a.astype(np.float64), b.astype(np.float64), 2.0)
    run(s, ad, [1, 0, 1], 2)
    s.load(0, None, None)
    run(s, [None, ad[1]], [1, 0, 1], 3)


@pytest.mark.parametrize("m", [3, 80])
def test_on_another_stream_and_in_a_graph(m):
    s, ad = make(700, 512, [16, 24, 3], "bf16", 2)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    ids = [(5 * i) % 4 - 1 for i in range(m)]
    run(s, ad, ids, 1, stream=st.cuda_stream)
    sq.workspace_reserve(st.cuda_stream, 1 << 22)
    x, y = torch.zeros(m, 512, device="cuda"), torch.zeros(m, 700, device="cuda")
    dst, di = torch.zeros(m, 700, device="cuda"), torch.zeros(m, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        sq.lora_add_dev(s, x.data_ptr(), m, di.data_ptr(), y.data_ptr(), dst.data_ptr(), st.cuda_stream)
    for rep in range(4):  # other rows, other adapters
        ids = [(i + rep) % 4 - 1 for i in range(m)]
        x.copy_(torch.randn(m, 512))
        y.copy_(torch.randn(m, 700))
        di.copy_(torch.tensor(ids, dtype=torch.int32))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(ad, x, y, ids, dst)
        run(s, ad, ids, rep)


@pytest.mark.parametrize("rows,cols,rank", [(130, 544, 12), (300, 4096, 20)])
def test_more_adapters_than_a_wave_has_lanes(rows, cols, rank):
    s, ad = make(rows, cols, [rank if i % 5 else 0 for i in range(90)], "f16", 4)
    rng = np.random.default_rng(rows)
    for m in (1, 30, 64):
        run(s, ad, [int(i) for i in rng.permutation(90)[:m]], m)                     # every row another one
    run(s, ad, [int(i) for i in rng.integers(-2, 92, size=200)], 2, in_place=True)   # up to 64 units of 64 rows


def test_calls_on_two_streams_at_once():
    sets = [make(700, 2176, [16, 24, 3], "bf16", 2), make(130, 512, [9, 40], "f32", 3)]
    st = [torch.cuda.Stream() for _ in range(2)]
    g = torch.Generator().manual_seed(1)
    jobs = []
    for i in range(24):
        s, ad = sets[i // 2 % 2]
        m = (1, 33, 90)[i % 3]
        ids = [(i + r) % 5 - 1 for r in range(m)]
        x, y = torch.randn(m, s.cols, generator=g).cuda(), torch.randn(m, s.rows, generator=g).cuda()
        jobs.append((s, ad, ids, x, y, torch.empty_like(y), torch.tensor(ids, dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()
    for i, (s, ad, ids, x, y, dst, di) in enumerate(jobs):
        sq.lora_add_dev(s, x.data_ptr(), len(ids), di.data_ptr(), y.data_ptr(), dst.data_ptr(), st[i % 2].cuda_stream)
    torch.cuda.synchronize()
    for s, ad, ids, x, y, dst, di in jobs:
        check(ad, x, y, ids, dst)


def test_refusals():
    s, _ = make(64, 128, [4], "f16", 1)
    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()
    for args in ((0, 1, p, p, p), (p, 0, p, p, p), (p, -1, p, p, p), (p, 1, 0, p, p), (p, 1, p, 0, p), (p, 1, p, p, 0),
                 (p + 4, 1, p, p, p)):
        with pytest.raises(sq.SllmError) as e:
            sq.lora_add_dev(s, *args)
        assert e.value.status == 1
    a, b = torch.zeros(4, 128, dtype=torch.float16), torch.zeros(64, 4, dtype=torch.float16)
    for slot, aa, bb in ((1, a, b), (-1, a, b), (0, a[:, :64], b), (0, a, b[:32]), (0, a.float(), b), (0, a, b.cuda()),
                         (0, torch.zeros(5, 128, dtype=torch.float16), torch.zeros(64, 5, dtype=torch.float16))):
        with pytest.raises(sq.SllmError):
            s.load(slot, aa, bb)
