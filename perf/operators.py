"""The operators of a batch of sequences, measured: the pages of a shared cache, the attention of a batch over
them, and low-rank adapters beside a shared projection.

Each case is one call (or one step's calls) as a server makes them of sllm_qmm: `own` is the library's entry
points, otherwise the same operator in elementary torch operations. Head layouts and widths are those of this
repository's configurations (SmolLM2-135M / 1.7B and Llama-3-8B shapes) or generic.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-5
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the smallest attention call: one sequence of a small model, one new token (latency)
        {"name": "attn_one_135m", "op": "attn", "heads": 9, "kv_heads": 3, "dk": 64, "type": "f32", "page": 16,
         "batch": 1, "prefix": 0, "own": 130, "new": 1, "extras": False},
        # a decode step of 16 unrelated sequences of different lengths, Llama-3-8B heads, f32 pages
        {"name": "attn_ragged16_8b", "op": "attn", "heads": 32, "kv_heads": 8, "dk": 128, "type": "f32", "page": 32,
         "batch": 16, "prefix": 0, "own": 1900, "new": 1, "extras": False},
        # 64 chats on one 4000-token system prompt, f16 pages
        {"name": "attn_prefix64_8b", "op": "attn", "heads": 32, "kv_heads": 8, "dk": 128, "type": "f16", "page": 64,
         "batch": 64, "prefix": 4000, "own": 300, "new": 1, "extras": False},
        # eight samples of one long document, f32 pages, with biases and QK norm
        {"name": "attn_prefix8_long", "op": "attn", "heads": 32, "kv_heads": 8, "dk": 128, "type": "f32", "page": 64,
         "batch": 8, "prefix": 16000, "own": 77, "new": 1, "extras": True},
        # prompts of several users behind a shared system prompt, of different odd lengths
        {"name": "attn_prompts5", "op": "attn", "heads": 32, "kv_heads": 8, "dk": 128, "type": "f16", "page": 64,
         "batch": 5, "prefix": 1000, "own": 1, "new": 211, "extras": False},
        # four beams of a small model: fork, write a row each, drop two, compact
        {"name": "pages_beam4_135m", "op": "pages", "layers": 30, "kv_heads": 3, "dk": 64, "type": "f32", "page": 16,
         "rows": 203, "children": 4},
        # 32 samples of one 2000-token prompt, Llama-3-8B layers: fork, write a row each, drop half, compact
        {"name": "pages_fork32_8b", "op": "pages", "layers": 32, "kv_heads": 8, "dk": 128, "type": "f16", "page": 64,
         "rows": 2023, "children": 32},
        # one request's adapter on a small projection (latency)
        {"name": "lora_one_135m", "op": "lora", "rows": 576, "cols": 576, "rank": 8, "type": "f16", "adapters": 1, "m": 1},
        # 32 requests, an adapter each, beside an 8B model's q projection
        {"name": "lora_decode32_8b", "op": "lora", "rows": 4096, "cols": 4096, "rank": 16, "type": "f16",
         "adapters": 32, "m": 32},
        # 61 requests on seven adapters, beside the FFN's up projection
        {"name": "lora_decode61_up", "op": "lora", "rows": 14336, "cols": 4096, "rank": 20, "type": "bf16",
         "adapters": 7, "m": 61},
        # prompt rows of three requests, f32 adapters of rank 64
        {"name": "lora_prompt700", "op": "lora", "rows": 4096, "cols": 14336, "rank": 64, "type": "f32",
         "adapters": 3, "m": 700},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (32, 32, 64), (9, 3, 64), (32, 4, 128), (16, 16, 80), (40, 8, 128), (8, 1, 256), (12, 12, 64)]


def _draw_attn(rng):
    h, kv, dk = rng.choice(HEADS)
    batch = _log(rng, 1, 64)
    c = {"op": "attn", "heads": h, "kv_heads": kv, "dk": dk, "type": rng.choice(["f16", "f32"]),
         "page": rng.choice([16, 32, 64, 128]), "batch": batch,
         "prefix": rng.choice([0, _log(rng, 16, 16000), _log(rng, 16, 16000)]), "own": _log(rng, 1, 2000),
         "new": rng.choice([1, 1, 1, _log(rng, 2, 250)]), "extras": rng.random() < 0.3}
    # no more positions, pairs and bytes than the listed cases have
    while c["batch"] * (c["prefix"] + c["own"]) > 280000 or _pairs(c) * h * dk > 5.5e9 or work(c)["bytes"] > 1.6e8:
        c["batch"] = max(1, c["batch"] * 2 // 3)
        c["own"] = max(1, c["own"] * 3 // 4)
        c["new"] = max(1, c["new"] * 3 // 4)
    return c


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "pages", "lora", "lora"])
    if op == "attn":
        return _draw_attn(rng)
    if op == "pages":
        _, kv, dk = rng.choice(HEADS)
        c = {"op": op, "layers": _log(rng, 1, 32), "kv_heads": kv, "dk": dk, "type": rng.choice(["f16", "f32"]),
             "page": rng.choice([16, 32, 64]), "rows": _log(rng, 1, 2000), "children": _log(rng, 2, 32)}
        while _pool_pages(c) * _page_bytes(c) > 5.6e8:
            c["layers"] = max(1, c["layers"] * 2 // 3)
            c["rows"] = max(1, c["rows"] * 2 // 3)
            c["children"] = max(2, c["children"] * 3 // 4)
        return c
    c = {"op": op, "rows": _log(rng, 64, 14336), "cols": 32 * _log(rng, 2, 448), "rank": _log(rng, 1, 64),
         "type": rng.choice(["f16", "bf16", "f32"]), "adapters": _log(rng, 1, 32), "m": _log(rng, 1, 700)}
    while work(c)["flops"] > 1.6e9 or c["adapters"] * c["rank"] > 512:
        c["adapters"] = max(1, c["adapters"] * 2 // 3)
        c["m"] = max(1, c["m"] * 3 // 4)
    return c


# ----------------------------------------------------------------- sizes ----

def _share(n, i):
    """A length of 1 .. n that sequence i takes of a case's largest one n."""
    return max(1, n * ((i * 37 + 63) % 64 + 1) // 64)


def _lens(c):
    """Per sequence: rows of its own behind the prefix, and new rows of the step."""
    own_rows = np.array([_share(c["own"], i) for i in range(c["batch"])])
    new = np.array([c["new"] if c["new"] == 1 else _share(c["new"], i) for i in range(c["batch"])])
    return own_rows, new


def _pairs(c):
    """(query row, position) pairs of a step."""
    o, n = (a.astype(np.float64) for a in _lens(c))
    return float((n * (c["prefix"] + o) + n * (n + 1) / 2).sum())


def _page_bytes(c):
    return 2 * c["layers"] * c["kv_heads"] * c["page"] * c["dk"] * DTYPES[c["type"]].itemsize


def _pool_pages(c):
    return -(-c["rows"] // c["page"]) + c["children"] + 1


def _moves(c):
    """The survivors' own pages before and after the compaction: those above the pool's used part go, in order,
    to the free ones below it."""
    base = -(-c["rows"] // c["page"])
    held = base + np.arange(0, c["children"], 2)
    used = base + len(held)
    to = held.copy()
    to[held >= used] = np.setdiff1d(np.arange(used), np.append(np.arange(base), held))
    return held, to


def _ranks(c):
    """The adapters' ranks: the case's rank and, beyond the first, some lower ones."""
    return [c["rank"] if i % 3 < 2 else max(1, c["rank"] // 2 + 1) for i in range(c["adapters"])]


def work(c):
    size = DTYPES[c["type"]].itemsize
    if c["op"] == "attn":
        o, n = _lens(c)
        kvn, qn, m = c["kv_heads"] * c["dk"], c["heads"] * c["dk"], int(n.sum())
        read = (c["prefix"] + int(o.sum())) * 2 * kvn * size
        return {"bytes": float(read + m * (8 * qn + 2 * kvn * (4 + size))), "flops": 4.0 * _pairs(c) * qn}
    if c["op"] == "pages":
        row = 2 * c["layers"] * c["kv_heads"] * c["dk"] * size
        held, to = _moves(c)
        rows = c["children"] * (c["rows"] % c["page"]) + int((held != to).sum()) * c["page"]
        return {"bytes": float(2 * row * rows + 16 * c["children"]), "flops": 0.0}
    used = set(_ids(c).tolist()) - {-1}
    r = sum(_ranks(c)[i] for i in used)
    per = np.array(_ranks(c) + [0])[_ids(c)].sum()
    return {"bytes": float(r * (c["rows"] + c["cols"]) * size + 4 * c["m"] * (c["cols"] + 2 * c["rows"])),
            "flops": 2.0 * float(per) * (c["rows"] + c["cols"])}


def _ids(c):
    """The rows' adapters: requests of a decode step in any order, a prompt's rows together; some rows have none."""
    i = np.arange(c["m"])
    a = c["adapters"]
    ids = i * a // c["m"] if c["m"] > 64 else (i * 5 + 2) % a
    return np.where(i % 11 == 10, -1, ids).astype(np.int32)


# ----------------------------------------------------------------- inputs ----

def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt * 7919 + 17) & 0x7FFFFFFF)


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _freqs(dk):
    return torch.tensor([1.0 / math.pow(10000.0, 2.0 * i / dk) for i in range(dk // 2)], dtype=torch.float32).cuda()


def _tables(c):
    """The sequences' page tables as the cache's rules give them (lowest free page first): the prefix's pages,
    then, sequence by sequence, the copy of the prefix's last page where it is not full, and further pages; the
    step's new rows come after all sequences' own ones. -1 behind a table's end."""
    p, page = c["prefix"], c["page"]
    o, n = _lens(c)
    tabs = [list(range(p // page)) for _ in range(c["batch"])]
    free = -(-p // page)
    for rows in (o, n):
        for i, t in enumerate(tabs):
            have = p + (int(o[i]) if rows is n else 0)
            more = -(-(have + int(rows[i])) // page) - len(t)
            t += range(free, free + more)
            free += more
    t = np.full((c["batch"], max(len(t) for t in tabs)), -1, np.int64)
    for i, row in enumerate(tabs):
        t[i, :len(row)] = row
    return t, free


def _attn_inputs(c, seed, pages):
    """The pool's K and V, the step's q / k / v rows and the layer's constants."""
    g = _gen(seed, 1)
    qn, kvn, m = c["heads"] * c["dk"], c["kv_heads"] * c["dk"], int(_lens(c)[1].sum())
    shape = (pages, c["kv_heads"], c["page"], c["dk"])
    d = {"K": _normal(g, *shape, std=0.7).to(DTYPES[c["type"]]), "V": _normal(g, *shape).to(DTYPES[c["type"]]),
         "q": _normal(g, m, qn), "k": _normal(g, m, kvn, std=0.7), "v": _normal(g, m, kvn), "freqs": _freqs(c["dk"])}
    if c["extras"]:
        d["qb"], d["kb"], d["vb"] = _normal(g, qn, std=0.3), _normal(g, kvn, std=0.3), _normal(g, kvn, std=0.3)
        d["qw"], d["kw"] = 1 + _normal(g, c["dk"], std=0.1), 0.7 + _normal(g, c["dk"], std=0.07)
    return d


def _pool_inputs(c, seed):
    g = _gen(seed, 2)
    shape = (c["layers"], _pool_pages(c), c["kv_heads"], c["page"], c["dk"])
    return tuple(torch.randn(*shape, generator=g, device="cuda", dtype=DTYPES[c["type"]]) for _ in range(2))


def _lora_inputs(c, seed):
    g = _gen(seed, 3)
    dt = DTYPES[c["type"]]
    pairs = [(_normal(g, r, c["cols"], std=c["cols"] ** -0.5).to(dt), _normal(g, c["rows"], r, std=0.3).to(dt), 16.0 / (r + 8 * (i % 2)))
             for i, r in enumerate(_ranks(c))]
    return pairs, _normal(g, c["m"], c["cols"]), _normal(g, c["m"], c["rows"])


class _Mem:
    """Device memory of the library's as a tensor's storage; it keeps its owner alive."""

    def __init__(self, ptr, shape, dtype, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<f4" if dtype == "f32" else "<f2",
                                         "data": (ptr, False), "version": 2}


def _lib():
    d = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scriptling-llm-lib_amd")
    if d not in sys.path:
        sys.path.insert(0, d)
    import sllm_qmm
    return sllm_qmm


def _pool_views(cache, c, layers, pages):
    k, v = cache.data()
    shape = (layers, pages, c["kv_heads"], c["page"], c["dk"])
    return tuple(torch.as_tensor(_Mem(p, shape, c["type"], cache), device="cuda") for p in (k, v))


def prepare(c, seed):
    torch.cuda.set_device(0)
    s = {"c": c}
    st = torch.cuda.current_stream().cuda_stream
    if c["op"] == "attn":
        tab, pages = _tables(c)
        o, n = _lens(c)
        s |= _attn_inputs(c, seed, pages)
        s["out"] = torch.empty(int(n.sum()), c["heads"] * c["dk"], device="cuda")
        if own:
            sq = _lib()
            cache = sq.PageCache(1, c["kv_heads"], c["dk"], c["page"], pages, c["type"])
            k, v = _pool_views(cache, c, 1, pages)
            batch = sq.PageBatch(cache, c["heads"], c["batch"], int(n.sum()))
            base = cache.add()
            cache.extend(base, c["prefix"], st)
            seqs = cache.fork(base, c["prefix"], c["batch"])
            for i in range(c["batch"]):
                cache.extend(seqs[i], int(o[i]), st)
            k[0], v[0] = s["K"], s["V"]
            batch.begin(seqs, n.tolist(), st)
            p = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
            size = lambda name: s[name].numel() if name in s else 0  # noqa: E731
            s["params"] = sq.AttnParams(
                n_heads=c["heads"], n_kv_heads=c["kv_heads"], d_k=c["dk"], rope_half_dim=c["dk"] // 2,
                rope_freqs=p("freqs"), q_bias=p("qb"), q_bias_len=size("qb"), k_bias=p("kb"), k_bias_len=size("kb"),
                v_bias=p("vb"), v_bias_len=size("vb"), q_norm_w=p("qw"), k_norm_w=p("kw"), norm_eps=EPS)
            s["K"], s["V"], s["batch"], s["stream"], s["sq"] = k[0], v[0], batch, st, sq
        else:
            # the step's description, as a program without pages would keep it
            pos = np.concatenate([c["prefix"] + o[i] + np.arange(n[i]) for i in range(c["batch"])])
            seq = np.repeat(np.arange(c["batch"]), n)
            col = np.concatenate([np.arange(n[i]) for i in range(c["batch"])])
            s["pos"], s["seq"], s["col"] = (torch.from_numpy(a).cuda() for a in (pos, seq, col))
            s["tab"] = torch.from_numpy(np.maximum(tab, 0)).cuda()
            s["most"] = int(n.max())
            s["total"] = torch.from_numpy(c["prefix"] + o + n).cuda()
    elif c["op"] == "pages":
        s["K"], s["V"] = _pool_inputs(c, seed)
        if own:
            sq = _lib()
            pages = _pool_pages(c)
            cache = sq.PageCache(c["layers"], c["kv_heads"], c["dk"], c["page"], pages, c["type"])
            batch = sq.PageBatch(cache, c["kv_heads"], c["children"], c["children"])
            k, v = _pool_views(cache, c, c["layers"], pages)
            s["base"] = cache.add()
            cache.extend(s["base"], c["rows"], st)
            k.copy_(s["K"])
            v.copy_(s["V"])
            s["K"], s["V"], s["cache"], s["batch"], s["stream"], s["held"] = k, v, cache, batch, st, []
    else:
        pairs, s["x"], s["y"] = _lora_inputs(c, seed)
        s["ids"] = torch.from_numpy(_ids(c)).cuda()
        s["dst"] = torch.empty_like(s["y"])
        if own:
            sq = _lib()
            s["set"] = sq.LoraSet(c["rows"], c["cols"], c["adapters"], c["rank"], c["type"])
            for i, (a, b, scale) in enumerate(pairs):
                s["set"].load(i, a.cpu(), b.cpu(), scale)
            s["sq"], s["stream"] = sq, st
        else:
            s["A"] = torch.cat([a for a, _, _ in pairs])
            s["B"] = torch.cat([b for _, b, _ in pairs], 1)
            s["of"] = torch.from_numpy(np.repeat(np.arange(c["adapters"]), _ranks(c))).cuda()
            s["scale"] = torch.tensor([p[2] for p in pairs], device="cuda")
    return s


# -------------------------------------------------------------------- run ----

def _rows_plain(s, x, bias, w, rotate):
    """bias, per-head RMSNorm and rotation of one step's rows of heads: (rows, heads, d_k)."""
    c = s["c"]
    if bias in s:
        x = x + s[bias]
    x = x.reshape(x.shape[0], -1, c["dk"])
    if w in s:
        x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * s[w]
    if not rotate:
        return x
    ang = (s["freqs"] * s["pos"].float()[:, None]).double()[:, None]
    cs, sn = ang.cos().float(), ang.sin().float()
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cs - b * sn, a * sn + b * cs], -1).reshape(x.shape)


def _attn_plain(s):
    c = s["c"]
    B, kv, dk, page = c["batch"], c["kv_heads"], c["dk"], c["page"]
    rep = c["heads"] // kv
    at = s["tab"][s["seq"], s["pos"] // page], s["pos"] % page
    s["K"][at[0], :, at[1]] = _rows_plain(s, s["k"], "kb", "kw", True).to(s["K"].dtype)
    s["V"][at[0], :, at[1]] = _rows_plain(s, s["v"], "vb", "", False).to(s["V"].dtype)
    K = s["K"][s["tab"]].float().permute(0, 2, 1, 3, 4).reshape(B, kv, -1, dk)
    V = s["V"][s["tab"]].float().permute(0, 2, 1, 3, 4).reshape(B, kv, -1, dk)
    there = torch.arange(K.shape[2], device="cuda")
    V = V.masked_fill((there >= s["total"][:, None])[:, None, :, None], 0.0)
    q = torch.zeros(B, s["most"], c["heads"], dk, device="cuda")
    q[s["seq"], s["col"]] = _rows_plain(s, s["q"], "qb", "qw", True)
    last = torch.zeros(B, s["most"], dtype=torch.long, device="cuda")
    last[s["seq"], s["col"]] = s["pos"]
    q = q.reshape(B, s["most"], kv, rep, dk).permute(0, 2, 3, 1, 4).reshape(B, kv, -1, dk)
    p = (q @ K.transpose(2, 3).contiguous()).reshape(B, kv, rep, s["most"], -1) / math.sqrt(dk)
    p = p.masked_fill((there > last[..., None])[:, None, None], -math.inf)
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    o = (p.reshape(B, kv, rep * s["most"], -1) @ V).reshape(B, kv, rep, s["most"], dk)
    s["out"] = o.permute(0, 3, 1, 2, 4)[s["seq"], s["col"]].reshape(-1, c["heads"] * dk)
    return s["out"], s["K"], s["V"]


def _pages_plain(s):
    c = s["c"]
    base, tail = -(-c["rows"] // c["page"]), c["rows"] % c["page"]
    kids = base + torch.arange(c["children"], device="cuda")
    held, to = _moves(c)
    src, dst = (torch.from_numpy(a[held != to]).cuda() for a in (held, to))
    if tail:
        for pool in (s["K"], s["V"]):
            pool[:, kids, :, :tail] = pool[:, base - 1:base, :, :tail].clone()
    for pool in (s["K"], s["V"]):
        pool[:, dst] = pool[:, src]
    head = np.broadcast_to(np.arange(c["rows"] // c["page"]), (len(to), c["rows"] // c["page"]))
    return s["K"], s["V"], np.concatenate([head, to[:, None]], 1).astype(np.int32)


def _lora_plain(s):
    t = s["x"] @ s["A"].float().t()
    mine = s["of"][None] == s["ids"][:, None]
    t = torch.where(mine, t * s["scale"][s["of"]], torch.zeros_like(t))
    return s["y"] + t @ s["B"].float().t()


def run(s):
    c = s["c"]
    if c["op"] == "attn":
        if own:
            s["sq"].page_attention_dev(s["batch"], 0, s["params"], s["q"].data_ptr(), s["k"].data_ptr(),
                                       s["v"].data_ptr(), s["out"].data_ptr(), s["stream"])
            return s["out"], s["K"], s["V"]
        return _attn_plain(s)
    if c["op"] == "pages":
        if own:
            cache = s["cache"]
            cache.free(s["held"])
            kids = cache.fork(s["base"], c["rows"], c["children"])
            s["batch"].begin(kids, [1] * c["children"], s["stream"])
            cache.free(kids[1::2])
            cache.compact(s["stream"])
            s["held"] = kids[0::2]
            return s["K"], s["V"], cache.tables(s["held"])
        return _pages_plain(s)
    if own:
        s["sq"].lora_add_dev(s["set"], s["x"].data_ptr(), c["m"], s["ids"].data_ptr(), s["y"].data_ptr(),
                             s["dst"].data_ptr(), s["stream"])
        return s["dst"]
    return _lora_plain(s)


# ------------------------------------------------------------------ exact ----

def _exact_rows(d, c, x, bias, w, pos):
    x = x.double()
    if bias in d:
        x = x + d[bias].double()
    x = x.reshape(len(pos), -1, c["dk"])
    if w in d:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dk"] + EPS) * d[w].double()
    # the angle is the float32 product of frequency and position
    ang = (pos.float()[:, None] * d["freqs"]).double()[:, None, :]
    z = torch.polar(torch.ones_like(ang), ang) * torch.view_as_complex(x.reshape(*x.shape[:2], -1, 2).contiguous())
    return torch.view_as_real(z).reshape(x.shape)


def _exact_attn(c, seed):
    tab, pages = _tables(c)
    o, n = _lens(c)
    d = _attn_inputs(c, seed, pages)
    K, V, outs, r = d["K"].double(), d["V"].double(), [], 0
    rep, dk, dt = c["heads"] // c["kv_heads"], c["dk"], DTYPES[c["type"]]
    for i in range(c["batch"]):
        rows = slice(r, r + int(n[i]))
        r += int(n[i])
        pos = torch.arange(c["prefix"] + int(o[i]), c["prefix"] + int(o[i]) + int(n[i]), device="cuda")
        t = torch.from_numpy(tab[i][tab[i] >= 0]).cuda()
        q, k = _exact_rows(d, c, d["q"][rows], "qb", "qw", pos), _exact_rows(d, c, d["k"][rows], "kb", "kw", pos)
        v = d["v"][rows].double()
        v = (v + d["vb"].double() if "vb" in d else v).reshape(len(pos), -1, dk)
        where = t[pos // c["page"]], pos % c["page"]
        K[where[0], :, where[1]], V[where[0], :, where[1]] = k, v
        total = int(pos[-1]) + 1
        # the attention reads the rows as the cache's type holds them
        hk, hv = (a[t].to(dt).double().transpose(0, 1).reshape(c["kv_heads"], -1, dk)[:, :total] for a in (K, V))
        mask = torch.arange(total, device="cuda")[None] > pos[:, None]
        out = torch.empty(len(pos), c["heads"], dk, dtype=torch.float64, device="cuda")
        for h in range(c["heads"]):
            w = (q[:, h] @ hk[h // rep].t().contiguous()) * dk ** -0.5
            out[:, h] = torch.softmax(w.masked_fill(mask, -math.inf), 1) @ hv[h // rep]
        outs.append(out.reshape(len(pos), -1))
    return torch.cat(outs), K, V


def _exact_pages(c, seed):
    """The pools after the step, page by page, as the rules say; copied values are exact as they are."""
    pools = _pool_inputs(c, seed)
    full, tail = divmod(c["rows"], c["page"])
    first = full + (tail > 0)
    for pool in pools:
        for i in range(c["children"] if tail else 0):
            pool[:, first + i, :, :tail] = pool[:, full, :, :tail]
        kept = list(range(first, first + c["children"], 2))
        used = first + len(kept)
        gaps = [p for p in range(first, used) if p not in kept]
        for gap, p in zip(gaps, [p for p in kept if p >= used]):
            pool[:, gap] = pool[:, p].clone()
    return (*pools, None)


def exact(c, seed):
    if c["op"] == "attn":
        return _exact_attn(c, seed)
    if c["op"] == "pages":
        return _exact_pages(c, seed)
    pairs, x, y = _lora_inputs(c, seed)
    ids, out = torch.from_numpy(_ids(c)).cuda(), y.double()
    for i, (a, b, scale) in enumerate(pairs):
        rows = (ids == i).nonzero()[:, 0]
        out[rows] += scale * ((x[rows].double() @ a.double().t().contiguous()) @ b.double().t().contiguous())
    return out
