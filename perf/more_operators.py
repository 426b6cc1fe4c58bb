"""The operators of drafted tokens, measured: attention of trees of drafted tokens over a page cache, the rules that
logits pass before a token is chosen, the path of a tree that the choices accept, and the move of its rows in the cache.

Each case is one call as a server makes it of sllm_qmm: `own` is the library's entry points, otherwise the same
operator in elementary torch operations. Head layouts, widths and vocabularies are those of this repository's
configurations (SmolLM2-135M / 1.7B and Llama-3-8B shapes) or generic.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-5
DTYPES = {"f32": torch.float32, "f16": torch.float16}


def listed():
    return [
        # the smallest attention call: one sequence of a small model with a few drafted tokens (latency)
        {"name": "tree_one_135m", "op": "tree", "heads": 9, "kv_heads": 3, "dk": 64, "type": "f32", "page": 16,
         "batch": 1, "prefix": 0, "own": 130, "nodes": 8, "extras": False},
        # 16 chats of different lengths with up to 16 drafted tokens each, Llama-3-8B heads, f16 pages
        {"name": "tree_ragged16_8b", "op": "tree", "heads": 32, "kv_heads": 8, "dk": 128, "type": "f16", "page": 64,
         "batch": 16, "prefix": 0, "own": 1900, "nodes": 16, "extras": False},
        # one long document with a wide tree of drafts
        {"name": "tree_long_8b", "op": "tree", "heads": 32, "kv_heads": 8, "dk": 128, "type": "f16", "page": 64,
         "batch": 1, "prefix": 0, "own": 16000, "nodes": 61, "extras": False},
        # twelve samples behind one system prompt, f32 pages, with biases and QK norm
        {"name": "tree_prefix12_8b", "op": "tree", "heads": 32, "kv_heads": 8, "dk": 128, "type": "f32", "page": 32,
         "batch": 12, "prefix": 3000, "own": 200, "nodes": 13, "extras": True},
        # the tokens of one row of a small model: a repetition penalty over a short window (latency)
        {"name": "logits_one_135m", "op": "logits", "vocab": 49152, "batch": 1, "nodes": 0, "history": 64, "biases": 0,
         "allowed": 1.0, "dst": False},
        # 64 chats with penalties over what they have written so far and a few biases; the logits are kept
        {"name": "logits_chats64_8b", "op": "logits", "vocab": 128256, "batch": 64, "nodes": 0, "history": 4000,
         "biases": 20, "allowed": 1.0, "dst": True},
        # four requests with a grammar and a tree of drafts each: few tokens are allowed at each node
        {"name": "logits_grammar_trees_8b", "op": "logits", "vocab": 128256, "batch": 4, "nodes": 16, "history": 900,
         "biases": 3, "allowed": 0.01, "dst": True},
        # an odd vocabulary, half of it allowed, the logits kept
        {"name": "logits_odd_7", "op": "logits", "vocab": 32003, "batch": 7, "nodes": 0, "history": 500, "biases": 300,
         "allowed": 0.5, "dst": True},
        # one sequence's accepted path (latency)
        {"name": "accept_one", "op": "accept", "batch": 1, "nodes": 8},
        # many sequences with wide trees
        {"name": "accept_many", "op": "accept", "batch": 200, "nodes": 64},
        # one sequence of a small model keeps three of its rows
        {"name": "keep_one_135m", "op": "keep", "layers": 30, "kv_heads": 3, "dk": 64, "type": "f32", "page": 16,
         "batch": 1, "own": 50, "nodes": 8, "kept": 3},
        # 24 sequences of an 8B model
        {"name": "keep_batch24_8b", "op": "keep", "layers": 32, "kv_heads": 8, "dk": 128, "type": "f16", "page": 16,
         "batch": 24, "own": 40, "nodes": 32, "kept": 6},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (32, 32, 64), (9, 3, 64), (32, 4, 128), (16, 16, 80), (40, 8, 128), (8, 1, 256), (12, 12, 64)]


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "logits", "logits", "accept", "keep"])
    h, kv, dk = rng.choice(HEADS)
    if op == "tree":
        c = {"op": op, "heads": h, "kv_heads": kv, "dk": dk, "type": rng.choice(["f16", "f32"]),
             "page": rng.choice([16, 32, 64, 128]), "batch": _log(rng, 1, 40),
             "prefix": rng.choice([0, 0, _log(rng, 16, 8000)]), "own": _log(rng, 1, 16000), "nodes": _log(rng, 1, 130),
             "extras": rng.random() < 0.3}
        # no more positions, pairs and bytes than the listed cases have
        while c["batch"] * (c["prefix"] + c["own"]) > 100000 or _pairs(c) * h * dk > 2.0e9 or work(c)["bytes"] > 1.2e8:
            c["batch"] = max(1, c["batch"] * 2 // 3)
            c["own"] = max(1, c["own"] * 3 // 4)
            c["nodes"] = max(1, c["nodes"] * 3 // 4)
        return c
    if op == "logits":
        c = {"op": op, "vocab": rng.choice([49152, 128256, _log(rng, 1000, 150000)]), "batch": _log(rng, 1, 64),
             "nodes": rng.choice([0, 0, _log(rng, 1, 32)]), "history": rng.choice([0, _log(rng, 1, 4000)]),
             "biases": rng.choice([0, _log(rng, 1, 300)]), "allowed": rng.choice([1.0, 1.0, 0.5, 0.1, 0.01]),
             "dst": rng.random() < 0.5}
        while c["batch"] * max(1, c["nodes"]) > 64:
            c["batch"] = max(1, c["batch"] * 2 // 3)
            c["nodes"] = c["nodes"] * 3 // 4
        return c
    if op == "accept":
        return {"op": op, "batch": _log(rng, 1, 200), "nodes": _log(rng, 1, 64)}
    c = {"op": op, "layers": _log(rng, 1, 32), "kv_heads": kv, "dk": dk, "type": rng.choice(["f16", "f32"]),
         "page": rng.choice([16, 32, 64]), "batch": _log(rng, 1, 24), "own": _log(rng, 1, 100), "nodes": _log(rng, 2, 40),
         "kept": _log(rng, 1, 8)}
    c["kept"] = min(c["kept"], (c["nodes"] + 1) // 2)
    while _tables(c)[1] * 2 * _row_bytes(c) * c["page"] > 2.6e8:
        c["layers"] = max(1, c["layers"] * 2 // 3)
        c["batch"] = max(1, c["batch"] * 3 // 4)
    return c


# ----------------------------------------------------------------- sizes ----

def _share(n, i):
    """A length of 1 .. n that sequence i takes of a case's largest one n."""
    return max(1, n * ((i * 37 + 63) % 64 + 1) // 64)


def _lens(c):
    """Per sequence: rows of its own behind the prefix, and nodes of its tree (from half of the case's number on)."""
    own_rows = np.array([_share(c.get("own", 1), i) for i in range(c["batch"])])
    nodes = np.array([c["nodes"] - (c["nodes"] // 2) * ((i * 29) % 16) // 16 for i in range(c["batch"])])
    return own_rows, nodes


def _parents(n, i):
    """Sequence i's tree of n drafted tokens, parents before children: pairs (a binary tree), some chains of the root's
    children, or one chain with side steps."""
    r = np.arange(n)
    p = [(r - 1) // 2, np.where(r <= 4, 0, r - 4), r - 1 - (r % 3 == 0)][i % 3]
    return np.where(r == 0, -1, np.maximum(p, 0))


def _ancestors(p):
    """Which nodes a node sees: itself and its ancestors."""
    a = np.eye(len(p), dtype=bool)
    for r in range(1, len(p)):
        a[r] |= a[p[r]]
    return a


def _step(c):
    """The step's rows: each one's sequence, number in it and parent there, and depth in its tree."""
    n = _lens(c)[1]
    par = [_parents(int(n[i]), i) for i in range(c["batch"])]
    seq = np.repeat(np.arange(c["batch"]), n)
    col = np.concatenate([np.arange(k) for k in n])
    depth = np.concatenate([_ancestors(p).sum(1) - 1 for p in par])
    return seq, col, np.concatenate(par), depth, par


def _pairs(c):
    """(query row, position) pairs of a step."""
    o, n = (a.astype(np.float64) for a in _lens(c))
    return float((n * (c["prefix"] + o)).sum() + (_step(c)[3] + 1).sum())


def _row_bytes(c):
    return c["layers"] * c["kv_heads"] * c["dk"] * DTYPES[c["type"]].itemsize


def work(c):
    if c["op"] == "tree":
        o, n = _lens(c)
        size, kvn, qn, m = DTYPES[c["type"]].itemsize, c["kv_heads"] * c["dk"], c["heads"] * c["dk"], int(n.sum())
        read = (c["prefix"] + int(o.sum())) * 2 * kvn * size
        return {"bytes": float(read + m * (8 * qn + 2 * kvn * (4 + size))), "flops": 4.0 * _pairs(c) * qn}
    if c["op"] == "logits":
        rows = int(_lens(c)[1].sum()) if c["nodes"] else c["batch"]
        per = 4.0 * c["vocab"] * (c["allowed"] + c["dst"]) + (c["vocab"] / 8 if c["allowed"] < 1 else 0)
        return {"bytes": rows * per + c["batch"] * (4.0 * c["history"] + 8.0 * c["biases"]), "flops": 0.0}
    if c["op"] == "accept":
        return {"bytes": float(16 * _lens(c)[1].sum() + 8 * c["batch"]), "flops": 0.0}
    moved = int((np.minimum(c["kept"], (_lens(c)[1] + 1) // 2) - 1).sum())
    return {"bytes": 4.0 * _row_bytes(c) * moved + 4.0 * int(_lens(c)[1].sum()), "flops": 0.0}


# ----------------------------------------------------------------- inputs ----

def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt * 7919 + 17) & 0x7FFFFFFF)


def _host(seed, salt):
    return np.random.RandomState((int(seed) * 1000003 + salt * 7919 + 17) & 0x7FFFFFFF)


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _freqs(dk):
    return torch.tensor([1.0 / math.pow(10000.0, 2.0 * i / dk) for i in range(dk // 2)], dtype=torch.float32).cuda()


def _tables(c):
    """The sequences' page tables as the cache's rules give them (lowest free page first): the prefix's pages,
    then, sequence by sequence, the copy of the prefix's last page where it is not full, and further pages; the
    trees' rows come after all sequences' own ones. -1 behind a table's end."""
    p, page = c.get("prefix", 0), c["page"]
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


def _tree_inputs(c, seed, pages):
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


def _logits_inputs(c, seed):
    """The logits; each request's penalties, the tokens it has written (frequent ones often) and its biases; each row's
    allowed tokens as bits, two rows in three with a mask; the tokens of the trees' nodes."""
    g, rs = _gen(seed, 2), _host(seed, 2)
    rows, v = (int(_lens(c)[1].sum()) if c["nodes"] else c["batch"]), c["vocab"]
    d = {"logits": _normal(g, rows, v, std=3.0)}
    hist = np.array([_share(c["history"], i) if c["history"] else 0 for i in range(c["batch"])])
    bias = np.array([_share(c["biases"], i) if c["biases"] else 0 for i in range(c["batch"])])
    d["history"] = np.minimum(np.exp(rs.uniform(0, math.log(v), int(hist.sum()))).astype(np.int32), v - 1)
    # (a request's biased tokens are different ones)
    d["bias_tokens"] = np.concatenate([rs.randint(0, v) + np.arange(b) * max(1, v // max(1, b)) for b in bias]).astype(np.int64) % v
    d["bias_values"] = rs.normal(size=int(bias.sum())).astype(np.float32) * 4
    some = rs.rand(3, c["batch"]).astype(np.float32)
    d["repeat"] = 1 + 0.3 * some[0]
    d["frequency"], d["presence"] = (np.where(np.arange(c["batch"]) % 2, x, 0).astype(np.float32) for x in some[1:])
    d["hist"], d["bias"] = hist, bias
    if c["allowed"] < 1:
        words = -(-v // 32)
        ok = torch.rand(rows, words * 32, generator=g, device="cuda") < c["allowed"]
        bit = ok.view(rows, words, 32).long() << torch.arange(32, device="cuda")
        d["masks"] = bit.sum(2).to(torch.int64).to(torch.int32)
        d["mask_ids"] = torch.from_numpy(np.where(np.arange(rows) % 3 == 2, -1, rs.permutation(rows)).astype(np.int32)).cuda()
    if c["nodes"]:
        d["tokens"] = torch.from_numpy(np.minimum(np.exp(rs.uniform(0, math.log(v), rows)).astype(np.int32), v - 1)).cuda()
    return d


def _accept_inputs(c, seed):
    """The nodes' tokens, and the token chosen behind each: that of one of its children more often than not."""
    rs = _host(seed, 3)
    seq, col, par, _, _ = _step(c)
    at = np.concatenate([[0], np.cumsum(_lens(c)[1])])[seq]
    tokens, chosen = (rs.randint(0, 40, len(seq)).astype(np.int32) for _ in range(2))
    r = np.nonzero((col > 0) & (rs.rand(len(seq)) < 0.7))[0]
    chosen[(at + par)[r]] = tokens[r]
    return tokens, chosen


def _keep_inputs(c, seed):
    """The pools, and the rows that each sequence keeps: its first, then later ones, behind the places they go to (those of
    a wide tree's deeper levels)."""
    g, rs = _gen(seed, 4), _host(seed, 4)
    shape = (c["layers"], _tables(c)[1], c["kv_heads"], c["page"], c["dk"])
    pools = tuple(torch.randn(*shape, generator=g, device="cuda", dtype=DTYPES[c["type"]]) for _ in range(2))
    n = _lens(c)[1]
    kept, at = np.full(int(n.sum()), -1, np.int32), 0
    for k in n:
        m = min(c["kept"], (int(k) + 1) // 2)
        kept[at:at + m] = at + np.append([0], np.sort(rs.permutation(np.arange(m, int(k)))[:m - 1]))
        at += int(k)
    return pools, kept


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


def _own_step(c, layers, heads):
    """A cache of the case's sequences and a batch with the step of their trees."""
    sq, st = _lib(), torch.cuda.current_stream().cuda_stream
    o, n = _lens(c)
    pages = _tables(c)[1]
    cache = sq.PageCache(layers, c["kv_heads"], c["dk"], c["page"], pages, c["type"])
    batch = sq.PageBatch(cache, heads, c["batch"], int(n.sum()))
    base = cache.add()
    cache.extend(base, c.get("prefix", 0), st)
    seqs = cache.fork(base, c.get("prefix", 0), c["batch"])
    for i in range(c["batch"]):
        cache.extend(seqs[i], int(o[i]), st)
    return sq, st, cache, batch, seqs, n.tolist(), _step(c)[2].tolist(), pages


def _small(c):
    """A case without a cache of its own as one with the smallest cache, whose batch holds the trees."""
    return {**c, "kv_heads": 1, "dk": 8, "page": 16, "type": "f32", "own": 1}


def prepare(c, seed):
    torch.cuda.set_device(0)
    s = {"c": c}
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    if c["op"] == "tree":
        tab, pages = _tables(c)
        s |= _tree_inputs(c, seed, pages)
        o, n = _lens(c)
        s["out"] = torch.empty(int(n.sum()), c["heads"] * c["dk"], device="cuda")
        if own:
            sq, st, cache, batch, seqs, rows, parents, _ = _own_step(c, 1, c["heads"])
            k, v = _pool_views(cache, c, 1, pages)
            k[0], v[0] = s["K"], s["V"]
            batch.begin_tree(seqs, rows, parents, st)
            p = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
            size = lambda name: s[name].numel() if name in s else 0  # noqa: E731
            s["params"] = sq.AttnParams(
                n_heads=c["heads"], n_kv_heads=c["kv_heads"], d_k=c["dk"], rope_half_dim=c["dk"] // 2,
                rope_freqs=p("freqs"), q_bias=p("qb"), q_bias_len=size("qb"), k_bias=p("kb"), k_bias_len=size("kb"),
                v_bias=p("vb"), v_bias_len=size("vb"), q_norm_w=p("qw"), k_norm_w=p("kw"), norm_eps=EPS)
            s["K"], s["V"], s["batch"], s["stream"], s["sq"] = k[0], v[0], batch, st, sq
        else:
            # the step's description, as a program without pages would keep it
            seq, col, _, depth, par = _step(c)
            start = c["prefix"] + o
            s["seq"], s["col"], s["at"], s["pos"] = (torch.from_numpy(a).cuda() for a in (seq, col, start[seq] + col, start[seq] + depth))
            s["tab"] = torch.from_numpy(np.maximum(tab, 0)).cuda()
            s["most"], s["start"] = int(n.max()), torch.from_numpy(start).cuda()
            sees = np.zeros((c["batch"], s["most"], s["most"]), bool)
            for i, p in enumerate(par):
                sees[i, :len(p), :len(p)] = _ancestors(p)
            s["sees"], s["total"] = torch.from_numpy(sees).cuda(), torch.from_numpy(start + n).cuda()
    elif c["op"] == "logits":
        d = _logits_inputs(c, seed)
        s |= {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in d.items()}
        rows = d["logits"].shape[0]
        s["chosen"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["dst"] = torch.empty_like(d["logits"]) if c["dst"] else None
        if own:
            sq = _lib()
            rules = np.zeros(c["batch"], sq.LOGITS_RULE)
            rules["repeat"], rules["frequency"], rules["presence"] = d["repeat"], d["frequency"], d["presence"]
            rules["history"], rules["biases"] = d["hist"], d["bias"]
            rules["history_at"], rules["bias_at"] = np.cumsum(d["hist"]) - d["hist"], np.cumsum(d["bias"]) - d["bias"]
            s["rules"], s["bias_tokens"] = torch.from_numpy(rules.view(np.int32)).cuda(), s["bias_tokens"].int()
            p = lambda name: s[name].data_ptr() if name in s and s[name].numel() else None  # noqa: E731
            s["params"] = sq.LogitsParams(
                rules=p("rules"), n_rules=c["batch"], history=p("history"), n_history=s["history"].numel(),
                bias_tokens=p("bias_tokens"), bias_values=p("bias_values"), n_biases=s["bias_tokens"].numel(),
                masks=p("masks"), n_masks=rows if "masks" in s else 0, mask_ids=p("mask_ids"), tokens=p("tokens"))
            s["sq"], s["stream"], s["batch"] = sq, torch.cuda.current_stream().cuda_stream, None
            if c["nodes"]:
                _, st, s["cache"], s["batch"], seqs, n, parents, _ = _own_step(_small(c), 1, 1)
                s["batch"].begin_tree(seqs, n, parents, st)
        else:
            # each row's request, and with trees the nodes (of the same request) that it sees
            if c["nodes"]:
                seq, _, _, _, par = _step(c)
                sees = np.zeros((rows, rows), bool)
                for i, p in enumerate(par):
                    at = int(_lens(c)[1][:i].sum())
                    sees[at:at + len(p), at:at + len(p)] = _ancestors(p)
                s["sees"] = torch.from_numpy(sees).cuda()
            else:
                seq = np.arange(rows)
            s["of"] = torch.from_numpy(seq).cuda()
            s["hist_of"], s["bias_of"] = (torch.from_numpy(np.repeat(np.arange(c["batch"]), d[k])).cuda() for k in ("hist", "bias"))
    elif c["op"] == "accept":
        tokens, chosen = _accept_inputs(c, seed)
        s["tokens"], s["chosen"] = i32(tokens), i32(chosen)
        seq, col, par, _, pars = _step(c)
        if own:
            sq, st, s["cache"], s["batch"], seqs, n, parents, _ = _own_step(_small(c), 1, 1)
            s["batch"].begin_tree(seqs, n, parents, st)
            s["sq"], s["stream"] = sq, st
            s["kept"] = torch.empty(len(seq), dtype=torch.int32, device="cuda")
            s["counts"], s["next"] = (torch.empty(c["batch"], dtype=torch.int32, device="cuda") for _ in range(2))
        else:
            n = _lens(c)[1]
            most = int(n.max())
            first = np.cumsum(n) - n
            sees, up = np.zeros((c["batch"], most, most), bool), np.zeros((c["batch"], most), np.int64)
            for i, p in enumerate(pars):
                sees[i, :len(p), :len(p)], up[i, :len(p)] = _ancestors(p), np.maximum(p, 0)
            s["sees"], s["up"] = torch.from_numpy(sees).cuda(), torch.from_numpy(up).cuda()
            s["seq"], s["col"], s["first"], s["n"] = (torch.from_numpy(a).cuda() for a in (seq, col, first, n))
    else:
        (s["K"], s["V"]), kept = _keep_inputs(c, seed)
        s["kept"] = i32(kept)
        if own:
            sq, st, cache, batch, seqs, n, parents, pages = _own_step(c, c["layers"], c["kv_heads"])
            batch.begin_tree(seqs, n, parents, st)
            k, v = _pool_views(cache, c, c["layers"], pages)
            k.copy_(s["K"])
            v.copy_(s["V"])
            s["K"], s["V"], s["batch"], s["stream"], s["sq"] = k, v, batch, st, sq
        else:
            seq, col = _step(c)[:2]
            at = _lens(c)[0][seq] + col
            s["page"], s["slot"] = (torch.from_numpy(a).cuda() for a in (_tables(c)[0][seq, at // c["page"]], at % c["page"]))
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


def _tree_plain(s):
    c = s["c"]
    B, kv, dk, page, most = c["batch"], c["kv_heads"], c["dk"], c["page"], s["most"]
    rep = c["heads"] // kv
    at = s["tab"][s["seq"], s["at"] // page], s["at"] % page
    s["K"][at[0], :, at[1]] = _rows_plain(s, s["k"], "kb", "kw", True).to(s["K"].dtype)
    s["V"][at[0], :, at[1]] = _rows_plain(s, s["v"], "vb", "", False).to(s["V"].dtype)
    K = s["K"][s["tab"]].float().permute(0, 2, 1, 3, 4).reshape(B, kv, -1, dk)
    V = s["V"][s["tab"]].float().permute(0, 2, 1, 3, 4).reshape(B, kv, -1, dk)
    there = torch.arange(K.shape[2], device="cuda")
    V = V.masked_fill((there >= s["total"][:, None])[:, None, :, None], 0.0)
    q = torch.zeros(B, most, c["heads"], dk, device="cuda")
    q[s["seq"], s["col"]] = _rows_plain(s, s["q"], "qb", "qw", True)
    # a row sees the cached rows before the tree, itself and its ancestors; a row that is none sees the cached ones
    node = (there - s["start"][:, None])[:, None].expand(B, most, -1)
    mine = s["sees"].gather(2, node.clamp(0, most - 1)) & (node < most)
    sees = (node < 0) | mine
    q = q.reshape(B, most, kv, rep, dk).permute(0, 2, 3, 1, 4).reshape(B, kv, -1, dk)
    p = (q @ K.transpose(2, 3).contiguous()).reshape(B, kv, rep, most, -1) / math.sqrt(dk)
    p = p.masked_fill(~sees[:, None, None], -math.inf)
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    o = (p.reshape(B, kv, rep * most, -1) @ V).reshape(B, kv, rep, most, dk)
    s["out"] = o.permute(0, 3, 1, 2, 4)[s["seq"], s["col"]].reshape(-1, c["heads"] * dk)
    return s["out"], s["K"], s["V"]


def _logits_plain(s):
    c = s["c"]
    x, B, v = s["logits"], c["batch"], c["vocab"]
    rows = x.shape[0]
    count = torch.zeros(B, v, device="cuda")
    count.index_put_((s["hist_of"], s["history"].long()), torch.ones((), device="cuda"), accumulate=True)
    count = count[s["of"]]
    if "tokens" in s:
        count.scatter_add_(1, s["tokens"].long().expand(rows, rows), s["sees"].float())
    bias = torch.zeros(B, v, device="cuda")
    bias[s["bias_of"], s["bias_tokens"]] = s["bias_values"]
    repeat, frequency, presence = (s[k][s["of"]][:, None] for k in ("repeat", "frequency", "presence"))
    y = torch.where(x > 0, x / repeat, x * repeat)
    y = y - (frequency * count + presence)
    y = torch.where(count > 0, y, x) + bias[s["of"]]
    if "masks" in s:
        ok = (s["masks"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).reshape(rows, -1)[:, :v].bool()
        y = y.masked_fill(~(ok[s["mask_ids"].clamp(min=0).long()] | (s["mask_ids"] < 0)[:, None]), -math.inf)
    # the first of the largest values that are numbers; -1 where nothing is above -inf
    z = y.masked_fill(y.isnan(), -math.inf)
    top = z.amax(1, keepdim=True)
    first = torch.where(z == top, torch.arange(v, device="cuda", dtype=torch.int32), v).amin(1)
    chosen = torch.where(top[:, 0] == -math.inf, -1, first).int()
    return (chosen, y) if c["dst"] else chosen


def _accept_plain(s):
    seq, col = s["seq"], s["col"]
    B, most = s["up"].shape
    tokens, chosen = (torch.full((B, most), f, dtype=torch.int32, device="cuda") for f in (-1, -2))
    tokens[seq, col], chosen[seq, col] = s["tokens"], s["chosen"]
    # a node follows its parent where it holds the token chosen there; of several such siblings the first
    node = torch.arange(most, device="cuda")
    like = (s["up"][:, :, None] == s["up"][:, None]) & (tokens[:, :, None] == tokens[:, None]) & (node[:, None] > node) & (node > 0)
    follows = ((chosen.gather(1, s["up"]) == tokens) & ~like.any(2)) | (node == 0)
    path = ~(s["sees"] & ~follows[:, None]).any(2) & (node < s["n"][:, None])
    count = path.sum(1)
    place = torch.where(path, path.cumsum(1) - 1, most)
    kept = torch.full((B, most + 1), -1, dtype=torch.long, device="cuda")
    kept.scatter_(1, place, s["first"][:, None] + node.expand(B, most))
    last = (path * node).amax(1, keepdim=True)
    return torch.where(kept[seq, col] >= 0, kept[seq, col], -1).int(), count.int(), chosen.gather(1, last)[:, 0]


def _keep_plain(s):
    to = (s["kept"] >= 0).nonzero()[:, 0]
    src = s["kept"][to].long()
    for pool in (s["K"], s["V"]):
        pool[:, s["page"][to], :, s["slot"][to]] = pool[:, s["page"][src], :, s["slot"][src]]
    return s["K"], s["V"]


def run(s):
    c = s["c"]
    if c["op"] == "tree":
        if own:
            s["sq"].page_attention_dev(s["batch"], 0, s["params"], s["q"].data_ptr(), s["k"].data_ptr(),
                                       s["v"].data_ptr(), s["out"].data_ptr(), s["stream"])
            return s["out"], s["K"], s["V"]
        return _tree_plain(s)
    if c["op"] == "logits":
        if own:
            s["sq"].logits_rules_dev(s["logits"].data_ptr(), s["logits"].shape[0], c["vocab"], s["params"],
                                     s["dst"].data_ptr() if c["dst"] else 0, s["chosen"].data_ptr(), s["batch"], s["stream"])
            return (s["chosen"], s["dst"]) if c["dst"] else s["chosen"]
        return _logits_plain(s)
    if c["op"] == "accept":
        if own:
            s["sq"].page_accept_dev(s["batch"], s["tokens"].data_ptr(), s["chosen"].data_ptr(), s["kept"].data_ptr(),
                                    s["counts"].data_ptr(), s["next"].data_ptr(), s["stream"])
            return s["kept"], s["counts"], s["next"]
        return _accept_plain(s)
    if own:
        s["sq"].page_keep_dev(s["batch"], s["kept"].data_ptr(), s["stream"])
        return s["K"], s["V"]
    return _keep_plain(s)


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


def _up(p, r):
    """Node r and its ancestors."""
    path = []
    while r >= 0:
        path.append(r)
        r = int(p[r])
    return path


def _exact_tree(c, seed):
    tab, pages = _tables(c)
    o, n = _lens(c)
    d = _tree_inputs(c, seed, pages)
    K, V, outs, at = d["K"].double(), d["V"].double(), [], 0
    rep, dk, dt = c["heads"] // c["kv_heads"], c["dk"], DTYPES[c["type"]]
    for i in range(c["batch"]):
        start, m, p = c["prefix"] + int(o[i]), int(n[i]), _parents(int(n[i]), i)
        rows = slice(at, at + m)
        at += m
        paths = [_up(p, r) for r in range(m)]
        pos = torch.tensor([start + len(x) - 1 for x in paths], device="cuda")
        held = torch.arange(start, start + m, device="cuda")
        t = torch.from_numpy(tab[i][tab[i] >= 0]).cuda()
        q, k = _exact_rows(d, c, d["q"][rows], "qb", "qw", pos), _exact_rows(d, c, d["k"][rows], "kb", "kw", pos)
        v = d["v"][rows].double()
        v = (v + d["vb"].double() if "vb" in d else v).reshape(m, -1, dk)
        where = t[held // c["page"]], held % c["page"]
        K[where[0], :, where[1]], V[where[0], :, where[1]] = k, v
        # the attention reads the rows as the cache's type holds them
        hk, hv = (a[t].to(dt).double().transpose(0, 1).reshape(c["kv_heads"], -1, dk)[:, :start + m] for a in (K, V))
        hidden = np.ones((m, start + m), bool)
        hidden[:, :start] = False
        for r, x in enumerate(paths):
            hidden[r, [start + y for y in x]] = False
        hidden = torch.from_numpy(hidden).cuda()
        out = torch.empty(m, c["heads"], dk, dtype=torch.float64, device="cuda")
        for h in range(c["heads"]):
            w = (q[:, h] @ hk[h // rep].t().contiguous()) * dk ** -0.5
            out[:, h] = torch.softmax(w.masked_fill(hidden, -math.inf), 1) @ hv[h // rep]
        outs.append(out.reshape(m, -1))
    return torch.cat(outs), K, V


def _exact_logits(c, seed):
    d = _logits_inputs(c, seed)
    x = d["logits"].cpu().numpy().astype(np.float64)
    v, row, chosen = c["vocab"], 0, []
    of_h, of_b = np.append(0, np.cumsum(d["hist"])), np.append(0, np.cumsum(d["bias"]))
    tokens = d["tokens"].cpu().numpy() if "tokens" in d else None
    ids = d["mask_ids"].cpu().numpy() if "masks" in d else None
    words = d["masks"].cpu().numpy() if "masks" in d else None
    for i in range(c["batch"]):
        p = _parents(int(_lens(c)[1][i]), i) if c["nodes"] else [-1]
        first = row
        for r in range(len(p)):
            count = np.bincount(d["history"][of_h[i]:of_h[i + 1]], minlength=v)
            if tokens is not None:
                np.add.at(count, tokens[first + np.array(_up(p, r))], 1)
            y, seen = x[row], count > 0
            rep, fr, pr = (float(d[k][i]) for k in ("repeat", "frequency", "presence"))
            y[seen] = np.where(y[seen] > 0, y[seen] / rep, y[seen] * rep) - fr * count[seen] - pr
            y[d["bias_tokens"][of_b[i]:of_b[i + 1]]] += d["bias_values"][of_b[i]:of_b[i + 1]]
            if ids is not None and ids[row] >= 0:
                y[np.unpackbits(words[ids[row]].view(np.uint8), bitorder="little")[:v] == 0] = -np.inf
            chosen.append(int(np.argmax(y)) if y.max() > -np.inf else -1)
            row += 1
    chosen = torch.tensor(chosen, dtype=torch.int32)
    return (chosen, torch.from_numpy(x)) if c["dst"] else chosen


def _exact_accept(c, seed):
    tokens, chosen = _accept_inputs(c, seed)
    kept, counts, after, at = np.full(len(tokens), -1, np.int32), [], [], 0
    for i, n in enumerate(_lens(c)[1]):
        p, node, path = _parents(int(n), i), 0, []
        while node is not None:
            path.append(node)
            node = next((r for r in range(node + 1, int(n)) if p[r] == node and tokens[at + r] == chosen[at + node]), None)
        kept[at:at + len(path)] = at + np.array(path)
        counts.append(len(path))
        after.append(int(chosen[at + path[-1]]))
        at += int(n)
    return torch.from_numpy(kept), torch.tensor(counts, dtype=torch.int32), torch.tensor(after, dtype=torch.int32)


def _exact_keep(c, seed):
    """The pools after the step, row by row; copied values are exact as they are."""
    pools, kept = _keep_inputs(c, seed)
    tab, o = _tables(c)[0], _lens(c)[0]
    seq, col = _step(c)[:2]
    for to in range(len(kept)):
        if kept[to] >= 0:
            i = seq[to]
            a, b = int(o[i] + col[to]), int(o[i] + col[kept[to]])
            for pool in pools:
                pool[:, tab[i, a // c["page"]], :, a % c["page"]] = pool[:, tab[i, b // c["page"]], :, b % c["page"]].clone()
    return pools


def exact(c, seed):
    return {"tree": _exact_tree, "logits": _exact_logits, "accept": _exact_accept, "keep": _exact_keep}[c["op"]](c, seed)
