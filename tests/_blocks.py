"""Steps whose rows fill every kind of block that the batch attention has: what they are (test_gpu_blocks.py runs them), and
what they are to plan (test_block_plans_cpu.py, by the host's code alone). From 257 workgroups on a step's blocks are as large
as its rows fill, whatever pieces are estimated to cost."""
from collections import namedtuple

import numpy as np

# parents: the kind and nodes of each sequence's tree, None: rows that follow one another (rows[i] of sequence i)
Step = namedtuple("Step", "name heads kv dk page dtype prefix owns rows trees wanted groups")


def tree(n, kind, rng):
    """Parents of n rows."""
    r = np.arange(n)
    if kind == "binary":
        return np.where(r == 0, -1, (r - 1) // 2).tolist()
    if kind == "wide":
        return np.where(r == 0, -1, np.maximum(0, r - max(1, n // 3))).tolist()
    return [-1 if i == 0 else int(rng.integers(0, i)) for i in range(n)]


def parents(step, seed=0):
    rng = np.random.default_rng(seed)
    return [tree(n, step.trees[i % len(step.trees)], rng) for i, n in enumerate(step.rows)]


def merge_groups(pieces, pairs, dk):
    """Groups of lanes that merge the states of a row's head (page attention's launch): 0 without a merge."""
    lanes = 32 if dk <= 128 else 64
    g = 256 // lanes if pieces else 0
    while g > 1 and (2 * g > pieces or pairs * g * lanes > 320000):
        g //= 2
    return g


def steps():
    """wanted: shape, tree, causal of blocks that there have to be (shapes: rows for all waves together, 16 rows of a wave, 32);
    groups: how many merge a row's states (None: not said)."""
    out = []
    for dt in ("f32", "f16"):
        for dk in (128, 96, 64, 192, 256):
            wide = 2 if dk <= 128 else 1
            # 130 rows: the last block of a prompt leaves three waves without rows
            out.append(Step(f"prompts_{dt}_{dk}", 32, 8, dk, 32, dt, 0, [20 + 7 * i for i in range(7)], [130] * 7, None,
                            {(wide, 0, 1)}, None))
            out.append(Step(f"trees61_{dt}_{dk}", 32, 8, dk, 16, dt, 0, [15 + 13 * i for i in range(17)], [61] * 17,
                            ["random", "wide", "binary"], {(wide, 1, 0)}, None))
        for dk in (128, 72):
            out.append(Step(f"short_prompts_{dt}_{dk}", 32, 8, dk, 16, dt, 0, [3 * i for i in range(40)], [12] * 40, None,
                            {(1, 0, 1)}, None))
            out.append(Step(f"trees12_{dt}_{dk}", 32, 8, dk, 16, dt, 300, [3 * i for i in range(40)], [12] * 40,
                            ["wide", "random"], {(1, 1, 0), (2, 0, 0)}, 1))
        out.append(Step(f"samples_{dt}", 32, 8, 128, 32, dt, 3000, [60 + i for i in range(12)], [13] * 12, ["binary"],
                        {(1, 1, 0), (2, 0, 0)}, 2))
        out.append(Step(f"wide_far_{dt}", 32, 8, 128, 64, dt, 0, [16000], [61], ["wide"], {(2, 1, 0)}, 4))
        out.append(Step(f"small_far_{dt}", 32, 8, 128, 64, dt, 0, [9000], [8], ["binary"], {(0, 1, 0)}, 8))
        out.append(Step(f"small_far_{dt}_192", 32, 8, 192, 64, dt, 0, [7000], [8], ["binary"], {(0 if dt == "f32" else 1, 1, 0)}, 4))
        # a tree of more rows than a piece has positions: most rows see nothing of most of its pieces
        out.append(Step(f"large_{dt}", 8, 2, 128, 32, dt, 0, [2500], [500], ["random"], {(0 if dt == "f32" else 2, 1, 0)}, 1 if dt == "f32" else 2))
    return out
