"""How a step's rows and positions are cut into blocks and pieces (the host's part of a step's begin)."""
import pytest

import _blocks
from _plans import CLANG, compile_program, plan


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not CLANG:
        pytest.skip("no clang++ (vector types)")
    return compile_program(tmp_path_factory.mktemp("plans"))


@pytest.mark.parametrize("heads,kv,dk,prefix,owns,least", [
    # single rows with few workgroups: pieces of about four tiles (us measured in one piece each, and so: 18.3, 15.2; 22.3,
    # 17.8; 14.8, 13.1; 16.0, 13.9)
    (6, 2, 136, 0, [300], 3),
    (6, 2, 136, 0, [300] * 30, 3),
    (12, 12, 64, 0, [2000], 12),
    (40, 8, 128, 0, [2000], 12),
    # a prefix of many rows: 76 pieces and more of a kv head's (11 tiles each and 8: 34.9, 29.7)
    (12, 12, 64, 4000, [max(1, 150 * ((i * 37 + 63) % 64 + 1) // 64) for i in range(64)], 16),
])
def test_positions_are_cut_finely_where_pieces_are_cheap(program, heads, kv, dk, prefix, owns, least):
    assert plan(program, heads, kv, dk, "f32", 32, prefix, owns, [1] * len(owns)).pieces >= least


@pytest.mark.parametrize("step", _blocks.steps(), ids=lambda s: s.name)
def test_steps_of_the_gpu_tests_plan_their_blocks(program, step):
    """test_gpu_blocks.py reaches each kind of block, and each number of groups that merge states, by these steps."""
    p = plan(program, step.heads, step.kv, step.dk, step.dtype, step.page, step.prefix, step.owns, step.rows,
             _blocks.parents(step) if step.trees else None)
    have = {(b.shape, b.tree, b.causal) for b in p.blocks}
    assert step.wanted <= have, have
    if step.groups is not None:
        assert _blocks.merge_groups(p.pieces, sum(step.rows) * step.heads, step.dk) == step.groups, p.pieces
    if len(step.rows) > 1:  # (that other choices are not looked at does not hang on the estimate)
        rows = {(b.shape, b.tree, b.causal): 0 for b in p.blocks}
        for b in p.blocks:
            rows[b.shape, b.tree, b.causal] += b.many
        assert sum(rows.values()) * step.kv > 256
