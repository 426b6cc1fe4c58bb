"""How a step's rows and positions are cut into blocks and pieces (the host's part of a step's begin)."""
import pytest

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
