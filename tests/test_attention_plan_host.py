"""The forms of attention's forward pass that its plan gives to the GPU tests' shapes."""

import ctypes

import pytest

from flicker_amd import _lib
from tests.attention_forms import FORMS
from tests.test_gpu_attention_forms import LONG_ROWS


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.fail("libflicker_hip.so is not built (python -m flicker_amd.build)")
    return _lib.lib()


def blocks_of(lib, sizes, backward=0):
    blocks = (ctypes.c_int * 8)(*[-1] * 8)
    assert lib.flk_attention_blocks(*sizes, backward, blocks) == 0
    return tuple(blocks)


@pytest.mark.parametrize("form", FORMS)
def test_forms(lib, form):
    sizes, want = FORMS[form]
    assert blocks_of(lib, sizes) == (*want, 0, 0, 0, 0)
    rows, whole, cut, _ = want
    batch, heads, kv_heads, queries, _ = sizes
    groups, length = (kv_heads, heads // kv_heads * queries) if rows == 16 else (heads, queries)
    assert whole + cut == batch * groups * -(-length // rows)


def test_few_rows_of_long_lists(lib):
    """Each of the four waves of a block, or of a piece, walks more than 64 units."""
    for batch, heads, keys in LONG_ROWS:
        rows, whole, cut, pieces, *_ = blocks_of(lib, (batch, heads, 1, 1, keys))
        assert rows == 16 and whole + cut == batch and (pieces > 1) == (cut > 0)
        assert -(-keys // 32) // pieces > 4 * 64


def test_backward(lib):
    """Gradients: blocks of queries and of 128 keys."""
    q_rows, q_whole, q_cut, q_pieces, k_rows, k_whole, k_cut, k_pieces = blocks_of(lib, (1, 24, 24, 4608, 4608), 1)
    assert q_rows in (192, 256) and q_whole + q_cut == 24 * -(-4608 // q_rows) and (q_pieces > 1) == (q_cut > 0)
    assert k_rows == 128 and k_whole + k_cut == 24 * 36 and (k_pieces > 1) == (k_cut > 0)


def test_nothing_and_refusals(lib):
    for sizes, backward in (((0, 2, 2, 4, 4), 0), ((1, 2, 2, 0, 4), 0), ((1, 2, 2, 4, 0), 1)):
        assert blocks_of(lib, sizes, backward) == (0,) * 8
    assert blocks_of(lib, (1, 2, 2, 4, 0))[:3] == (16, 2, 0)
    blocks = (ctypes.c_int * 8)()
    assert lib.flk_attention_blocks(1, 3, 2, 4, 4, 0, blocks) == -1 and lib.flk_attention_blocks(1, 2, 2, 4, 4, 0, None) == -1
