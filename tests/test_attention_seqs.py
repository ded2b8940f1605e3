"""attention_seqs: what the causal models' attention takes as its sequence list."""
import numpy as np
import pytest

import gemma_embed as ge

ROWS = [(0, 3, 0, 5), (3, 1, 5, 0xffffffff)]


@pytest.mark.parametrize("seqs", [ROWS, tuple(ROWS), np.array(ROWS), np.array(ROWS, np.uint64), np.array(ROWS, np.uint32),
                                  np.array(ROWS, np.uint32, order="F"), np.array(ROWS * 2, np.uint32)[::2], np.array(ROWS).ravel()])
def test_whole_numbers(seqs):
    s = ge.attention_seqs(seqs)
    assert s.dtype == np.uint32 and s.flags.c_contiguous and s.shape[1] == 4
    assert np.array_equal(s, np.asarray(seqs).reshape(-1, 4))


def test_none_and_the_array_itself():
    for empty in ([], (), np.zeros((0, 4), np.uint32), np.zeros(0)):
        assert ge.attention_seqs(empty).shape == (0, 4)
    a = np.array(ROWS, np.uint32)
    assert ge.attention_seqs(a) is a


@pytest.mark.parametrize("seqs", [[(0, 1, 0, 1.5)], [(0.0, 1.0, 0.0, 1.0)], [(0, 1, 0, float("nan"))], np.zeros((2, 4), np.float32),
                                  [("0", "1", "0", "1")], [(True, True, False, True)]])
def test_other_numbers_are_refused(seqs):
    """Not cut to whole numbers."""
    with pytest.raises(TypeError):
        ge.attention_seqs(seqs)


@pytest.mark.parametrize("seqs", [[(0, 1, 0)] * 4, [(0, 1, 0, 1, 0)] * 4, np.zeros((4, 3), np.uint32), np.zeros((3, 2), np.int64),
                                  np.zeros((2, 2, 4), np.int64), np.zeros(6, np.int64)])
def test_rows_of_another_length_are_refused(seqs):
    """Not taken as others of four."""
    with pytest.raises(ValueError):
        ge.attention_seqs(seqs)


@pytest.mark.parametrize("seqs", [[(0, -1, 0, 1)], [(0, 1 << 32, 0, 1)], [(0, 1 << 63, 0, 1)]])
def test_rows_past_32_bits_are_refused(seqs):
    """Past 63 bits numpy makes floats of them."""
    with pytest.raises((OverflowError, TypeError)):
        ge.attention_seqs(seqs)
