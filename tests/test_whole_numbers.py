"""Step metadata that 32 bits do not hold is refused before the library sees it: a cast would make other
sequences, rows or pages of it."""

import numpy as np
import pytest

from nanollvm_amd import Context, IllegalArgumentException, _native as N, step

BAD = [[2 ** 32], np.array([2 ** 31]), np.array([-2 ** 31 - 1]), np.array([2 ** 32 + 3], np.uint64),
       [1.5], [float("nan")], np.array([1e10]), ["a"], [2 ** 70]]


def bare_context():
    c = Context.__new__(Context)
    c._h = None
    return c


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_values_beyond_int32(bad):
    with pytest.raises(ValueError):
        N.i32(bad)
    c = bare_context()
    value = np.asarray(bad).tolist()[0]
    with pytest.raises(IllegalArgumentException):
        c.set_encoder(bad, [4])
    with pytest.raises(IllegalArgumentException):
        c.set_encoder([4], bad)
    for group in ((value, 2, 64), (0, value, 64), (0, 2, value)):
        with pytest.raises(IllegalArgumentException):
            c.share_prefixes([group])
    with pytest.raises(IllegalArgumentException):
        c.set(is_prefill=False, context_lens=bad)
    with pytest.raises(IllegalArgumentException):
        c.set(is_prefill=False, context_lens=[1], block_tables=np.asarray([bad]))
    table = np.zeros((1, 4), np.int32)
    with pytest.raises(step.MetadataError):
        step.find_shared_prefixes(table, bad, 16)
    with pytest.raises(step.MetadataError):
        step.find_shared_prefixes(np.asarray([bad]), [1], 16)
    with pytest.raises(step.MetadataError):
        step.find_shared_prefixes(table, [1], value)


def test_groups_of_other_shapes():
    c = bare_context()
    for bad in ([(0, 2)], [(0, 2, 64, 1)], [(0, 2, 64), (2, 2)], [3]):
        with pytest.raises(IllegalArgumentException):
            c.share_prefixes(bad)


def test_values_that_fit():
    for good in ([2 ** 31 - 1, -2 ** 31], np.array([5, 7], np.int64), np.array([1.0, 2.0]), [],
                 np.arange(6).reshape(2, 3)[:, ::2], [True]):
        got = N.i32(good)
        assert got.dtype == np.int32 and got.flags.c_contiguous
        assert np.array_equal(got, np.asarray(good))
    table = np.tile(np.arange(4), (3, 1))
    assert step.find_shared_prefixes(table, np.array([40, 41, 42], np.int64), 16) == [(0, 3, 32)]
