"""The check of held keys finds keys of other positions (planted on the host)."""

import numpy as np
import pytest

from checks4 import frequencies, held_fast, rotate
from keys4 import rounded, scale_of, wrong_keys


def test_the_form_is_the_other_restatement():
    x = np.random.default_rng(1).standard_normal((40, 2, 64)).astype(np.float32)
    mine = [rounded(b.astype(np.float64), scale_of(np.abs(b.astype(np.float64)).max()))
            for b in x.reshape(-1, 32)]
    assert np.array_equal(np.array(mine).reshape(x.shape), held_fast(x))


@pytest.mark.parametrize("interleaved", [False, True])
def test_keys_of_other_positions_are_found(interleaved):
    f, _ = frequencies(64, 1e4, "linear", 2.0)
    r = np.random.default_rng(2)
    for n in range(30):  # one token at a time, as decode steps write them
        k = r.standard_normal((1, 2, 128)).astype(np.float32)
        at = np.array([int(r.integers(1, 390))])
        held = held_fast(rotate(k, at, f, 1.0, interleaved).astype(np.float32))
        assert wrong_keys(held, k, at, f, interleaved) == 0
        for shift in (-1, 1, 2, 3):
            assert wrong_keys(held, k, at + shift, f, interleaved) >= 2, (n, shift)
        # One wrong scale of one block, a sign, a code.
        assert wrong_keys(np.concatenate([held[..., :96], 2 * held[..., 96:]], -1), k, at, f, interleaved) == 2
        turned = held.copy()
        turned[0, 1, int(np.abs(held[0, 1]).argmax())] *= -1
        assert wrong_keys(turned, k, at, f, interleaved) == 1
