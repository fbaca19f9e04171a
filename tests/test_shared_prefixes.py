"""nva_find_shared_prefixes on the CPU: the runs found over step tables, against a search over every
cut of the step, and its refusals."""

import ctypes
import itertools

import numpy as np
import pytest

from nanollvm_amd import _native as N
from nanollvm_amd import step


def saving(groups, block):
    return sum((n - 1) * (t // block) for _, n, t in groups)


def common_pages(tables, cached, block, a, b):
    pages = 0
    most = min(c // block for c in cached[a:b])
    while pages < min(most, tables.shape[1]) and tables[a, pages] >= 0 and \
            len(set(tables[a:b, pages].tolist())) == 1:
        pages += 1
    return pages


def best_saving(tables, cached, block):
    n = len(cached)
    best = 0
    for cuts in itertools.product([0, 1], repeat=max(0, n - 1)):
        at, total = 0, 0
        for i in range(1, n + 1):
            if i == n or cuts[i - 1]:
                total += (i - at - 1) * common_pages(tables, cached, block, at, i)
                at = i
        best = max(best, total)
    return best


@pytest.mark.parametrize("seed", range(40))
def test_the_cut_saves_the_most_pages(seed):
    r = np.random.default_rng(seed)
    n, width, block = int(r.integers(1, 9)), int(r.integers(1, 6)), int(r.choice([1, 4, 16]))
    # Tables from a small trie, so that prefixes nest.
    tables = np.full((n, width), -1, np.int32)
    for b in range(n):
        for j in range(int(r.integers(0, width + 1))):
            tables[b, j] = 10 * j + int(r.integers(0, 2))
    cached = r.integers(0, block * width + block, n)
    got = step.find_shared_prefixes(tables, cached, block)
    at = 0
    for first, num, tokens in got:
        assert first >= at and num >= 2 and tokens > 0 and tokens % block == 0
        assert tokens // block == common_pages(tables, cached, block, first, first + num)
        at = first + num
    assert at <= n
    assert saving(got, block) == best_saving(tables, cached, block)


def test_two_prompts_and_strangers():
    tables = np.array([[7, 8, 9, 1], [7, 8, 9, 2], [7, 8, 3, -1], [4, 5, -1, -1], [6, 0, -1, -1],
                       [6, 0, -1, -1]], np.int32)
    assert step.find_shared_prefixes(tables, [50, 49, 48, 32, 32, 31], 16) == [(0, 3, 32),
                                                                               (4, 2, 16)]


def test_only_full_cached_pages_count():
    tables = np.array([[1, 2], [1, 2]], np.int32)
    assert step.find_shared_prefixes(tables, [15, 200], 16) == []
    assert step.find_shared_prefixes(tables, [16, 200], 16) == [(0, 2, 16)]
    assert step.find_shared_prefixes(tables, [1000, 200], 16) == [(0, 2, 32)]


def test_empty_steps():
    assert step.find_shared_prefixes(np.zeros((0, 3), np.int32), [], 16) == []
    assert step.find_shared_prefixes(np.zeros((3, 0), np.int32), [5, 5, 5], 16) == []
    assert step.find_shared_prefixes(np.array([[1]], np.int32), [16], 16) == []


def test_refusals():
    lib = N.load()
    t = np.zeros((2, 2), np.int32)
    c = np.zeros(2, np.int32)
    g = (N.PrefixGroup * 1)()
    n = ctypes.c_int(7)
    ok = (t.ctypes.data, 2, 2, c.ctypes.data, 16, g, ctypes.byref(n))
    assert lib.nva_find_shared_prefixes(*ok) == N.NVA_OK and n.value == 0
    for i, bad in ((0, None), (1, -1), (2, -1), (3, None), (4, 0), (5, None), (6, None)):
        args = list(ok)
        args[i] = bad
        assert lib.nva_find_shared_prefixes(*args) == N.NVA_E_ARG, i
    with pytest.raises(step.MetadataError):
        step.find_shared_prefixes(t, [1], 16)
    with pytest.raises(step.MetadataError):
        step.find_shared_prefixes(t[0], [1, 1], 16)


def test_null_contexts_are_refused():
    lib = N.load()
    assert lib.nva_step_share_prefixes(None, None, 0) == N.NVA_E_ARG
    assert lib.nva_step_set_encoder(None, None, None, 0) == N.NVA_E_ARG
    assert lib.nva_cross_attention_forward(None, None, None, None, None, 0, 0, 0,
                                           None) == N.NVA_E_ARG
    assert lib.nva_cross_attention_forward_noalloc(None, None, None, None, None, 0, 0, 0,
                                                   None) == N.NVA_E_ARG
