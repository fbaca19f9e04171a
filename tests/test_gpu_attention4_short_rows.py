"""Decode rows about the lengths up to which they are not split, of few and of many rows, against 64 bits."""

import pytest

from checks4 import close
from nanollvm_amd import Context
from test_gpu_attention4 import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("d,hq,hkv,rows,limit", [(64, 4, 1, 3, 32), (64, 8, 8, 9, 48), (128, 16, 1, 2, 32),
                                                 (128, 32, 8, 5, 48), (256, 4, 1, 5, 28), (256, 4, 1, 40, 48),
                                                 (256, 17, 1, 3, 28), (512, 8, 1, 5, 8), (512, 8, 1, 60, 12),
                                                 (512, 20, 1, 20, 12)])
def test_about_the_limit(ctx, d, hq, hkv, rows, limit):
    for extra, window in ((0, 0), (1, 0), (700, 32 * limit - 62), (700, 32 * limit - 30)):
        n = 32 * limit + extra
        lens = [n, max(1, n - 33), max(1, n // 2), 1] * (rows // 4 + 1)
        case = Case([(m - 1, 1) for m in lens[:rows]], hq, hkv, d, block=64, window=window, seed=rows)
        close(case.run(ctx), case.want(), f"{rows} rows of {n}, window {window}")
