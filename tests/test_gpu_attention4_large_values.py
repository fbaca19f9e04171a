"""Values of V as large as the 4-bit form holds, over the 4-bit arena: what a query gets is a mean of them and
finite, however their scores rise along the keys and however many keys there are.  Against 64 bits, and the
blocks of 32 dims whose values are ordinary by themselves."""

import numpy as np
import pytest

from checks4 import close, dev, held_fast
from nanollvm_amd import Context
from test_gpu_attention4 import Case

pytestmark = pytest.mark.gpu

LARGEST = 6 * 2.0 ** 125


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def rising(case, rise, exponent, where):
    """Scores that rise by `rise` (in powers of two, as near as 4 bits hold them) from key tile to key tile, and
    the first 32 dims of V about 2^exponent at the keys that `where` picks by their place along the keys."""
    r = np.random.default_rng(7)
    case.q[:] = 0
    case.q[..., 0] = 1
    case.scale = float(np.float32(np.log(2.0)))
    at = 0
    for b, (c, n) in enumerate(case.seqs):
        key = np.arange(c + n)
        k = np.zeros((c + n, case.hkv, case.d), np.float32)
        k[..., 0] = (rise * (key // 32))[:, None]
        v = r.standard_normal(k.shape).astype(np.float32)
        large = where(key / (c + n))
        v[large, :, :32] = np.ldexp(r.uniform(0.5, 1, v[large, :, :32].shape), exponent)
        case.k[b], case.v[b] = k[:c], v[:c]
        case.k_new[at:at + n], case.v_new[at:at + n] = k[c:], v[c:]
        at += n


def check(case, ctx, what):
    got, want = case.run(ctx).cpu().numpy(), case.want()
    assert np.all(np.isfinite(got)), what
    close(got, want, what)
    close(got[..., 32:], want[..., 32:], what + ", ordinary dims")


EVERYWHERE = lambda at: at >= 0  # noqa: E731
EARLY = lambda at: at < 0.4  # noqa: E731
LATE = lambda at: at > 0.6  # noqa: E731

DECODE = [(399, 1), (31, 1), (64, 1), (0, 1), (3000, 1)]
PROMPTS = [(300, 40), (0, 100), (64, 3), (31, 1)]


@pytest.mark.parametrize("where", [EVERYWHERE, EARLY, LATE], ids=["everywhere", "early", "late"])
@pytest.mark.parametrize("rise", [0, 1, 20, 30])
@pytest.mark.parametrize("d,hq", [(64, 4), (128, 1), (128, 8), (128, 16), (256, 3), (256, 8), (512, 4)])
def test_decode(ctx, d, hq, rise, where):
    """Kernels of up to 4, 8 and 16 columns; rows of one workgroup and rows of many."""
    case = Case(DECODE, hq, 1, d, block=64, seed=d + hq)
    rising(case, rise, 100, where)
    check(case, ctx, f"decode {hq}/1/{d}, rise {rise}")


@pytest.mark.parametrize("where", [EVERYWHERE, EARLY, LATE], ids=["everywhere", "early", "late"])
@pytest.mark.parametrize("rise", [0, 20, 30])
@pytest.mark.parametrize("d,hq", [(64, 4), (128, 8), (256, 3), (512, 2)])
def test_prompts(ctx, d, hq, rise, where):
    case = Case(PROMPTS, hq, 1, d, block=32, seed=d + hq)
    rising(case, rise, 100, where)
    check(case, ctx, f"prompts {hq}/1/{d}, rise {rise}")


@pytest.mark.parametrize("exponent", [60, 66, 67, 68, 87, 127])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
def test_sizes_of_values(ctx, d, exponent):
    """Just within and beyond the values that are treated apart, up to the largest."""
    for seqs, hq in ((DECODE, 2), (PROMPTS, 4)):
        case = Case(seqs, hq, 1, d, block=32, seed=d)
        rising(case, 23, exponent, EVERYWHERE)
        check(case, ctx, f"2^{exponent}, d {d}")


@pytest.mark.parametrize("d", [64, 128, 256, 512])
def test_the_largest_value_at_every_key(ctx, d):
    """Keys alike: the mean is the value itself, where a sum of probabilities of 1 would pass all bounds.  The
    mean is off by its weights' sum and division: less than the path's bar of it."""
    for seqs, hq in (([(20000, 1), (500, 1)], 2), ([(0, 300), (700, 5)], 4)):
        case = Case(seqs, hq, 1, d, block=64, seed=d, fill=False)
        for x in (*case.k, case.k_new):
            x[:] = 1
        for x in (*case.v, case.v_new):
            x[:] = LARGEST
            x[..., 1::2] = -LARGEST
        assert np.all(held_fast(case.v_new) == case.v_new)
        got = case.run(ctx).cpu().numpy().astype(np.float64) / LARGEST
        close(got, np.broadcast_to(np.where(np.arange(d) % 2, -1.0, 1.0), got.shape), f"d {d}")


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [0, 50])
def test_large_values_that_no_query_sees(ctx, d, window):
    """Behind the last key and before the window they change no bit."""
    for seqs, hq in (([(199, 1), (40, 1), (0, 1)], 2), ([(100, 33), (0, 5)], 4)):
        case = Case(seqs, hq, 1, d, block=32, window=window, seed=d)
        base = case.run(ctx).cpu().numpy()
        plain = case.arena

        def arena(c):
            a = plain(c)
            seen = [case.slots(b, max(0, n - window + 1) if window else 0, n + m)
                    for b, (n, m) in enumerate(seqs)]
            rest = np.setdiff1d(np.arange(case.blocks * 32), np.concatenate(seen)).astype(np.int32)
            x = np.full((len(rest), 1, d), LARGEST, np.float32)
            a.write_rows(0, dev(rest), dev(x), dev(x))
            return a
        case.arena = arena
        assert np.array_equal(case.run(ctx).cpu().numpy(), base)
