"""The 4-bit form: rounding against its definition in 64 bits, and rows in and out of the 4-bit arena."""

import numpy as np
import pytest
import torch

from checks4 import dev, held, held_fast, quantize, values
from nanollvm_amd import (Context, IllegalArgumentException, KvCacheArena4, UnsupportedShapeError,
                          quantize4)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def unpack(codes):
    c = codes.cpu().numpy()
    return np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], 2 * c.shape[-1])


def edges():
    """Blocks at the borders of the form."""
    r = np.random.default_rng(3)
    rows = []
    for unit in (2.0 ** -20, 1.0, 2.0 ** 100):
        mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
        row = np.concatenate([mid, -mid, np.nextafter(np.float32(mid), np.float32(9)),
                              np.nextafter(np.float32(mid), np.float32(0)), [6, -6, 0, -0.0]])
        rows.append(row * unit)  # ties and either side of them
    for top in (1.0, 1.5, np.nextafter(np.float32(1.5), np.float32(2)), 1.999, 2.0, 6.0, 3.0):
        rows.append(np.concatenate([[top], r.uniform(-top, top, 31)]))
    rows.append(np.zeros(32))
    rows.append(np.full(32, -0.0))
    tiny = np.float32(2.0 ** -149)
    rows.append(np.full(32, tiny))
    rows.append(np.linspace(-40, 40, 32) * tiny)
    rows.append(r.uniform(-1, 1, 32) * 2.0 ** -125)   # scale byte 0 and next to it
    rows.append(r.uniform(-1, 1, 32) * 2.0 ** -123)
    big = float(np.finfo(np.float32).max)
    rows.append(np.full(32, big))
    rows.append(r.uniform(-1, 1, 32) * big)
    rows.append(np.concatenate([[big, -big, 6 * 2.0 ** 125, 5 * 2.0 ** 125], np.ones(28)]))
    rows.append(np.concatenate([[1e30, 1e-30], np.geomspace(1e-38, 1e29, 30)]))
    for odd in (np.inf, -np.inf, np.nan):
        rows.append(np.concatenate([[odd], np.ones(31)]))
        rows.append(np.concatenate([np.ones(31), [odd]]))
    return np.array(rows).astype(np.float32)


def test_the_plain_forms_agree():
    x = edges()
    x = x[np.isfinite(x).all(1)]
    assert np.array_equal(held(x), held_fast(x))


def test_borders(ctx):
    x = edges()
    codes, scales = quantize4(dev(x), ctx)
    want_codes, want_scales = quantize(x)
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(unpack(codes), want_codes)


@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (7, 5, 96), (1000, 4096), (0, 64), (33, 20000 // 32 * 32)])
def test_random_rows(ctx, shape):
    r = np.random.default_rng(sum(shape))
    x = (r.standard_normal(shape) * np.exp2(r.integers(-30, 30, shape[:-1] + (1,)))).astype(np.float32)
    codes, scales = quantize4(dev(x), ctx)
    assert codes.shape == shape[:-1] + (shape[-1] // 2,)
    assert scales.shape == shape[:-1] + (shape[-1] // 32,)
    assert np.array_equal(values(unpack(codes), scales.cpu().numpy()), held_fast(x))


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("hkv,block", [(1, 32), (3, 96), (8, 256)])
def test_arena_rows_come_back(ctx, d, hkv, block):
    """Every slot once, in any order: each holds its own row, bit for bit."""
    blocks = 3
    r = np.random.default_rng(d + hkv)
    slots = r.permutation(blocks * block).astype(np.int32)
    k, v = (r.standard_normal((len(slots), hkv, d)).astype(np.float32) for _ in range(2))
    with KvCacheArena4(ctx, 1, blocks, block, hkv, d) as arena:
        zero = [x.cpu().numpy() for x in arena.read_rows(0, dev(slots))]
        assert not np.any(zero[0]) and not np.any(zero[1])
        arena.write_rows(0, dev(slots), dev(k), dev(v))
        got = [x.cpu().numpy() for x in arena.read_rows(0, dev(slots))]
        assert np.array_equal(got[0], held_fast(k)) and np.array_equal(got[1], held_fast(v))
        # One row written again leaves the others as they are.
        one = np.full((1, hkv, d), 100.0, np.float32)
        arena.write_rows(0, dev(slots[5:6]), dev(one), dev(-one))
        again = [x.cpu().numpy() for x in arena.read_rows(0, dev(slots))]
        assert np.array_equal(again[0][5], held_fast(one)[0])
        assert np.array_equal(again[1][5], -held_fast(one)[0])
        others = np.arange(len(slots)) != 5
        assert np.array_equal(again[0][others], got[0][others])
        assert np.array_equal(again[1][others], got[1][others])


def test_slots_outside_the_arena(ctx):
    with KvCacheArena4(ctx, 2, 2, 32, 2, 64, allocate=[False, True]) as arena:
        x = np.ones((5, 2, 64), np.float32)
        slots = np.array([-1, 64, 3, 2 ** 31 - 1, -2 ** 31], np.int32)
        arena.write_rows(1, dev(slots), dev(x), dev(x))
        k, v = arena.read_rows(1, dev(slots))
        want = np.zeros_like(x)
        want[2] = 1
        assert np.array_equal(k.cpu().numpy(), want) and np.array_equal(v.cpu().numpy(), want)
        every = dev(np.arange(64, dtype=np.int32))
        assert float(arena.read_rows(1, every)[0].sum()) == 2 * 64
        arena.write_rows(1, dev(slots[:0]), dev(x[:0]), dev(x[:0]))
        assert arena.read_rows(1, dev(slots[:0]))[0].shape == (0, 2, 64)
        with pytest.raises(IllegalArgumentException):
            arena.write_rows(0, dev(slots), dev(x), dev(x))  # no pages
        with pytest.raises(IllegalArgumentException):
            arena.read_rows(2, dev(slots))


def test_blocks_that_are_not_finite(ctx):
    x = np.random.default_rng(1).standard_normal((3, 1, 128)).astype(np.float32)
    x[1, 0, 40] = np.inf
    x[2, 0, 127] = np.nan
    want = held_fast(np.nan_to_num(x, nan=0, posinf=0))
    want[1, 0, 32:64] = np.nan
    want[2, 0, 96:] = np.nan
    with KvCacheArena4(ctx, 1, 1, 32, 1, 128) as arena:
        s = dev(np.arange(3, dtype=np.int32))
        arena.write_rows(0, s, dev(x), dev(x))
        for got in arena.read_rows(0, s):
            assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


def test_the_arena_is_an_eighth(ctx):
    args = dict(num_layers=2, block_size=256, num_kv_heads=8, head_dim=128, fraction=0.5)
    blocks, free = KvCacheArena4.blocks_that_fit(ctx, **args)
    per = 2 * 256 * 8 * 128 * 2 * 34 // 64
    assert blocks == int(free * 0.5) // per


def test_refusals(ctx):
    with pytest.raises(UnsupportedShapeError):
        quantize4(torch.zeros(2, 48, device="cuda"), ctx)
    with pytest.raises(IllegalArgumentException):
        quantize4(torch.zeros(2, 64), ctx)
    with pytest.raises(IllegalArgumentException):
        quantize4(torch.zeros(2, 128, device="cuda")[:, ::2], ctx)
    with pytest.raises(IllegalArgumentException):
        quantize4(torch.zeros(2, 64, device="cuda", dtype=torch.float16), ctx)
    for d, block, what in ((96, 32, UnsupportedShapeError), (128, 16, UnsupportedShapeError),
                           (128, 0, IllegalArgumentException)):
        with pytest.raises(what):
            KvCacheArena4(ctx, 1, 1, block, 1, d)
    with KvCacheArena4(ctx, 1, 1, 32, 2, 64) as arena:
        x, s = torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
        for slots, k, v in ((s.long(), x, x), (s.cpu(), x, x), (s[:2], x, x), (s, x[:, :1], x),
                            (s, x, x.half()), (s, x.cpu(), x),
                            (torch.zeros(6, dtype=torch.int32, device="cuda")[::2], x, x)):
            with pytest.raises(IllegalArgumentException):
                arena.write_rows(0, slots, k, v)
