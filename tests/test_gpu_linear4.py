"""Projections with 4-bit weights against 64 bits over the values that the weights are held as."""

import numpy as np
import pytest
import torch

from checks4 import close, dev, held_fast, values
from nanollvm_amd import (Context, IllegalArgumentException, Linear4, UnsupportedShapeError,
                          quantize4)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def data(rows, inner, outer, bias, seed):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, inner)).astype(np.float32)
    w = (r.standard_normal((outer, inner)) / np.sqrt(inner)).astype(np.float32)
    return x, w, r.standard_normal(outer).astype(np.float32) if bias else None


def want(x, w, b):
    y = x.astype(np.float64) @ held_fast(w).T
    return y if b is None else y + b


def check(ctx, rows, inner, outer, bias=False):
    x, w, b = data(rows, inner, outer, bias, rows + inner + outer)
    with Linear4.from_weight(ctx, dev(w), None if b is None else dev(b)) as lin:
        close(lin.forward(dev(x), ctx), want(x, w, b), f"{rows} x {inner} -> {outer}")


@pytest.mark.parametrize("rows", [1, 2, 5, 15, 16, 17, 31, 33, 48, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("inner,outer", [(32, 1), (96, 17), (128, 128), (160, 250), (2048, 1024)])
def test_shapes(ctx, rows, inner, outer):
    check(ctx, rows, inner, outer, bias=rows % 2 == 1)


@pytest.mark.parametrize("rows,inner,outer", [(1, 16384, 64), (3, 64, 20000), (700, 8192, 40),
                                              (1025, 544, 1000), (16, 11008, 100), (200, 32, 32),
                                              (66, 8192, 129)])
def test_long_and_wide(ctx, rows, inner, outer):
    check(ctx, rows, inner, outer)


def test_inputs_of_any_magnitude(ctx):
    """Rows 2^60 apart stay apart, and small inputs beside large ones count in full."""
    x, w, _ = data(40, 256, 48, False, 3)
    x *= np.exp2(np.linspace(-60, 60, 40)).astype(np.float32)[:, None]
    w *= np.exp2(np.linspace(-30, 30, 48)).astype(np.float32)[:, None]
    for rows in (3, 40):
        with Linear4.from_weight(ctx, dev(w)) as lin:
            got = lin.forward(dev(x[:rows]), ctx).cpu().numpy().astype(np.float64)
        ref = want(x[:rows], w, None)
        size = np.abs(x[:rows].astype(np.float64)) @ np.abs(held_fast(w)).T
        # Three exact parts a product, 3 * 256 fp32 sums at 2^-24 each.
        assert np.all(np.abs(got - ref) <= 3 * 256 * 2.0 ** -24 * size)
    x = np.zeros((1, 64), np.float32)
    x[0, 0], x[0, 1:] = 1, 2.0 ** -23
    with Linear4.from_weight(ctx, torch.ones(16, 64, device="cuda")) as lin:
        got = lin.forward(dev(x), ctx).cpu().numpy()
    assert np.all(np.abs(got - (1 + 63 * 2.0 ** -23)) <= 2.0 ** -22)


@pytest.mark.parametrize("rows", [4, 40, 100])
def test_values_that_are_not_finite(ctx, rows):
    """They reach their own row or out alone; a block of W that is NaN is NaN in its out."""
    x, w, _ = data(rows, 128, 40, False, rows)
    w = np.abs(w) + 1.0  # no code of 0, which would make NaN of an infinity
    clean = want(x, w, None)
    x[1, 5] = np.inf
    x[2, 70] = np.nan
    x[3, 127] = np.frombuffer(b"\x01\x00\x80\x7f", np.float32)[0]  # a NaN with its payload below
    w[7, 40] = np.nan
    with Linear4.from_weight(ctx, dev(w)) as lin:
        got = lin.forward(dev(x), ctx).cpu().numpy()
    assert np.isnan(got[:, 7]).all() and np.isnan(got[2]).all() and np.isnan(got[3]).all()
    others = [o for o in range(40) if o != 7]
    assert np.all(np.isposinf(got[1, others]))
    rest = [r for r in range(rows) if r not in (1, 2, 3)]
    close(got[np.ix_(rest, others)], clean[np.ix_(rest, others)])


def test_every_scale_byte_and_code(ctx):
    """Weights that come in the form: any scale byte, subnormal units included."""
    scales = np.arange(0, 253, dtype=np.uint8)[:, None]
    codes = np.tile(np.arange(32, dtype=np.uint8) % 16, (253, 1))
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    w = values(codes, scales)
    with Linear4(ctx, dev(packed), dev(scales)) as lin:
        for i in range(0, 32, 5):
            x = np.zeros((1, 32), np.float32)
            x[0, i] = 1
            got = lin.forward(dev(x), ctx).cpu().numpy()[0].astype(np.float64)
            assert np.array_equal(got, w[:, i])


def test_leading_dims_and_no_rows(ctx):
    x, w, b = data(6, 64, 24, True, 1)
    with Linear4.from_weight(ctx, dev(w), dev(b)) as lin:
        y = lin.forward(dev(x.reshape(2, 3, 64)), ctx)
        assert y.shape == (2, 3, 24)
        close(y.reshape(6, 24), want(x, w, b))
        assert lin.forward(dev(x[:0]), ctx).shape == (0, 24)
        close(lin.forward(dev(x[0]), ctx), want(x, w, b)[0])


def test_results_repeat_bit_for_bit(ctx):
    for rows in (1, 50, 200):
        x, w, _ = data(rows, 4096, 200, False, rows)
        with Linear4.from_weight(ctx, dev(w)) as lin:
            first = lin.forward(dev(x), ctx)
            for _ in range(3):
                assert torch.equal(lin.forward(dev(x), ctx), first)


@pytest.mark.parametrize("rows", [3, 40, 150])
def test_captured(ctx, rows):
    """Replays after other sizes have run through the same work area."""
    x, w, _ = data(rows, 2048, 300, False, rows)
    big, wide, _ = data(3000, 2048, 300, False, 1)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), Context(0, stream=s) as c, Linear4.from_weight(c, dev(w)) as lin:
        xin = dev(x)
        lin.forward(xin, c)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = lin.forward(xin, c)
        for turn in range(3):
            if turn == 2:
                lin.forward(dev(big), c)  # a larger work area
                xin.copy_(dev(2 * x))
            y.fill_(float("nan"))
            s.synchronize()
            g.replay()
            s.synchronize()
            close(y, want((2 if turn == 2 else 1) * x, w, None), f"replay {turn}")


def test_refusals(ctx):
    codes = torch.zeros(4, 32, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(4, 2, dtype=torch.uint8, device="cuda")
    for c, s, b in ((codes.cpu(), scales, None), (codes, scales[:, :1], None), (codes[:2], scales, None),
                    (codes.int(), scales, None), (codes[:, ::2], scales, None),
                    (codes, scales, torch.zeros(3, device="cuda")), (codes, scales, torch.zeros(4)),
                    (codes[:0], scales[:0], None)):
        with pytest.raises(IllegalArgumentException):
            Linear4(ctx, c, s, b)
    with pytest.raises(UnsupportedShapeError):
        Linear4(ctx, codes[:, :24].contiguous(), scales)  # 48 inputs
    with Linear4(ctx, codes, scales) as lin:
        for x in (torch.zeros(2, 32, device="cuda"), torch.zeros(2, 64),
                  torch.zeros(2, 64, device="cuda").double(), torch.zeros(2, 128, device="cuda")[:, ::2]):
            with pytest.raises(IllegalArgumentException):
                lin.forward(x, ctx)
    assert quantize4(torch.zeros(3, 0, device="cuda"), ctx)[0].shape == (3, 0)
