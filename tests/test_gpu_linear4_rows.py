"""Projections with 4-bit weights of more rows than are taken at once."""

import numpy as np
import pytest
import torch

from checks4 import close, dev
from nanollvm_amd import Context, Linear4
from test_gpu_linear4 import data, want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [16383, 16384, 16385, 16400, 16384 + 64, 16384 + 65, 40000])
def test_rows_in_turns(rows):
    x, w, b = data(rows, 96, 40, True, rows)
    with Context(0) as ctx, Linear4.from_weight(ctx, dev(w), dev(b)) as lin:
        close(lin.forward(dev(x), ctx), want(x, w, b), f"{rows} rows")


def test_captured_turns():
    x, w, _ = data(20000, 64, 24, False, 3)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), Context(0, stream=s) as c, Linear4.from_weight(c, dev(w)) as lin:
        xin = dev(x)
        lin.forward(xin, c)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = lin.forward(xin, c)
        for turn in range(3):
            xin.copy_(dev((turn + 1) * x))
            y.fill_(float("nan"))
            s.synchronize()
            g.replay()
            s.synchronize()
            close(y, want(np.float32(turn + 1) * x, w, None), f"replay {turn}")
