"""Steps built on the device, eager and replayed, with nothing taken from the device but what is checked: the
tables, slots, positions and offsets of every step against the host's model of them, the keys that the arena
holds against those of the model's positions, and attention over them with queries at the model's positions."""

import numpy as np
import pytest
import torch

from checks4 import Tables, attention, close, dev, held_fast, rotate
from keys4 import wrong_keys
from nanollvm_amd import Context
from test_gpu_device_step import BLOCK, D, HQ, Model, i32

pytestmark = pytest.mark.gpu


class Exact(Model):
    """A layer whose twin follows from the step's numbers alone."""

    def __init__(self, ctx, rows, window=0, seed=0):
        tokens, blocks = 400, 200
        super().__init__(ctx, rows, tokens, blocks=blocks, window=window, seed=seed)
        order = np.random.default_rng(seed).permutation(blocks)  # (as the tables hand them out)
        self.plain = Tables(rows, tokens, blocks, BLOCK, order.tolist())

    def step(self, new, tokens, keep, host, out):
        before = list(self.plain.lens)
        self.tables._step = (tokens, len(new))  # (a replay's views)
        outcome = self.plain.extend(new, tokens, 400, keep)
        self.plain.check(self.tables, outcome, f"step {new}")
        (code, _), slots, positions, cu = outcome
        if code == 0:
            q, k, v = host
            used = cu[-1]
            rk, rv = (x.cpu().numpy() for x in self.arena.read_rows(0, i32(slots[:used])))
            assert np.array_equal(rv, held_fast(v[:used]))
            assert wrong_keys(rk, k[:used], positions[:used], self.f, True) == 0
            for b in range(len(new)):
                stay = before[b] if keep is None else keep[b]
                rows = slice(cu[b], cu[b + 1])
                self.keys[b] = [np.concatenate([old[:stay], x[rows].astype(np.float64)])
                                for old, x in zip(self.keys[b], (rk, rv))]
        # What earlier steps wrote is still there.
        for b, n in enumerate(self.plain.lens):
            if n:
                at, t = np.arange(n), np.asarray(self.plain.blocks[b])
                held = [x.cpu().numpy() for x in self.arena.read_rows(0, i32(t[at // BLOCK] * BLOCK + at % BLOCK))]
                assert all(np.array_equal(x, y) for x, y in zip(held, self.keys[b]))
        want = np.zeros((tokens, HQ, D))
        q = rotate(host[0], positions, self.f, 1.0, True)
        for b in range(len(new)):
            rows = slice(cu[b], cu[b + 1])
            if cu[b + 1] > cu[b]:
                k, v = self.keys[b]
                want[rows] = attention(q[rows], k, v, len(k) - (cu[b + 1] - cu[b]), D ** -0.5, self.window)
        close(out, want, f"step {new}")


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("window", [0, 40])
def test_eager_steps(fused, window):
    with Context(0) as ctx:
        m = Exact(ctx, 5, window=window, seed=11)
        for new, pad, keep in (([40, 1, 0, 33, 5], 3, None), ([1, 1, 0, 1, 1], 0, None), ([1] * 5, 1, None),
                               ([4, 1, 20, 4, 1], 0, None), ([1] * 5, 2, [42, 4, 18, 36, 7]),
                               ([0, 0, 0, 0, 70], 7, [43, 0, 19, 37, 0]), ([300] * 5, 0, None),
                               ([1, 0, 1, 1, 1], 0, None), ([0] * 5, 4, None)):
            tokens = min(sum(new) + pad, 800)
            host = m.inputs(tokens)
            ctx.extend(m.tables, i32(new), tokens, 400, None if keep is None else i32(keep))
            out, _ = m.forward(*(dev(x) for x in host), fused)
            m.step(new, tokens, keep, host, out)
        m.close()


@pytest.mark.parametrize("fused", [False, True])
def test_replayed_steps(fused):
    """Every replay of one graph is the next token of the rows that go on, after eager steps between."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), Context(0, stream=s) as ctx:
        m = Exact(ctx, 4, seed=13)

        def eager(new, tokens, keep=None):
            host = m.inputs(tokens)
            ctx.extend(m.tables, i32(new), tokens, 400, None if keep is None else i32(keep))
            out, _ = m.forward(*(dev(x) for x in host), fused)
            s.synchronize()
            m.step(new, tokens, keep, host, out)

        eager([60, 30, 7, 0], 100)
        eager([1, 1, 1, 0], 4)
        new = i32([1, 1, 1, 0])
        q, k, v = (dev(x) for x in m.inputs(4))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ctx.extend(m.tables, new, 4, 1)
            out, _ = m.forward(q, k, v, fused)
        for turn in range(12):
            if turn == 4:
                eager([0, 0, 0, 100], 110)
                new.copy_(i32([1, 0, 1, 1]))
            if turn == 8:  # a rejected draft, a row that ends, one that takes its place
                eager([2, 40, 0, 1], 43, [50, 0, 0, 99])
                new.copy_(i32([1, 1, 0, 1]))
            host = m.inputs(4)
            for t, x in zip((q, k, v), host):
                t.copy_(dev(x))
            out.fill_(float("nan"))
            s.synchronize()
            g.replay()
            s.synchronize()
            m.step(new.tolist(), 4, None, host, out)
        m.close()
