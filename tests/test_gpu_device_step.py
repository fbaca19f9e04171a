"""Steps built on the device as they are used: block tables, rotary positions, the 4-bit arena's
attention and a 4-bit projection one after the other, eager and captured, against 64 bits."""

import numpy as np
import pytest
import torch

from checks4 import Tables, attention, close, dev, frequencies, held_fast, rotate
from nanollvm_amd import (Attention, BlockTables, Context, IllegalArgumentException, KvCacheArena4,
                          Linear4, RotaryEmbedding)

pytestmark = pytest.mark.gpu

HQ, HKV, D, BLOCK, OUT = 8, 2, 128, 32, 96


def i32(x):
    return dev(np.asarray(x, np.int32))


class Model:
    """One attention layer over device-built steps, and its 64-bit twin."""

    def __init__(self, ctx, rows, max_tokens=400, step=800, blocks=200, window=0, seed=0):
        self.ctx, self.rows = ctx, rows
        r = self.r = np.random.default_rng(seed)
        self.window = window
        self.tables = BlockTables(ctx, rows, max_tokens, step, blocks, BLOCK,
                                  r.permutation(blocks))
        self.plain = Tables(rows, max_tokens, blocks, BLOCK)
        self.arena = KvCacheArena4(ctx, 1, blocks, BLOCK, HKV, D)
        self.rope = RotaryEmbedding.scaled(ctx, D, 64, max_tokens, 1e4, interleaved=True,
                                           scaling="linear", factor=2.0)
        self.f, _ = frequencies(64, 1e4, "linear", 2.0)
        self.w = (r.standard_normal((OUT, HQ * D)) / 32).astype(np.float32)
        self.proj = Linear4.from_weight(ctx, dev(self.w))
        self.layer = Attention(HQ, D, D ** -0.5, HKV, window)
        self.keys = [[np.zeros((0, HKV, D))] * 2 for _ in range(rows)]

    def inputs(self, tokens):
        return [self.r.standard_normal((tokens, h, D)).astype(np.float32) for h in (HQ, HKV, HKV)]

    def forward(self, q, k, v, fused):
        self.ctx.bind_kv_cache(self.arena)
        if fused:
            out = self.layer.forward_with_rope(self.rope, None, q, k, v, self.ctx)
        else:
            q, k = self.rope.forward(None, q, k, self.ctx)
            out = self.layer.forward(q, k, v, self.ctx)
        return out, self.proj.forward(out.view(len(q), -1), self.ctx)

    def advance(self, new, tokens, keep, k, v):
        """The keys and values of every sequence after the step."""
        before = list(self.plain.lens)
        (code, _), _, positions, cu = self.plain.extend(new, tokens, 400, keep)
        if code:
            return
        k = rotate(k, positions, self.f, 1.0, True).astype(np.float32)
        for b in range(len(new)):
            stay = before[b] if keep is None else keep[b]
            rows = slice(cu[b], cu[b + 1])
            self.keys[b] = [np.concatenate([old[:stay], held_fast(x[rows])])
                            for old, x in zip(self.keys[b], (k, v))]

    def held_keys(self):
        """Takes the rows that the arena holds, so that one code's border in k is not compared."""
        t = self.tables.block_tables.cpu().numpy()
        for b, n in enumerate(self.plain.lens):
            if n:
                at = np.arange(n)
                slots = i32(t[b][at // BLOCK] * BLOCK + at % BLOCK)
                k, v = (x.cpu().numpy().astype(np.float64) for x in self.arena.read_rows(0, slots))
                assert np.array_equal(v, self.keys[b][1])
                # The fp32 rotation differs from the 64-bit one in its last bits: a code, or the
                # scale of one block of 32, only where a value lies that near a border.
                assert np.sum(k != self.keys[b][0]) <= 32
                self.keys[b][0] = k

    def close(self):
        for x in (self.proj, self.rope, self.arena, self.tables):
            x.close()


def project(m, out):
    return out.reshape(len(out), -1) @ held_fast(m.w).T


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("window", [0, 40])
def test_a_service(fused, window):
    """Prompts, decode steps with idle rows, a rejected draft, a request that ends and one that takes its
    row, padding, and a step that does not fit."""
    with Context(0) as ctx:
        m = Model(ctx, 5, window=window)
        for new, pad, keep in (([70, 1, 0, 33, 5], 3, None), ([1, 1, 0, 1, 1], 0, None),
                               ([4, 1, 20, 4, 1], 0, None), ([1] * 5, 2, [73, 3, 18, 36, 7]),
                               ([0, 0, 0, 0, 90], 7, [74, 0, 19, 37, 0]),
                               ([300, 300, 300, 300, 300], 0, None), ([1, 0, 1, 1, 1], 0, None),
                               ([0] * 5, 4, None)):
            tokens = min(sum(new) + pad, 800)
            q, k, v = m.inputs(tokens)
            ctx.extend(m.tables, i32(new), tokens, 400, None if keep is None else i32(keep))
            out, y = m.forward(dev(q), dev(k), dev(v), fused)
            m.advance(new, tokens, keep, k, v)
            m.held_keys()
            close_to_held(m, new, tokens, q, out)
            close(y, project(m, out.cpu().numpy().astype(np.float64)), "projection")
            got = out.cpu().numpy()
            used = int(m.tables.cu_q[-1])
            assert not np.any(got[used:])
        m.close()


def close_to_held(m, new, tokens, q, out):
    """out against attention over the keys that the arena holds."""
    cu = m.tables.cu_q.tolist()
    pos = m.tables.positions.cpu().numpy()
    q = rotate(q, pos, m.f, 1.0, True)
    want = np.zeros((tokens, HQ, D))
    for b in range(m.rows):
        rows = slice(cu[b], cu[b + 1])
        n = cu[b + 1] - cu[b]
        if n:
            k, v = m.keys[b]
            want[rows] = attention(q[rows], k, v, len(k) - n, D ** -0.5, m.window)
    close(out, want, f"step {new}")


def test_captured_decode_grows():
    """One graph of extend, rotation, attention and projection: every replay serves the next token, over
    new blocks and idle rows, with eager prompts between."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), Context(0, stream=s) as ctx:
        m = Model(ctx, 4, seed=3)
        def eager(new, tokens, keep=None):
            q, k, v = m.inputs(tokens)
            ctx.extend(m.tables, i32(new), tokens, 400, None if keep is None else i32(keep))
            out, _ = m.forward(dev(q), dev(k), dev(v), True)
            m.advance(new, tokens, keep, k, v)
            s.synchronize()
            m.held_keys()
            close_to_held(m, new, tokens, q, out)
        eager([60, 30, 7, 0], 100)
        eager([1, 1, 1, 0], 4)
        new = i32([1, 1, 1, 0])
        q, k, v = (dev(x) for x in m.inputs(4))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ctx.extend(m.tables, new, 4, 1)
            out, y = m.forward(q, k, v, True)
        for turn in range(45):
            if turn == 20:
                eager([0, 0, 0, 250], 260)  # more rows and keys than the captured step's
                new.copy_(i32([1, 0, 1, 1]))
            host = m.inputs(4)
            for t, x in zip((q, k, v), host):
                t.copy_(dev(x))
            out.fill_(float("nan"))
            s.synchronize()
            g.replay()
            s.synchronize()
            n = new.tolist()
            m.advance(n, 4, None, *host[1:])
            m.tables._step = (4, 4)
            m.held_keys()
            close_to_held(m, n, 4, host[0], out)
            close(y, project(m, out.cpu().numpy().astype(np.float64)), f"replay {turn}")
        assert m.tables.status()[0] == 0
        m.close()


def test_two_graphs_share_the_work_areas():
    """Graphs of two layers and two batch sizes, replayed in turn after a larger eager step has replaced
    the work areas."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), Context(0, stream=s) as ctx:
        models = [Model(ctx, n, seed=n) for n in (3, 6)]
        graphs = []
        for m in models:
            new = [20 + 9 * i for i in range(m.rows)]
            q, k, v = m.inputs(sum(new))
            ctx.extend(m.tables, i32(new), sum(new), 400)
            m.forward(dev(q), dev(k), dev(v), True)
            m.advance(new, sum(new), None, k, v)
            one = i32([1] * m.rows)
            q, k, v = (dev(x) for x in m.inputs(m.rows))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                ctx.extend(m.tables, one, m.rows, 1)
                out, _ = m.forward(q, k, v, True)
            graphs.append((g, q, k, v, out, one))
        big = Model(ctx, 9, step=3000, blocks=900, seed=7)
        new = [300] * 9
        q, k, v = big.inputs(2700)
        ctx.extend(big.tables, i32(new), 2700, 400)
        big.forward(dev(q), dev(k), dev(v), True)
        for turn in range(4):
            for m, (g, q, k, v, out, _) in zip(models, graphs):
                out.fill_(float("nan"))
                s.synchronize()
                g.replay()
                s.synchronize()
                host = [x.cpu().numpy() for x in (q, k, v)]
                m.advance([1] * m.rows, m.rows, None, *host[1:])
                m.tables._step = (m.rows, m.rows)
                m.held_keys()
                close_to_held(m, [1] * m.rows, m.rows, host[0], out)
        for m in (*models, big):
            m.close()


def test_refusals():
    with Context(0) as ctx:
        m = Model(ctx, 2)
        q, k, v = (dev(x) for x in m.inputs(3))
        ctx.bind_kv_cache(m.arena)
        ctx.extend(m.tables, i32([1, 1]), 3, 1)
        m.layer.forward(q, k, v, ctx)
        with pytest.raises(IllegalArgumentException):
            m.layer.forward(q[:2], k[:2], v[:2], ctx)  # rows of another number
        short = RotaryEmbedding.scaled(ctx, D, 64, 399, 1e4)
        with pytest.raises(IllegalArgumentException):
            m.layer.forward_with_rope(short, None, q, k, v, ctx)  # tables of 400 tokens
        short.close()
        for blocks, block in ((199, BLOCK), (200, 2 * BLOCK)):
            with KvCacheArena4(ctx, 1, blocks, block, HKV, D) as other:
                ctx.bind_kv_cache(other)
                with pytest.raises(IllegalArgumentException):
                    m.layer.forward(q, k, v, ctx)
        ctx.bind_kv_cache(m.arena)
        # The capture of a step larger than any before it.
        s = torch.cuda.Stream()
        with torch.cuda.stream(s), Context(0, stream=s) as c:
            n = Model(c, 2)
            failed = None
            g = torch.cuda.CUDAGraph()
            q, k, v = (dev(x) for x in n.inputs(3))
            one = i32([1, 1])
            s.synchronize()
            c.bind_kv_cache(n.arena)
            with torch.cuda.graph(g, stream=s):
                c.extend(n.tables, one, 3, 1)
                try:
                    n.layer.forward(q, k, v, c)
                except IllegalArgumentException as e:
                    failed = e
            assert failed is not None
            n.close()
        m.close()
