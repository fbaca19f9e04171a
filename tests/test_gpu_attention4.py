"""Attention over the 4-bit arena against 64 bits: the keys and values are those that the 4-bit form
holds, so what is left are fp32 products and sums (the path's bar)."""

import numpy as np
import pytest
import torch

from checks4 import attention, close, dev, held_fast
from nanollvm_amd import (Attention, BlockTables, Context, IllegalArgumentException, KvCacheArena4,
                          NullPointerException, NvaError, RMSNorm, RotaryEmbedding,
                          UnsupportedShapeError)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


class Case:
    """Sequences of (cached, new) tokens over an arena in random order of blocks, whose other slots hold
    large values that no query may see."""

    def __init__(self, seqs, hq, hkv, d, block=32, window=0, seed=0, scale=None, fill=True):
        r = np.random.default_rng(seed)
        self.seqs, self.hq, self.hkv, self.d, self.block = seqs, hq, hkv, d, block
        self.window, self.scale = window, float(np.float32(d ** -0.5 if scale is None else scale))
        need = [-(-(c + n) // block) for c, n in seqs]
        self.blocks = sum(need) + 2
        ids = iter(r.permutation(self.blocks)[:sum(need)].tolist())
        self.tables = [[next(ids) for _ in range(m)] for m in need]
        self.q, self.k_new, self.v_new = (
            r.standard_normal((sum(n for _, n in seqs), h, d)).astype(np.float32)
            for h in (hq, hkv, hkv))
        self.k, self.v = ([r.standard_normal((c, hkv, d)).astype(np.float32) for c, _ in seqs]
                          for _ in range(2))
        self.fill = fill

    def slots(self, b, lo, hi):
        t, at = np.asarray(self.tables[b], np.int64), np.arange(lo, hi)
        return (t[at // self.block] * self.block + at % self.block if hi > lo else at).astype(np.int32)

    def new_slots(self):
        return np.concatenate([self.slots(b, c, c + n) for b, (c, n) in enumerate(self.seqs)])

    def arena(self, ctx):
        a = KvCacheArena4(ctx, 1, self.blocks, self.block, self.hkv, self.d)
        if self.fill:
            every = np.arange(self.blocks * self.block, dtype=np.int32)
            x = np.full((len(every), self.hkv, self.d), 3e3, np.float32)
            a.write_rows(0, dev(every), dev(x), dev(x))
        for b, (c, _) in enumerate(self.seqs):
            if c:
                a.write_rows(0, dev(self.slots(b, 0, c)), dev(self.k[b]), dev(self.v[b]))
        return a

    def step(self, decode=None):
        lens = [c + n for c, n in self.seqs]
        table = np.full((len(self.seqs), max(1, max(map(len, self.tables)))), -1, np.int32)
        for row, t in zip(table, self.tables):
            row[:len(t)] = t
        what = dict(slot_mapping=self.new_slots(), block_tables=table)
        if decode if decode is not None else all(n == 1 for _, n in self.seqs):
            return dict(is_prefill=False, context_lens=lens, **what)
        return dict(is_prefill=True, cu_seqlens_q=np.cumsum([0] + [n for _, n in self.seqs]),
                    cu_seqlens_k=np.cumsum([0] + lens), max_seqlen_q=max(n for _, n in self.seqs),
                    max_seqlen_k=max(lens), **what)

    def want(self, q=None, k_new=None, v_new=None):
        q = self.q if q is None else q
        k_new = held_fast(self.k_new if k_new is None else k_new)
        v_new = held_fast(self.v_new if v_new is None else v_new)
        out, at = [], 0
        for b, (c, n) in enumerate(self.seqs):
            k = np.concatenate([held_fast(self.k[b]) if c else k_new[:0], k_new[at:at + n]])
            v = np.concatenate([held_fast(self.v[b]) if c else v_new[:0], v_new[at:at + n]])
            out.append(attention(q[at:at + n], k, v, c, self.scale, self.window))
            at += n
        return np.concatenate(out)

    def layer(self, **kw):
        return Attention(self.hq, self.d, self.scale, self.hkv, self.window, **kw)

    def run(self, ctx, decode=None):
        with self.arena(ctx) as a:
            ctx.set(**self.step(decode))
            ctx.bind_kv_cache(a)
            out = self.layer().forward(dev(self.q), dev(self.k_new), dev(self.v_new), ctx)
            ctx.sync()
            ctx.clear()
            return out


HEADS = [(1, 1), (2, 1), (3, 1), (5, 1), (6, 2), (16, 1), (17, 1), (40, 1), (32, 8)]


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_decode(ctx, d, hq, hkv):
    """Lengths around the key tile and the block, one token and many workgroups."""
    lens = [1, 2, 31, 32, 33, 63, 64, 65, 96, 97, 300, 1111]
    case = Case([(n - 1, 1) for n in lens], hq, hkv, d, block=64, seed=d + hq)
    close(case.run(ctx), case.want(), f"decode {hq}/{hkv}/{d}")


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 1), (6, 2), (20, 1), (32, 8)])
def test_prefill(ctx, d, hq, hkv):
    seqs = [(0, 1), (0, 37), (33, 5), (100, 1), (64, 64), (0, 0), (7, 0), (250, 130), (31, 2)]
    case = Case(seqs, hq, hkv, d, block=32, seed=d + hq)
    close(case.run(ctx), case.want(), f"prefill {hq}/{hkv}/{d}")


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 5000])
def test_windows(ctx, d, window):
    case = Case([(200, 1), (0, 1), (499, 1), (31, 1), (window, 1)], 4, 2, d, window=window, seed=window)
    close(case.run(ctx), case.want(), f"window {window}, decode")
    case = Case([(200, 70), (0, 130), (31, 1), (window % 300, 40)], 4, 2, d, window=window,
                seed=window)
    close(case.run(ctx), case.want(), f"window {window}, prefill")


@pytest.mark.parametrize("block", [32, 96, 160, 256])
def test_blocks_of_any_multiple_of_32(ctx, block):
    case = Case([(700, 1), (95, 1), (96, 1), (block - 1, 1), (block, 1), (3 * block, 1)], 8, 2, 128,
                block=block, seed=block)
    close(case.run(ctx), case.want(), f"blocks of {block}")


@pytest.mark.parametrize("seqs,shape", [([(70000, 1)], (4, 1, 64)), ([(30000, 1), (5, 1)], (2, 2, 128)),
                                        ([(9000, 20), (20000, 1)], (8, 1, 256)),
                                        ([(12000, 1)], (8, 1, 512))])
def test_few_long_sequences(ctx, seqs, shape):
    """The keys of one sequence over many workgroups."""
    case = Case(seqs, *shape, block=256, seed=1, fill=False)
    close(case.run(ctx), case.want(), f"{seqs}")


def test_many_short_sequences(ctx):
    r = np.random.default_rng(8)
    for n in (255, 256, 257, 1300):
        case = Case([(int(c), 1) for c in r.integers(0, 70, n)], 4, 2, 64, seed=n)
        close(case.run(ctx), case.want(), f"{n} rows")
    seqs = [(int(c), int(n)) for c, n in zip(r.integers(0, 50, 700), r.integers(0, 5, 700))]
    case = Case(seqs, 6, 1, 64, seed=9)
    close(case.run(ctx), case.want(), "700 short chunks")


def test_scores_far_apart_and_equal(ctx):
    """One key outweighs all others in any tile; all keys alike give the mean."""
    for at in (0, 31, 32, 200, 400):
        case = Case([(400, 1)], 2, 1, 128, seed=at, scale=1.0)
        case.q[:] = 8.0
        if at < 400:
            case.k[0][at] = 40.0
        else:
            case.k_new[0] = 40.0
        close(case.run(ctx), case.want(), f"one key at {at}")
    case = Case([(400, 1)], 2, 1, 128, seed=1)
    case.k[0][:], case.k_new[:] = 1.0, 1.0
    close(case.run(ctx), case.want(), "keys alike")


def test_rows_without_keys_and_padding(ctx):
    """Context length 0, rows that no sequence covers, and rows whose keys all lie ahead."""
    case = Case([(40, 1), (0, 1), (9, 1)], 4, 2, 64, seed=3)
    with case.arena(ctx) as a:
        ctx.set(is_prefill=False, context_lens=[41, 0, 10], block_tables=case.step()["block_tables"],
                slot_mapping=case.new_slots())
        ctx.bind_kv_cache(a)
        out = case.layer().forward(dev(case.q), dev(case.k_new), dev(case.v_new), ctx).cpu().numpy()
        want = case.want()
        close(out[[0, 2]], want[[0, 2]])
        assert not np.any(out[1])
        # Fewer rows than sequences: the first ones.
        out = case.layer(write_kv=False).forward(dev(case.q[:1]), None, None, ctx)
        close(out, want[:1])
        # Row offsets that start behind row 0 and end before the last.
        ctx.set(is_prefill=True, cu_seqlens_q=[2, 3, 3, 4], cu_seqlens_k=[0, 41, 41, 51],
                max_seqlen_q=1, max_seqlen_k=41, block_tables=case.step()["block_tables"])
        q = np.zeros((6, 4, 64), np.float32)
        q[2], q[3] = case.q[0], case.q[2]
        out = case.layer(write_kv=False).forward(dev(q), None, None, ctx).cpu().numpy()
        close(out[2:4], want[[0, 2]])
        assert not np.any(out[[0, 1, 4, 5]])
        # Five queries over two keys: the first three see none.
        ctx.set(is_prefill=True, cu_seqlens_q=[0, 5], cu_seqlens_k=[0, 2], max_seqlen_q=5,
                max_seqlen_k=2, block_tables=[case.tables[0]])
        q = np.repeat(case.q[:1], 5, 0)
        out = case.layer(write_kv=False).forward(dev(q), None, None, ctx).cpu().numpy()
        assert not np.any(out[:3])
        k, v = held_fast(case.k[0][:2]), held_fast(case.v[0][:2])
        close(out[3:], attention(q[3:], k, v, 0, case.scale))
        assert case.layer().forward(dev(q[:0]), dev(case.k_new[:0]), dev(case.v_new[:0]),
                                    ctx).shape == (0, 4, 64)
        ctx.clear()


@pytest.mark.parametrize("d", [64, 128, 256, 512])
def test_blocks_that_are_not_finite_reach_what_sees_them(ctx, d):
    """A NaN in V is in the results of the queries that see the key, in that block of 32 dims; in K, in
    the whole of them; infinite queries and queries that are NaN keep to themselves."""
    case = Case([(40, 60), (50, 1)], 2, 1, d, block=32, seed=d)
    case.v_new[20, 0, 5] = np.nan      # key 60 of sequence 0
    case.v[1][33, 0, d - 1] = np.inf   # and one behind a tile's border
    want = case.want(v_new=np.nan_to_num(case.v_new, nan=0.0))
    want[20:60, :, :32] = np.nan
    k = held_fast(np.concatenate([case.k[1], case.k_new[60:]]))
    case.v[1][33, 0, d - 1] = 0
    v = held_fast(np.concatenate([case.v[1], case.v_new[60:]]))
    want[60:] = attention(case.q[60:], k, v, 50, case.scale)
    want[60:, :, d - 32:] = np.nan
    case.v[1][33, 0, d - 1] = np.inf
    close(case.run(ctx), want, "V")
    # The same keys under a window that leaves them behind.
    case.window = 10
    got = case.run(ctx).cpu().numpy()
    seen = np.isnan(got[:60, :, :32]).all((1, 2))
    assert np.array_equal(np.flatnonzero(seen), np.arange(20, 30))
    assert not np.isnan(got[60]).any()
    assert not np.isnan(got[:60, :, 32:]).any()
    # K, and a query.
    case = Case([(40, 60), (50, 1)], 2, 1, d, block=32, seed=d)
    clean = case.want()
    case.k_new[30] = np.nan
    case.q[3, 1, 7] = np.inf
    case.q[4, 0, 0] = np.nan
    got = case.run(ctx).cpu().numpy()
    assert np.isnan(got[30:60]).all()
    assert np.isnan(got[4, 0]).all() and not np.isnan(got[4, 1]).any()
    keep = [i for i in range(61) if i not in (3, 4) and not 30 <= i < 60]
    close(got[keep], clean[keep], "K")


def test_infinite_scores(ctx):
    """An infinite query makes scores of either sign of infinity: those of minus infinity weigh nothing."""
    case = Case([(6, 1)], 1, 1, 64, seed=2)
    case.q[:], case.k[0][:], case.k_new[:] = 0, 0, 1
    case.q[0, 0, 0] = -np.inf
    case.k[0][:, 0, 0] = 1
    case.k_new[:, 0, 0] = 1
    got = case.run(ctx).cpu().numpy()
    assert not np.any(got)  # every score is minus infinity


def test_stale_blocks_stay_out(ctx):
    """What an earlier sequence left behind the last key, NaN included, changes no bit."""
    case = Case([(40, 1), (33, 3)], 4, 2, 128, seed=6)
    base = case.run(ctx).cpu().numpy()
    plain = case.arena

    def arena(c):
        a = plain(c)
        own = np.concatenate([case.slots(b, 0, sum(s)) for b, s in enumerate(case.seqs)])
        rest = np.setdiff1d(np.arange(case.blocks * case.block), own).astype(np.int32)
        x = np.full((len(rest), 2, 128), np.nan, np.float32)
        a.write_rows(0, dev(rest), dev(x), dev(x))
        return a
    case.arena = arena
    assert np.array_equal(case.run(ctx).cpu().numpy(), base)


def test_shared_kv_layers_read_only(ctx):
    case = Case([(64, 1), (3, 1)], 4, 2, 128, seed=7)
    with case.arena(ctx) as a:
        ctx.set(**case.step())
        ctx.bind_kv_cache(a)
        first = case.layer().forward(dev(case.q), dev(case.k_new), dev(case.v_new), ctx)
        again = case.layer(write_kv=False).forward(dev(case.q), dev(-case.k_new), dev(-case.v_new),
                                                   ctx)
        assert torch.equal(first, again)
        close(first, case.want())
        ctx.clear()


def test_layers_of_different_head_dims(ctx):
    a = Case([(50, 1)], 4, 2, 256, seed=1)
    b = Case([(50, 1)], 4, 2, 64, seed=1)
    b.tables, b.blocks = a.tables, a.blocks
    with KvCacheArena4(ctx, 3, a.blocks, 32, 2, head_dims=[256, 128, 64],
                       allocate=[True, False, True]) as arena:
        for layer, c in ((0, a), (2, b)):
            arena.write_rows(layer, dev(c.slots(0, 0, 50)), dev(c.k[0]), dev(c.v[0]))
        ctx.set(**a.step())
        ctx.bind_kv_cache(arena)
        for layer, c in ((0, a), (2, b)):
            out = c.layer(kv_layer_index=layer).forward(dev(c.q), dev(c.k_new), dev(c.v_new), ctx)
            close(out, c.want())
        for layer in (1, 3):
            with pytest.raises(IllegalArgumentException):
                a.layer(kv_layer_index=layer).forward(dev(a.q), dev(a.k_new), dev(a.v_new), ctx)
        ctx.clear()


def test_blocks_behind_4_gib(ctx):
    """Byte offsets past 32 bits, in the arena and in the slots' products."""
    hkv, d, block = 8, 512, 256
    blocks = (5 << 30) // (block // 32 * hkv * 34 * d) + 1
    case = Case([(300, 1), (20, 40)], 8, hkv, d, block=block, seed=5, fill=False)
    case.tables = [[blocks - 1, 0], [blocks - 2]]
    case.blocks = blocks
    close(case.run(ctx), case.want(), "far blocks")


def test_results_repeat_bit_for_bit(ctx):
    case = Case([(5000, 1), (64, 1), (900, 1)], 8, 2, 128, seed=4)
    first = case.run(ctx)
    for _ in range(3):
        assert torch.equal(case.run(ctx), first)


def test_head_norms_rope_and_packed_rows(ctx):
    """The fused calls over the 4-bit arena are norms, rotation and attention one after the other, bit
    for bit."""
    case = Case([(40, 3), (0, 33)], 4, 2, 128, seed=12)
    r = np.random.default_rng(1)
    weights = [dev(r.standard_normal(128).astype(np.float32)) for _ in range(2)]
    pos = np.concatenate([np.arange(c, c + n) for c, n in case.seqs]).astype(np.float32)
    for rope in (RotaryEmbedding(ctx, 128, 128, 100, 1e4),
                 RotaryEmbedding.scaled(ctx, 128, 32, 100, 1e4, interleaved=True)):
        for norms in (False, True):
            got = []
            for way in range(4):
                with case.arena(ctx) as a:
                    ctx.set(positions=pos, **case.step())
                    ctx.bind_kv_cache(a)
                    q, k, v = dev(case.q), dev(case.k_new), dev(case.v_new)
                    qn, kn = (RMSNorm(w, 1e-6) if norms else None for w in weights)
                    vn = RMSNorm.weightless(1e-6) if norms else None
                    layer = case.layer()
                    if way == 0:
                        if norms:
                            q, k, v = (n.forward(x, ctx) for n, x in ((qn, q), (kn, k), (vn, v)))
                        q, k = rope.forward(None, q, k, ctx)
                        out = layer.forward(q, k, v, ctx)
                        close(out, case.want(*(x.cpu().numpy() for x in (q, k, v))))
                    elif way == 1:
                        out = layer.forward_with_norm_rope(rope, None, q, k, v, ctx, qn, kn, vn)
                    elif way == 2:
                        packed = torch.cat([x.reshape(len(q), -1) for x in (q, k, v)], 1)
                        out = layer.forward_packed_qkv(rope, None, packed, ctx, qn, kn, vn)
                    elif norms:
                        continue
                    else:
                        out = layer.forward_with_rope(rope, None, q, k, v, ctx)
                    got.append((out, *a.read_rows(0, dev(case.new_slots()))))
                    ctx.sync()
                    ctx.clear()
            for other in got[1:]:
                for x, y in zip(got[0], other):
                    assert torch.equal(x, y)
        rope.close()


def test_refusals(ctx):
    case = Case([(64, 1), (3, 1)], 4, 2, 128, seed=7)
    q, k, v = dev(case.q), dev(case.k_new), dev(case.v_new)
    layer, step = case.layer(), case.step()
    ctx.clear()
    with pytest.raises(NullPointerException):
        layer.forward(q, k, v, ctx)  # no arena
    with case.arena(ctx) as a:
        ctx.bind_kv_cache(a)
        with pytest.raises(NullPointerException):
            layer.forward(q, k, v, ctx)  # no step
        bad_table = step["block_tables"].copy()
        bad_table[0, 1] = case.blocks
        no_table = step["block_tables"].copy()
        no_table[1, 0] = -1
        for change in (dict(block_tables=bad_table), dict(block_tables=no_table),
                       dict(block_tables=step["block_tables"][:, :1]),
                       dict(context_lens=[65, 32 * 3 + 1]), dict(block_tables=None),
                       dict(slot_mapping=[0, case.blocks * 32])):
            ctx.set(**{**step, **change})
            ctx.bind_kv_cache(a)
            with pytest.raises(IllegalArgumentException):
                layer.forward(q, k, v, ctx)
        ctx.set(**step)
        ctx.bind_kv_cache(a)
        for other in (Attention(4, 64, 0.1, 2), Attention(4, 128, 0.1, 1)):
            x = torch.zeros(2, 4, other.head_dim, device="cuda")
            y = torch.zeros(2, other.num_kv_heads, other.head_dim, device="cuda")
            with pytest.raises(IllegalArgumentException):
                other.forward(x, y, y, ctx)
        with pytest.raises(IllegalArgumentException):
            layer.forward(q, None, None, ctx)
        three = [torch.cat([x, x[:1]]) for x in (q, k, v)]
        with pytest.raises(IllegalArgumentException):
            layer.forward(*three, ctx)  # more rows than sequences
        ctx.set(is_prefill=True, cu_seqlens_q=[0, 3, 5], cu_seqlens_k=[0, 65, 70], max_seqlen_q=3,
                max_seqlen_k=65, block_tables=step["block_tables"])
        with pytest.raises(IllegalArgumentException):
            layer.forward(q, k, v, ctx)  # offsets past the rows
        with Context(0) as other:
            other.set(**step)
            other.bind_kv_cache(a)
            with pytest.raises(IllegalArgumentException):
                layer.forward(q, k, v, other)
        ctx.clear()


def test_a_host_step_is_not_captured(ctx):
    case = Case([(64, 1), (3, 1)], 4, 2, 128, seed=7)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), Context(0, stream=s) as c, case.arena(c) as a:
        c.set(**case.step())
        c.bind_kv_cache(a)
        q, k, v = dev(case.q), dev(case.k_new), dev(case.v_new)
        layer = case.layer()
        layer.forward(q, k, v, c)
        failed = None
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            q.add_(0)
            try:
                layer.forward(q, k, v, c)
            except IllegalArgumentException as e:
                failed = e
        assert failed is not None
        c.clear()
