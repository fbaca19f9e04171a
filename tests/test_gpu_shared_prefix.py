"""Attention of steps that share prefixes (nva_step_share_prefixes) against 64 bits: decode, prefill
and mixed steps over the served head shapes, group sizes on both sides of the span kernel's and the
span tiles' columns, page sizes with and without a span kernel, and the calls around them."""

import ctypes

import numpy as np
import pytest
import torch

from gpu_checks import arena_views, bits, say, torch_view
from span_checks import SharedStep, attend, close, step_reference
from nanollvm_amd import (Attention, Context, IllegalArgumentException, KvCacheArena,
                          NullPointerException, RMSNorm, RotaryEmbedding, _native as N)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


class Setup:
    """The arena (NaN wherever no token was stored), inputs and layer of a step."""

    def __init__(self, ctx, st, shape, seed, window=0, groups=None, share=True):
        self.st, (self.hq, self.hkv, self.d) = st, shape
        self.scale = float(np.float32(self.d ** -0.5))
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def randn(*size):
            return torch.randn(*size, device="cuda", generator=g)

        self.arena = KvCacheArena(ctx, 1, st.num_blocks, st.block, self.hkv, self.d)
        n = st.num_blocks * st.block
        self.kp, self.vp = (x.view(n, self.hkv, self.d) for x in arena_views(self.arena))
        used = torch.from_numpy(np.unique(np.concatenate(st.slots))).cuda()
        for x in (self.kp, self.vp):
            x.fill_(float("nan"))
            x[used] = randn(len(used), self.hkv, self.d)
        self.q = randn(st.tokens, self.hq, self.d)
        self.k, self.v = (randn(st.tokens, self.hkv, self.d) for _ in range(2))
        self.new = torch.from_numpy(np.concatenate(
            [s[len(s) - m:] for s, m in zip(st.slots, st.new)])).cuda()
        self.attn = Attention(self.hq, self.d, self.scale, self.hkv, window, 0)
        ctx.set(**st.context_args())
        if share:
            ctx.share_prefixes(st.groups if groups is None else groups)
        ctx.bind_kv_cache(self.arena)

    def reference(self, window=0):
        k, v = self.kp.clone(), self.vp.clone()
        k[self.new], v[self.new] = self.k, self.v
        return step_reference(self.st, self.q, k, v, self.scale, window), k, v

    def check(self, ctx, name, window=0):
        st = self.st
        say(f"{name}: {len(st.keys)} sequences, {st.tokens} tokens, {self.hq}/{self.hkv}/{self.d}, "
            f"pages of {st.block}, longest {max(st.keys)}")
        want, k, v = self.reference(window)
        out = self.attn.forward(self.q, self.k, self.v, ctx)
        ctx.sync()
        close(out, want, name)
        for x, y in ((self.kp, k), (self.vp, v)):
            assert torch.equal(x.view(torch.int32), y.view(torch.int32)), f"{name}: pages differ"
        return out


def launches(ctx, *names):
    return [ctx.kernel_stats(n)[0] for n in names]


SHAPES = [(16, 8, 128), (32, 8, 128), (32, 8, 64), (4, 1, 256), (8, 1, 512), (40, 8, 128),
          (6, 6, 64), (14, 2, 128), (34, 2, 64), (71, 1, 64), (8, 8, 256), (4, 2, 32), (6, 3, 16)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("rows", [2, 9, 40])
def test_decode(ctx, shape, rows):
    """One group, rows of their own before and behind it, and a second group of another length."""
    r = np.random.default_rng(rows)
    st = SharedStep([(1, 0), (rows, 320), (2, 0), (3, 64), (1, 128)],
                    [(int(c), 1) for c in r.integers(0, 150, rows + 7)], 64, seed=rows)
    s = Setup(ctx, st, shape, seed=1)
    try:
        s.check(ctx, f"decode {shape} {rows} rows")
    finally:
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("block", [1, 8, 16, 24, 256])
@pytest.mark.parametrize("shape,rows", [((16, 8, 128), 5), ((16, 8, 128), 130), ((4, 1, 256), 20),
                                        ((32, 8, 64), 3)], ids=str)
def test_page_sizes(ctx, block, shape, rows):
    r = np.random.default_rng(block)
    pages = max(1, 600 // block)
    st = SharedStep([(rows, pages * block)], [(int(c), 1) for c in r.integers(0, 70, rows)], block,
                    seed=block)
    s = Setup(ctx, st, shape, seed=2)
    try:
        s.check(ctx, f"pages of {block}, {shape}")
    finally:
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 31, 33, 63, 64, 65, 511])
@pytest.mark.parametrize("rows", [3, 70])
def test_prefixes_that_end_inside_a_page(ctx, tokens, rows):
    """The group names fewer tokens than the pages share: each sequence reads the rest itself."""
    st = SharedStep([(rows, 512)], [(i % 5, 1) for i in range(rows)], 256, seed=tokens)
    s = Setup(ctx, st, (16, 8, 128), seed=3, groups=[(0, rows, tokens)])
    try:
        s.check(ctx, f"{tokens} of 512 tokens, {rows} rows")
    finally:
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("chunks", [(1, 2), (1, 33, 1, 140), (300, 1, 7, 64, 65, 129, 2)], ids=str)
def test_prefill_and_mixed(ctx, shape, chunks):
    own = [(0, n) for n in chunks] + [(5, 3), (40, 1), (0, 20)]
    st = SharedStep([(len(chunks), 384), (2, 128), (1, 0)], own, 64, seed=4, decode=False)
    s = Setup(ctx, st, shape, seed=4)
    try:
        s.check(ctx, f"prefill {shape} {chunks}")
    finally:
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("shape", [(16, 8, 128), (32, 8, 64), (4, 1, 256), (8, 1, 512), (40, 8, 128),
                                   (12, 12, 64), (34, 2, 64), (71, 1, 64)], ids=str)
@pytest.mark.parametrize("chunks", [(2, 1, 3), (9,) * 30 + (1, 40, 70)], ids=["few", "many"])
def test_prefill_over_long_prefixes(ctx, shape, chunks):
    """Prefixes long enough that a prefill step reads them as spans, of few and of many columns,
    beside query tiles and rows of its own and a sequence that shares nothing."""
    own = [(i % 3, n) for i, n in enumerate(chunks)] + [(70, 50)]
    st = SharedStep([(len(chunks), 8192), (1, 0)], own, 256, seed=20, decode=False)
    s = Setup(ctx, st, shape, seed=20)
    ctx.set_timing(True)
    try:
        ctx.reset_stats()
        s.check(ctx, f"prefill over 8192 tokens {shape} {len(chunks)} chunks")
        ran = dict(zip(("span", "span_tiles"), launches(ctx, "span", "span_tiles")))
        assert sum(ran.values()) >= 1, ran
    finally:
        ctx.set_timing(False)
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("shape", [(16, 8, 128), (32, 8, 64), (4, 1, 256), (8, 1, 512), (40, 8, 128),
                                   (34, 2, 64)], ids=str)
@pytest.mark.parametrize("prefix,chunks,shared", [(2048, (5, 3, 1, 2, 4, 5), True),
                                                  (64, (2, 1), False)], ids=["shared", "apart"])
def test_prefill_of_few_tokens_runs_row_by_row(ctx, shape, prefix, chunks, shared):
    """A step of a few tokens behind a prefix takes no query tiles: its rows, masked one by one, run as
    rows, beside the prefix's span where that pays."""
    st = SharedStep([(len(chunks), prefix)], [(3 * i, n) for i, n in enumerate(chunks)], 64, seed=22,
                    decode=False)
    s = Setup(ctx, st, shape, seed=22)
    ctx.set_timing(True)
    try:
        ctx.reset_stats()
        s.check(ctx, f"few tokens {shape} {prefix} {chunks}")
        tiles, rows, span = launches(ctx, "prefill", "decode", "span")
        assert tiles == 0 and rows + span >= 1, (tiles, rows, span)
        if not shared:
            assert (rows, span) == (1, 0)
        elif shape == (16, 8, 128):
            assert (rows, span) == (0, 1)
    finally:
        ctx.set_timing(False)
        ctx.clear()
        s.arena.close()


def test_prefill_chunks_that_fill_their_tiles_are_read_apart(ctx):
    st = SharedStep([(2, 1536)], [(0, 256), (0, 256)], 256, seed=21, decode=False)
    s = Setup(ctx, st, (16, 8, 128), seed=21)
    ctx.set_timing(True)
    try:
        ctx.reset_stats()
        s.check(ctx, "full chunks")
        assert launches(ctx, "span", "span_tiles") == [0, 0]
    finally:
        ctx.set_timing(False)
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("shape", [(16, 8, 128), (32, 8, 64), (4, 1, 256), (8, 1, 512)], ids=str)
def test_groups_on_both_kernels(ctx, shape):
    """Groups of few and of many columns in one decode step, beside long rows of their own: the span
    kernel, span tiles, and the rows on the second stream."""
    st = SharedStep([(3, 4096), (200, 2048), (2, 1024), (9, 0)],
                    [(i * 7 % 900, 1) for i in range(214)], 256, seed=22)
    s = Setup(ctx, st, shape, seed=22)
    try:
        s.check(ctx, f"few and many columns {shape}")
    finally:
        ctx.clear()
        s.arena.close()


def test_long_prefix_many_rows(ctx):
    st = SharedStep([(130, 20480), (60, 5120)], [(i % 300, 1) for i in range(190)], 256, seed=5)
    s = Setup(ctx, st, (16, 8, 128), seed=5)
    try:
        s.check(ctx, "190 rows, 20K prefix")
    finally:
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("rows", [3, 200])
def test_pages_behind_four_gib(ctx, rows):
    """Pages whose rows lie beyond 32-bit byte and float offsets, on the span kernel and the tiles."""
    st = SharedStep([(rows, 4096)], [(i % 50, 1) for i in range(rows)], 256, seed=24,
                    first_block=16500)
    s = Setup(ctx, st, (2, 2, 128), seed=24)
    assert s.arena.shape(0)[0] * 256 * 2 * 128 > 2 ** 30
    try:
        s.check(ctx, f"pages behind 4 GiB, {rows} rows")
    finally:
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("seed", range(48))
def test_drawn_steps(ctx, seed):
    """Steps of any shape: groups of one to many sequences, prefixes of one page to many, page sizes,
    own lengths, decode or prefill, groups that name part of what the pages share."""
    r = np.random.default_rng(1000 + seed)
    shape = SHAPES[int(r.integers(len(SHAPES)))]
    block = int(r.choice([4, 16, 24, 64, 256]))
    decode = bool(r.integers(2))
    groups, own = [], []
    for _ in range(int(r.integers(1, 5))):
        n = int(r.integers(1, 3 if r.integers(2) else 70))
        pages = int(np.exp(r.uniform(0, np.log(max(2, 6000 // block)))))
        groups.append((n, pages * block))
        own += [(int(r.integers(0, 90)), 1 if decode else int(r.integers(1, 60)) if n < 30 else
                 int(r.integers(1, 9))) for _ in range(n)]
    st = SharedStep(groups, own, block, seed=seed, decode=decode)
    named = [(a, n, int(r.integers(0, p + 1)) if r.integers(2) else p) for a, n, p in st.groups]
    s = Setup(ctx, st, shape, seed=seed, groups=named)
    try:
        s.check(ctx, f"drawn step {seed}: {shape} pages of {block} {groups} decode={decode}")
    finally:
        ctx.clear()
        s.arena.close()


def test_found_groups_use_both_kernels(ctx):
    """find_shared_prefixes gives the groups; a few rows and a short prefix run on the span kernel,
    many over a long one on span tiles, and without sharing neither runs."""
    ctx.set_timing(True)
    try:
        for rows, tokens, name in ((3, 512, "span"), (150, 512, "span"), (150, 8192, "span_tiles")):
            st = SharedStep([(rows, tokens)], [(3, 1)] * rows, 256, seed=6)
            assert st.found() == [(0, rows, tokens)]
            s = Setup(ctx, st, (16, 8, 128), seed=6, groups=st.found())
            try:
                ctx.reset_stats()
                shared = s.check(ctx, f"found, {rows} rows")
                counts = dict(zip(("span", "span_tiles"), launches(ctx, "span", "span_tiles")))
                assert counts[name] == 1 and sum(counts.values()) == 1, counts
                ctx.reset_stats()
                ctx.share_prefixes([])
                alone = s.check(ctx, f"not shared, {rows} rows")
                assert launches(ctx, "span", "span_tiles", "decode") == [0, 0, 1]
                close(shared, alone.double(), "shared against separate reads")
            finally:
                ctx.clear()
                s.arena.close()
    finally:
        ctx.set_timing(False)


@pytest.mark.parametrize("rows", [4, 90])
def test_sliding_window_layers_are_as_before(ctx, rows):
    st = SharedStep([(rows, 512)], [(i % 40, 1) for i in range(rows)], 64, seed=7)
    s = Setup(ctx, st, (16, 8, 128), seed=7, window=100)
    try:
        got = s.check(ctx, "window", window=100)
        ctx.share_prefixes([])
        want = s.attn.forward(s.q, s.k, s.v, ctx)
        assert torch.equal(got, want)
    finally:
        ctx.clear()
        s.arena.close()


def test_rows_behind_the_sequences_are_zero(ctx):
    """A prefill step whose q has rows behind the last sequence."""
    st = SharedStep([(4, 256)], [(0, 9), (0, 1), (3, 30), (0, 2)], 64, seed=8, decode=False)
    s = Setup(ctx, st, (16, 8, 128), seed=8)
    try:
        q = torch.cat([s.q, torch.randn(5, s.hq, s.d, device="cuda")])
        attn = Attention(s.hq, s.d, s.scale, s.hkv, write_kv=False)
        want, k, v = s.reference()
        s.kp.copy_(k)
        s.vp.copy_(v)
        out = attn.forward(q, None, None, ctx)
        ctx.sync()
        close(out[:st.tokens], want, "rows of the sequences")
        assert torch.equal(out[st.tokens:], torch.zeros_like(out[st.tokens:]))
    finally:
        ctx.clear()
        s.arena.close()


def test_fewer_rows_than_sequences(ctx):
    """A decode call of fewer rows than the step has sequences computes those."""
    st = SharedStep([(40, 512)], [(i, 1) for i in range(40)], 64, seed=9)
    s = Setup(ctx, st, (16, 8, 128), seed=9)
    try:
        attn = Attention(s.hq, s.d, s.scale, s.hkv, write_kv=False)
        want, k, v = s.reference()
        s.kp.copy_(k)
        s.vp.copy_(v)
        for n in (1, 2, 17, 39, 40):
            out = attn.forward(s.q[:n], None, None, ctx)
            ctx.sync()
            close(out, want[:n], f"{n} of 40 rows")
    finally:
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("rows", [3, 60])
@pytest.mark.parametrize("shape", [(16, 8, 128), (32, 8, 64), (4, 1, 256), (8, 1, 512)], ids=str)
def test_infinities_and_unlike_sizes(ctx, rows, shape):
    """A prefix key of -inf scores (weight 0), one V channel far above the others, a key of large
    magnitude, and a V of infinity that every row sees: its dim is infinite, the others are not."""
    st = SharedStep([(rows, 192)], [(i % 9, 1) for i in range(rows)], 64, seed=10)
    s = Setup(ctx, st, shape, seed=10)
    try:
        at = torch.from_numpy(st.slots[0]).cuda()
        s.q[..., 0] = s.q[..., 0].abs() + 0.5
        s.kp[at[70], :, 0] = -float("inf")
        s.kp[at[71]] *= 1e3
        s.vp[:, :, 3] *= 1e6
        s.vp[at[100], :, 1] = float("inf")
        want, _, _ = s.reference()
        out = s.attn.forward(s.q, s.k, s.v, ctx)
        ctx.sync()
        assert torch.equal(torch.isfinite(out), torch.isfinite(want))
        for dims in (slice(4, None), slice(3, 4), slice(2, 3)):
            x, y = out[..., dims].double(), want[..., dims]
            rel = float((x - y).norm() / y.norm())
            say(f"unlike sizes {shape} {rows} rows, dims {dims}: rel_l2={rel:.3e}")
            assert rel <= 1e-5
    finally:
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("shape", [(16, 8, 128), (32, 8, 64), (4, 1, 256), (8, 1, 512)], ids=str)
def test_infinities_and_unlike_sizes_on_span_tiles(ctx, shape):
    """The same over a prefix and rows that run on span tiles, whose segments with such keys are
    taken again on fp32 instructions."""
    st = SharedStep([(210, 4096)], [(i % 9, 1) for i in range(210)], 64, seed=23)
    s = Setup(ctx, st, shape, seed=23)
    ctx.set_timing(True)
    try:
        at = torch.from_numpy(st.slots[0]).cuda()
        s.q[..., 0] = s.q[..., 0].abs() + 0.5
        s.kp[at[70], :, 0] = -float("inf")
        s.kp[at[2071]] *= 30
        s.vp[:, :, 3] *= 1e6
        s.vp[at[3100], :, 1] = float("inf")
        want, _, _ = s.reference()
        ctx.reset_stats()
        out = s.attn.forward(s.q, s.k, s.v, ctx)
        ctx.sync()
        assert launches(ctx, "span_tiles") == [1]
        assert torch.equal(torch.isfinite(out), torch.isfinite(want))
        for dims in (slice(4, None), slice(3, 4), slice(2, 3)):
            x, y = out[..., dims].double(), want[..., dims]
            rel = float((x - y).norm() / y.norm())
            say(f"unlike sizes on span tiles {shape}, dims {dims}: rel_l2={rel:.3e}")
            assert rel <= 1e-5
    finally:
        ctx.set_timing(False)
        ctx.clear()
        s.arena.close()


@pytest.mark.parametrize("rows", [3, 60])
def test_a_prefix_of_no_weight(ctx, rows):
    """Every prefix score is -inf: the rows' own keys decide alone."""
    st = SharedStep([(rows, 128)], [(4, 1)] * rows, 64, seed=11)
    s = Setup(ctx, st, (16, 8, 128), seed=11)
    try:
        s.q[..., 0] = s.q[..., 0].abs() + 0.5
        s.kp[torch.from_numpy(st.slots[0][:128]).cuda(), :, 0] = -float("inf")
        s.check(ctx, f"prefix of no weight, {rows} rows")
    finally:
        ctx.clear()
        s.arena.close()


def test_fused_chain_over_packed_qkv(ctx):
    """The packed qkv call of a model layer (head norms, RoPE, store) with and without sharing."""
    shape = (16, 8, 128)
    for decode in (True, False):
        own = [(i % 7, 1 if decode else 1 + i % 30) for i in range(50)]
        st = SharedStep([(50, 512)], own, 256, seed=12, decode=decode)
        s = Setup(ctx, st, shape, seed=12)
        rope = RotaryEmbedding(ctx, s.d, s.d, 4096, 1e6)
        try:
            w = torch.rand(s.d, device="cuda") + 0.5
            qn, kn = RMSNorm(w, 1e-6), RMSNorm(w, 1e-6)
            qkv = torch.cat([s.q.view(st.tokens, -1), s.k.view(st.tokens, -1),
                             s.v.view(st.tokens, -1)], 1)
            pos = np.concatenate([np.arange(k - n, k) for k, n in zip(st.keys, st.new)])
            q_out, k_out = torch.empty_like(s.q), torch.empty_like(s.k)
            out = s.attn.forward_packed_qkv(rope, pos.astype(np.float32), qkv, ctx, q_norm=qn,
                                            k_norm=kn, q_out=q_out, k_out=k_out)
            ctx.sync()
            s.q, s.k = q_out, k_out
            want, k, v = s.reference()
            close(out, want, f"packed qkv, decode={decode}")
            assert torch.equal(s.kp.view(torch.int32), k.view(torch.int32))
        finally:
            ctx.clear()
            rope.close()
            s.arena.close()


def noalloc(ctx, s, q, k, v, out):
    st = N.load().nva_attention_forward_noalloc(
        ctx.handle, s.arena.handle, ctypes.byref(s.attn._desc), q.data_ptr(), k.data_ptr(),
        v.data_ptr(), q.shape[0], out.data_ptr())
    assert st == N.NVA_OK, N.load().nva_last_error(ctx.handle).decode()


@pytest.mark.parametrize("rows,decode", [(4, True), (100, True), (30, False)])
def test_no_alloc_graph_replays(rows, decode):
    """The no-allocation call gives the same bits, and a captured graph of it, replayed with other
    work between, the eager call's bits on the inputs then in place."""
    s1 = torch.cuda.Stream()
    with torch.cuda.stream(s1), Context(0, stream=s1) as ctx:
        own = [(i % 60, 1 if decode else 1 + i % 20) for i in range(rows)]
        st = SharedStep([(rows, 768)], own, 64, seed=13, decode=decode)
        s = Setup(ctx, st, (16, 8, 128), seed=13)
        try:
            want = s.check(ctx, f"graph {rows} rows")
            out = torch.full_like(want, float("nan"))
            noalloc(ctx, s, s.q, s.k, s.v, out)
            s1.synchronize()
            assert torch.equal(out, want)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s1):
                noalloc(ctx, s, s.q, s.k, s.v, out)
            s1.synchronize()
            for r in range(4):
                if r >= 2:
                    for t in (s.q, s.k, s.v):
                        t.normal_()
                    want = s.attn.forward(s.q, s.k, s.v, ctx)
                out.fill_(float("nan"))
                junk = torch.randn(1 << 20, device="cuda").sum()
                s1.synchronize()
                g.replay()
                s1.synchronize()
                say(f"graph {rows} rows: replay {r} ({float(junk):.1f})")
                assert torch.equal(out, want), f"replay {r}"
        finally:
            ctx.clear()
            s.arena.close()


def test_two_contexts_in_turn():
    """Two contexts on two streams, calls in turn: each keeps its own plan and partials."""
    runs = []
    try:
        for i, rows in enumerate((70, 5)):
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                ctx = Context(0, stream=stream)
                st = SharedStep([(rows, 1024)], [(2 * i + 1, 1)] * rows, 64, seed=14 + i)
                s = Setup(ctx, st, (16, 8, 128), seed=14 + i)
                runs.append((stream, ctx, s, s.reference()[0]))
            stream.synchronize()
        outs = []
        for _ in range(3):
            for stream, ctx, s, want in runs:
                with torch.cuda.stream(stream):
                    outs.append((s.attn.forward(s.q, s.k, s.v, ctx), want))
        torch.cuda.synchronize()
        for i, (out, want) in enumerate(outs):
            close(out, want, f"two contexts, call {i}")
    finally:
        for _, ctx, s, _ in runs:
            ctx.clear()
            s.arena.close()
            ctx.close()


def test_a_new_step_forgets_the_groups(ctx):
    st = SharedStep([(20, 512)], [(3, 1)] * 20, 64, seed=16)
    s = Setup(ctx, st, (16, 8, 128), seed=16)
    ctx.set_timing(True)
    try:
        ctx.set(**st.context_args())
        ctx.reset_stats()
        s.check(ctx, "after a new step")
        assert launches(ctx, "span", "span_tiles") == [0, 0]
    finally:
        ctx.set_timing(False)
        ctx.clear()
        s.arena.close()


def test_refusals(ctx):
    st = SharedStep([(4, 128), (3, 64)], [(9, 1)] * 7, 64, seed=17)
    s = Setup(ctx, st, (16, 8, 128), seed=17)
    try:
        for bad in ([(0, 4, 138)],               # more than is cached before the new token
                    [(0, 4, -1)], [(0, 0, 64)], [(-1, 2, 64)], [(5, 3, 64)],
                    [(0, 4, 64), (3, 2, 64)],    # overlapping
                    [(4, 3, 64), (0, 4, 64)],    # out of order
                    [(0, 2 ** 31 - 1, 64)]):
            with pytest.raises(IllegalArgumentException):
                ctx.share_prefixes(bad)
        ctx.share_prefixes([(0, 4, 137)])        # the tables part ways behind 128 tokens
        before = s.kp.clone()
        with pytest.raises(IllegalArgumentException, match="differ within"):
            s.attn.forward(s.q, s.k, s.v, ctx)
        ctx.sync()
        assert torch.equal(before.view(torch.int32), s.kp.view(torch.int32)), "nothing is stored"
        ctx.share_prefixes(st.groups)
        s.check(ctx, "after a refused group")
        args = st.context_args()
        args["block_tables"] = None
        ctx.set(**args)
        with pytest.raises(IllegalArgumentException):
            ctx.share_prefixes(st.groups)
        ctx.clear()
        with pytest.raises(NullPointerException):
            ctx.share_prefixes([])
    finally:
        ctx.clear()
        s.arena.close()
