"""Cross attention (nva_cross_attention_forward) against 64 bits: single tokens, beams, prompts and
full encoder layers, odd lengths and empty states, packed projections, and the calls around them."""

import ctypes

import numpy as np
import pytest
import torch

from gpu_checks import say
from span_checks import attend, close
from nanollvm_amd import (Context, CrossAttention, IllegalArgumentException, NullPointerException,
                          UnsupportedShapeError, _native as N)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


class Pool:
    """Encoder rows at random places of a pool, NaN between them; keys and values packed or apart."""

    def __init__(self, shape, lens, seed, packed, extra=0):
        self.hq, self.hkv, self.d = shape
        r = np.random.default_rng(seed)
        self.start, at = np.zeros(len(lens), np.int32), 3
        for i in r.permutation(len(lens)):
            self.start[i] = at
            at += lens[i] + int(r.integers(0, 4))
        self.rows = at + extra
        kv = torch.full((self.rows, 2, self.hkv, self.d) if packed else
                        (2, self.rows, self.hkv, self.d), float("nan"), device="cuda")
        self.k, self.v = kv.unbind(1 if packed else 0)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        for s, n in zip(self.start, lens):
            for x in (self.k, self.v):
                x[s:s + n] = torch.randn(n, self.hkv, self.d, device="cuda", generator=g)


def set_step(ctx, queries, lens, start):
    """A decode step if every sequence has one query, else a prefill."""
    if all(n == 1 for n in queries):
        ctx.set(is_prefill=False, context_lens=[7] * len(queries))
    else:
        cu = np.concatenate([[0], np.cumsum(queries)])
        ctx.set(is_prefill=True, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=max(queries),
                max_seqlen_k=max(queries))
    ctx.set_encoder(start, lens)


def reference(q, pool, queries, lens, start, scale):
    out, at = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), 0
    for n, m, s in zip(queries, lens, start):
        out[at:at + n] = attend(q[at:at + n], pool.k[s:s + m], pool.v[s:s + m], scale)
        at += n
    return out


def check(ctx, name, shape, queries, requests, beams=1, packed=True, seed=0, tail=0):
    """requests: encoder lengths; each is read by `beams` sequences in a row."""
    hq, hkv, d = shape
    pool = Pool(shape, requests, seed, packed)
    start, lens = np.repeat(pool.start, beams), np.repeat(np.asarray(requests, np.int32), beams)
    tokens = sum(queries)
    say(f"{name}: {shape} {len(queries)} sequences, {tokens} queries, {pool.rows} rows, "
        f"packed={packed}")
    q = torch.randn(tokens + tail, hq, d, device="cuda",
                    generator=torch.Generator(device="cuda").manual_seed(seed + 1))
    scale = float(np.float32(d ** -0.5))
    set_step(ctx, queries, lens, start)
    layer = CrossAttention(hq, d, scale, hkv)
    out = layer.forward(q, pool.k, pool.v, ctx)
    ctx.sync()
    close(out, reference(q, pool, queries, lens, start, scale), name)
    assert torch.equal(out[tokens:], torch.zeros_like(out[tokens:]))
    ctx.clear()


SHAPES = [(16, 16, 64), (12, 12, 64), (16, 8, 128), (32, 8, 64), (4, 1, 256), (8, 1, 512),
          (5, 1, 128), (34, 2, 64), (71, 1, 64), (12, 12, 32), (6, 3, 16), (2, 1, 4)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("packed", [True, False])
def test_single_tokens(ctx, shape, packed):
    check(ctx, "single tokens", shape, [1] * 11, [0, 1, 2, 15, 16, 17, 63, 64, 65, 300, 1111],
          packed=packed, seed=1)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("beams", [2, 5, 9])
def test_beams(ctx, shape, beams):
    lens = [33, 0, 500, 1, 129]
    check(ctx, f"{beams} beams", shape, [1] * (beams * len(lens)), lens, beams=beams,
          packed=beams == 5, seed=2)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("queries,lens", [
    ([3, 0, 1, 40], [70, 9, 0, 31]),
    ([257, 1, 130, 2, 65], [513, 1024, 1, 32, 33]),
    ([1, 500], [2000, 100]),
], ids=str)
def test_prompts(ctx, shape, queries, lens):
    check(ctx, "prompts", shape, queries, lens, seed=3, tail=3)


@pytest.mark.parametrize("shape", [(12, 12, 64), (12, 12, 32), (16, 8, 128)], ids=str)
def test_full_attention_of_an_encoder(ctx, shape):
    lens = [1, 7, 64, 0, 129, 512, 33]
    check(ctx, "full attention", shape, lens, lens, seed=4)


@pytest.mark.parametrize("seed", range(48))
def test_drawn_steps(ctx, seed):
    """Any head shape, numbers of requests, beams, queries and keys."""
    r = np.random.default_rng(2000 + seed)
    shape = SHAPES[int(r.integers(len(SHAPES)))]
    lens = [int(np.exp(r.uniform(0, np.log(3000)))) - 1 for _ in range(int(r.integers(1, 25)))]
    beams = int(r.choice([1, 1, 2, 3, 6]))
    most = int(r.choice([1, 4, 90]))
    queries = [int(r.integers(0 if most > 1 else 1, most + 1)) for _ in range(len(lens) * beams)]
    check(ctx, f"drawn step {seed}", shape, queries, lens, beams=beams, packed=bool(r.integers(2)),
          seed=seed, tail=int(r.integers(0, 3)) if any(n != 1 for n in queries) else 0)


@pytest.mark.parametrize("shape", [(4, 1, 256), (16, 8, 128), (12, 12, 64), (8, 1, 512)], ids=str)
@pytest.mark.parametrize("queries,lens", [
    ([333, 410, 250, 301, 377], [1777, 900, 1300, 33, 650]),                   # few tiles, one piece each
    ([90 + 7 * (i % 5) for i in range(40)], [13 + 37 * i % 97 for i in range(40)]),  # many short ones
    ([700, 20, 520], [5000, 129, 64]),                                        # one far longer
], ids=["even", "short", "uneven"])
def test_cuts_of_span_tiles(ctx, shape, queries, lens):
    check(ctx, "cuts", shape, queries, lens, packed=False, seed=23)


def test_many_sequences_of_one_key(ctx):
    check(ctx, "one key each", (16, 16, 64), [1] * 700, [1] * 700, seed=5)


def test_one_sequence_of_many_keys(ctx):
    check(ctx, "one long state", (16, 16, 64), [1], [150001], seed=6)
    check(ctx, "one long state, prompts", (16, 8, 128), [200], [40000], seed=6)


@pytest.mark.parametrize("queries", [1, 40])
def test_rows_behind_four_gib(ctx, queries):
    """Row offsets beyond 32 bits, in bytes and in floats."""
    hq, hkv, d = 8, 8, 64
    rows, width = 9_000_000, 2 * hkv * d          # 9.2e9 floats
    kv = torch.empty(rows * width, device="cuda").view(rows, 2, hkv, d)
    k, v = kv.unbind(1)
    lens, start = [300, 77, 1000], [rows - 300, 4_300_000, 1_048_500]
    for s, n in zip(start, lens):
        kv[s:s + n].normal_()
    q = torch.randn(queries * 3, hq, d, device="cuda")
    set_step(ctx, [queries] * 3, lens, start)
    say(f"rows behind 4 GiB: {queries} queries")
    out = CrossAttention(hq, d, 0.125, hkv).forward(q, k, v, ctx)
    ctx.sync()
    want = torch.cat([attend(q[i * queries:(i + 1) * queries], k[s:s + n], v[s:s + n], 0.125)
                      for i, (s, n) in enumerate(zip(start, lens))])
    close(out, want, "rows behind 4 GiB")
    ctx.clear()


@pytest.mark.parametrize("queries", [1, 30, 300])
@pytest.mark.parametrize("shape", [(16, 8, 128), (12, 12, 64), (4, 1, 256), (8, 1, 512)], ids=str)
def test_infinities(ctx, queries, shape):
    """Keys of -inf scores take no weight; where all are, the row is zero."""
    hq, hkv, d = shape
    pool = Pool(shape, [100, 40], 7, True)
    q = torch.randn(2 * queries, hq, d, device="cuda")
    q[..., 0] = q[..., 0].abs() + 0.5
    s0, s1 = (int(x) for x in pool.start)
    pool.k[s0 + 30, :, 0] = -float("inf")
    pool.k[s1:s1 + 40, :, 0] = -float("inf")
    pool.v[s0 + 30] = float("nan")                # beside weight 0 it would be NaN in any product
    pool.v[s0 + 30] = 1e30
    set_step(ctx, [queries] * 2, [100, 40], pool.start)
    scale = float(np.float32(d ** -0.5))
    out = CrossAttention(hq, d, scale, hkv).forward(q, pool.k, pool.v, ctx)
    ctx.sync()
    want = reference(q, pool, [queries] * 2, [100, 40], pool.start, scale)
    close(out, want, f"infinities {shape}")
    assert torch.equal(out[queries:], torch.zeros_like(out[queries:]))
    ctx.clear()


@pytest.mark.parametrize("shape", [(16, 8, 128), (12, 12, 64), (4, 1, 256), (8, 1, 512)], ids=str)
def test_infinities_on_span_tiles(ctx, shape):
    """Prompts long enough for span tiles: -inf scores, one sequence that has nothing else, and
    lengths around the tiles'."""
    hq, hkv, d = shape
    lens, queries = [3000, 2049, 31], [700, 300, 260]
    pool = Pool(shape, lens, 14, True)
    q = torch.randn(sum(queries), hq, d, device="cuda")
    q[..., 0] = q[..., 0].abs() + 0.5
    s0, s2 = int(pool.start[0]), int(pool.start[2])
    pool.k[s0 + 1030:s0 + 1070, :, 0] = -float("inf")
    pool.v[s0 + 1030] = 1e30
    pool.k[s2:s2 + 31, :, 0] = -float("inf")
    set_step(ctx, queries, lens, pool.start)
    scale = float(np.float32(d ** -0.5))
    ctx.set_timing(True)
    try:
        ctx.reset_stats()
        out = CrossAttention(hq, d, scale, hkv).forward(q, pool.k, pool.v, ctx)
        ctx.sync()
        assert ctx.kernel_stats("span_tiles")[0] == 1
    finally:
        ctx.set_timing(False)
    want = reference(q, pool, queries, lens, pool.start, scale)
    close(out, want, f"infinities on span tiles {shape}")
    assert torch.equal(out[1000:], torch.zeros_like(out[1000:]))
    ctx.clear()


@pytest.mark.parametrize("queries", [1, 30])
def test_large_scores_and_negative_scale(ctx, queries):
    """Scores of some hundreds, where one key has nearly all the weight; a negative scale."""
    shape = (16, 8, 128)
    for scale in (1.0, -0.5):
        pool = Pool(shape, [77, 500], 8, False)
        q = 3 * torch.randn(2 * queries, 16, 128, device="cuda")
        set_step(ctx, [queries] * 2, [77, 500], pool.start)
        out = CrossAttention(16, 128, scale, 8).forward(q, pool.k, pool.v, ctx)
        ctx.sync()
        want = reference(q, pool, [queries] * 2, [77, 500], pool.start, scale)
        # A score of 34 sigma * 3 * |scale|, off by half a step of its fp32 sum (2^-24 of it, times
        # sqrt(d) / 4 for the order of the sum) moves its weight by that: below 2^-15 in all.
        rel = float((out.double() - want).norm() / want.norm())
        say(f"large scores, scale {scale}: rel_l2={rel:.3e}")
        assert rel <= 2.0 ** -15
    ctx.clear()


@pytest.mark.parametrize("queries,lens,beams", [([1] * 6, [90, 1, 700], 2), ([50, 3], [300, 800], 1)])
def test_no_alloc_graph_replays(queries, lens, beams):
    """The no-allocation form: the same bits, also from a graph replayed over new inputs; the first
    form is refused under capture."""
    lib = N.load()
    s1 = torch.cuda.Stream()
    with torch.cuda.stream(s1), Context(0, stream=s1) as ctx:
        shape = (16, 8, 128)
        pool = Pool(shape, lens, 9, True)
        q = torch.randn(sum(queries), 16, 128, device="cuda")
        set_step(ctx, queries, np.repeat(lens, beams), np.repeat(pool.start, beams))
        layer = CrossAttention(16, 128, 0.1, 8)
        want = layer.forward(q, pool.k, pool.v, ctx)
        out = torch.full_like(want, float("nan"))

        def call(fn):
            return fn(ctx.handle, ctypes.byref(layer._desc), q.data_ptr(), pool.k.data_ptr(),
                      pool.v.data_ptr(), pool.rows, pool.k.stride(0), q.shape[0], out.data_ptr())

        assert call(lib.nva_cross_attention_forward_noalloc) == N.NVA_OK
        s1.synchronize()
        assert torch.equal(out, want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s1):
            refused = call(lib.nva_cross_attention_forward)
            st = call(lib.nva_cross_attention_forward_noalloc)
        assert refused == N.NVA_E_ARG and st == N.NVA_OK
        for r in range(4):
            if r >= 2:
                q.normal_()
                want = layer.forward(q, pool.k, pool.v, ctx)
            out.fill_(float("nan"))
            junk = torch.randn(1 << 20, device="cuda").sum()
            s1.synchronize()
            g.replay()
            s1.synchronize()
            say(f"cross graph: replay {r} ({float(junk):.1f})")
            assert torch.equal(out, want), f"replay {r}"
        ctx.clear()


def test_decoder_layer_in_one_graph():
    """Self attention over pages that share a prefix and cross attention on its output, captured as
    one graph: both plans stay in the device's scratch array, and replays give the eager bits."""
    from nanollvm_amd import Attention, KvCacheArena
    from span_checks import SharedStep
    lib = N.load()
    s1 = torch.cuda.Stream()
    with torch.cuda.stream(s1), Context(0, stream=s1) as ctx:
        st = SharedStep([(40, 1024)], [(i, 1) for i in range(40)], 64, seed=15)
        arena = KvCacheArena(ctx, 1, st.num_blocks, 64, 8, 128)
        try:
            lens = [50 + 20 * i for i in range(40)]
            pool = Pool((16, 8, 128), lens, 16, True)
            q = torch.randn(40, 16, 128, device="cuda")
            k, v = (torch.randn(40, 8, 128, device="cuda") for _ in range(2))
            ctx.set(**st.context_args())
            ctx.share_prefixes(st.groups)
            ctx.set_encoder(pool.start, lens)
            ctx.bind_kv_cache(arena)
            own, cross = Attention(16, 128, 0.09, 8), CrossAttention(16, 128, 0.09, 8)
            x, y = torch.empty_like(q), torch.empty_like(q)

            def layer():
                return [lib.nva_attention_forward_noalloc(
                            ctx.handle, arena.handle, ctypes.byref(own._desc), q.data_ptr(),
                            k.data_ptr(), v.data_ptr(), 40, x.data_ptr()),
                        lib.nva_cross_attention_forward_noalloc(
                            ctx.handle, ctypes.byref(cross._desc), x.data_ptr(), pool.k.data_ptr(),
                            pool.v.data_ptr(), pool.rows, pool.k.stride(0), 40, y.data_ptr())]

            assert layer() == [N.NVA_OK, N.NVA_OK]
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s1):
                got = layer()
            assert got == [N.NVA_OK, N.NVA_OK], lib.nva_last_error(ctx.handle)
            for r in range(4):
                for t in (q, k, v):
                    t.normal_()
                want_x = own.forward(q, k, v, ctx)
                want_y = cross.forward(want_x, pool.k, pool.v, ctx)
                x.fill_(float("nan"))
                y.fill_(float("nan"))
                s1.synchronize()
                g.replay()
                s1.synchronize()
                say(f"decoder layer graph: replay {r}")
                assert torch.equal(x, want_x) and torch.equal(y, want_y), f"replay {r}"
        finally:
            ctx.clear()
            arena.close()


def test_calls_that_do_not_fit_one_graph():
    """Under capture a call whose partials would overwrite the plan that the other attention holds in
    the scratch array is refused; outside capture both run and agree with the allocating forms."""
    from nanollvm_amd import Attention, KvCacheArena
    lib = N.load()
    tokens, keys, block = 1250, 6 * 4096, 64
    s1 = torch.cuda.Stream()
    with torch.cuda.stream(s1), Context(0, stream=s1) as ctx:
        arena = KvCacheArena(ctx, 1, (tokens + block - 1) // block, block, 64, 128)
        try:
            torch.manual_seed(18)
            q, k, v = (torch.randn(tokens, 64, 128, device="cuda") for _ in range(3))
            ctx.set(is_prefill=True, cu_seqlens_q=[0, tokens], cu_seqlens_k=[0, tokens],
                    slot_mapping=list(range(tokens)))
            ctx.set_encoder([0], [keys])
            ctx.bind_kv_cache(arena)
            # Head dim 32 runs row by row: six partials a row, 65 MB at the array's end.  The gathered
            # rows of a layer that shares another's pages put its plan 82 MB behind the array's start.
            cross, own = CrossAttention(64, 32, 0.1, 1), Attention(64, 128, 0.09, 64)
            shared = N.AttnDesc(64, 128, own.scale, 64, 0, 0, 0)
            x = torch.randn(tokens, 64, 32, device="cuda")
            pool = torch.randn(2, keys, 1, 32, device="cuda")
            out, y = torch.empty_like(q), torch.empty_like(x)
            want = own.forward(q, k, v, ctx)
            want_y = cross.forward(x, pool[0], pool[1], ctx)

            def self_call():
                return lib.nva_attention_forward_noalloc(
                    ctx.handle, arena.handle, ctypes.byref(shared), q.data_ptr(), None, None, tokens,
                    out.data_ptr())

            def cross_call():
                return lib.nva_cross_attention_forward_noalloc(
                    ctx.handle, ctypes.byref(cross._desc), x.data_ptr(), pool[0].data_ptr(),
                    pool[1].data_ptr(), keys, 32, tokens, y.data_ptr())

            for r in range(2):
                assert cross_call() == N.NVA_OK and self_call() == N.NVA_OK
                s1.synchronize()
                assert torch.equal(out, want) and torch.equal(y, want_y), f"turn {r}"
            y.zero_()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s1):
                refused = cross_call()
                message = lib.nva_last_error(ctx.handle)
                y.fill_(1.0)
            assert refused == N.NVA_E_ARG and b"do not fit one graph" in message
            assert cross_call() == N.NVA_OK and self_call() == N.NVA_OK
            s1.synchronize()
            assert torch.equal(out, want) and torch.equal(y, want_y), "after the refusal"
        finally:
            ctx.clear()
            arena.close()


def test_beside_the_decoder_layer(ctx):
    """A decoder step's self attention and cross attention in turn on one step: each keeps its plan,
    and new encoder rows replace the old."""
    from nanollvm_amd import Attention, KvCacheArena
    from span_checks import SharedStep, step_reference
    st = SharedStep([(12, 128)], [(i, 1) for i in range(12)], 64, seed=10)
    arena = KvCacheArena(ctx, 1, st.num_blocks, 64, 8, 128)
    try:
        pools = [Pool((16, 8, 128), [40 + i for i in range(12)], 11, True),
                 Pool((16, 8, 128), [300] * 12, 12, False)]
        q = torch.randn(12, 16, 128, device="cuda")
        k, v = (torch.randn(12, 8, 128, device="cuda") for _ in range(2))
        ctx.set(**st.context_args())
        ctx.share_prefixes(st.groups)
        ctx.bind_kv_cache(arena)
        self_attn, cross = Attention(16, 128, 0.09, 8), CrossAttention(16, 128, 0.09, 8)
        outs = []
        for pool, lens in zip(pools, ([40 + i for i in range(12)], [300] * 12)):
            ctx.set_encoder(pool.start, lens)
            for _ in range(2):
                x = self_attn.forward(q, k, v, ctx)
                outs.append((x, cross.forward(x, pool.k, pool.v, ctx), pool, lens))
        ctx.sync()
        kp, vp = (torch.from_numpy(a.reshape(-1, 8, 128)).cuda()
                  for a in (arena.get_key_cache(0), arena.get_value_cache(0)))
        want = step_reference(st, q, kp, vp, float(np.float32(0.09)))
        for x, y, pool, lens in outs:
            close(x, want, "self attention")
            close(y, reference(x, pool, [1] * 12, lens, pool.start, float(np.float32(0.09))),
                  "cross attention")
    finally:
        ctx.clear()
        arena.close()


def test_refusals(ctx):
    shape = (16, 8, 128)
    pool = Pool(shape, [10, 20], 13, True)
    q = torch.randn(2, 16, 128, device="cuda")
    layer = CrossAttention(16, 128, 0.1, 8)
    ctx.clear()
    with pytest.raises(NullPointerException):
        ctx.set_encoder([0], [1])
    ctx.set(is_prefill=False, context_lens=[3, 3])
    with pytest.raises(NullPointerException, match="encoder"):
        layer.forward(q, pool.k, pool.v, ctx)
    for start, lens in (([0], [1]), ([0, -1], [1, 1]), ([0, 0], [1, -1]), ([0, 0], [1])):
        with pytest.raises(IllegalArgumentException):
            ctx.set_encoder(start, lens)
    ctx.set_encoder([0, pool.rows - 5], [4, 6])
    with pytest.raises(IllegalArgumentException, match="encoder rows"):
        layer.forward(q, pool.k, pool.v, ctx)
    ctx.set_encoder([0, 2 ** 31 - 1], [4, 2 ** 31 - 1])
    with pytest.raises(IllegalArgumentException, match="encoder rows"):
        layer.forward(q, pool.k, pool.v, ctx)
    ctx.set_encoder(pool.start, [10, 20])
    with pytest.raises(IllegalArgumentException):      # three rows, two sequences
        layer.forward(torch.randn(3, 16, 128, device="cuda"), pool.k, pool.v, ctx)
    with pytest.raises(IllegalArgumentException):
        layer.forward(q.double(), pool.k, pool.v, ctx)
    with pytest.raises(IllegalArgumentException):
        layer.forward(q, pool.k[:, :4], pool.v[:, :4], ctx)
    with pytest.raises(IllegalArgumentException):
        layer.forward(q, pool.k[:-1], pool.v, ctx)
    with pytest.raises(IllegalArgumentException):      # rows not contiguous
        layer.forward(q, pool.k.transpose(1, 2).contiguous().transpose(1, 2), pool.v, ctx)
    with pytest.raises(IllegalArgumentException):      # a stride that is no multiple of 4 floats
        odd = torch.zeros(pool.rows, 1030, device="cuda")[:, :1024].unflatten(1, (8, 128))
        layer.forward(q, odd, odd, ctx)
    lib = N.load()
    out = torch.empty_like(q)
    desc = N.AttnDesc(16, 128, 0.1, 8, 64, 0, 0)       # a sliding window
    args = (q.data_ptr(), pool.k.data_ptr(), pool.v.data_ptr(), pool.rows, pool.k.stride(0), 2,
            out.data_ptr())
    assert lib.nva_cross_attention_forward(ctx.handle, ctypes.byref(desc), *args) == \
        N.NVA_E_UNSUPPORTED
    assert lib.nva_cross_attention_forward(ctx.handle, None, *args) == N.NVA_E_ARG
    with pytest.raises(UnsupportedShapeError):
        CrossAttention(2, 6, 0.1, 2).forward(torch.randn(2, 2, 6, device="cuda"),
                                             torch.randn(40, 2, 6, device="cuda"),
                                             torch.randn(40, 2, 6, device="cuda"), ctx)
    empty = torch.empty(0, 16, 128, device="cuda")
    assert layer.forward(empty, pool.k, pool.v, ctx).shape == (0, 16, 128)
    ctx.set_encoder([0, 0], [0, 0])                    # no rows at all: zeros
    none = torch.empty(0, 8, 128, device="cuda")
    assert torch.equal(layer.forward(q, none, none, ctx), torch.zeros_like(q))
    ctx.clear()
