"""Infinities and NaN in V at the edges of what a row sees: the result of a dim is what
sum_t w_t v_t is in 64 bits, with every weight w_t above 0, so an infinity at the first or last key
of a range gives an infinity of its sign (not NaN), a NaN gives NaN, and no other dim or row changes.

The lengths end inside the blocks of 8, 16 and 32 keys that the kernels take at a time, where the
lanes behind the last key and in front of the first must not bring its V in again at weight 0.
Finite values are held to the bar of every attention path (max-abs 1e-4, rel-L2 1e-5)."""

import numpy as np
import pytest
import torch

from gpu_checks import MAX_ABS, REL_L2, arena_views, say
from span_checks import SharedStep
from nanollvm_amd import Attention, Context, CrossAttention, KvCacheArena

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def weighted_sum(q, k, v, scale):
    """softmax(q k^T scale) v, q [hq, d], k and v [keys, hkv, d], all of the keys seen."""
    hq, hkv = q.shape[0], k.shape[1]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for h in range(hq):
        kv = h // (hq // hkv)
        s = (k[:, kv].double() @ q[h].double()) * scale
        w = torch.softmax(s, 0)
        assert float(w.min()) > 0
        out[h] = (w[:, None] * v[:, kv].double()).sum(0)
    return out


def same(got, want, name, some=True):
    for what in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(what(got), what(want)), f"{name}: {what.__name__} differs"
    fine = torch.isfinite(want)
    err = (got.double() - want)[fine]
    rel = float(err.norm() / want[fine].norm())
    say(f"{name}: max_abs={float(err.abs().max()):.3e} rel_l2={rel:.3e}, "
        f"{int((~fine).sum())} not finite")
    assert int((~fine).sum()) > 0 or not some
    assert float(err.abs().max()) <= MAX_ABS and rel <= REL_L2


def plant(v, first, last):
    """Dims 1 and 2 of the last key's row of v, 5 and 6 of the first one's."""
    v[last, :, 1], v[last, :, 2] = INF, -INF
    v[first, :, 5], v[first, :, 6] = -INF, float("nan")


SHAPES = [(12, 12, 64), (16, 8, 128), (40, 8, 128), (34, 2, 64), (4, 1, 256), (8, 1, 512)]
BY_ROWS = [(12, 12, 32), (6, 3, 16)]  # head dims that run row by row


@pytest.mark.parametrize("shape", SHAPES + BY_ROWS, ids=str)
@pytest.mark.parametrize("queries", [1, 4, 130])
def test_ends_of_encoder_states(ctx, shape, queries):
    hq, hkv, d = shape
    lens = [2, 15, 17, 33, 63, 65, 101, 300]
    g = torch.Generator(device="cuda").manual_seed(31)
    start = np.concatenate([[0], np.cumsum([n + 3 for n in lens])])[:-1]
    rows = int(start[-1]) + lens[-1] + 3
    k, v = (torch.full((rows, hkv, d), float("nan"), device="cuda") for _ in range(2))
    for s, n in zip(start, lens):
        for x in (k, v):
            x[s:s + n] = torch.randn(n, hkv, d, device="cuda", generator=g)
        plant(v, s, s + n - 1)
    q = torch.randn(queries * len(lens), hq, d, device="cuda", generator=g)
    if queries == 1:
        ctx.set(is_prefill=False, context_lens=[1] * len(lens))
    else:
        cu = np.arange(len(lens) + 1) * queries
        ctx.set(is_prefill=True, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=queries,
                max_seqlen_k=queries)
    ctx.set_encoder(start, lens)
    scale = float(np.float32(d ** -0.5))
    out = CrossAttention(hq, d, scale, hkv).forward(q, k, v, ctx)
    ctx.sync()
    ctx.clear()
    for i, (s, n) in enumerate(zip(start, lens)):
        for r in {0, queries // 2, queries - 1}:
            at = i * queries + r
            same(out[at], weighted_sum(q[at], k[s:s + n], v[s:s + n], scale),
                 f"{shape}, query {r} over {n} rows")


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("block,tokens,rows", [(64, 37, 3), (16, 192, 6), (256, 129, 9)])
def test_ends_of_shared_prefixes(ctx, shape, block, tokens, rows):
    """An infinity at the prefix's last key and at its first, and another at each row's own last one
    (the token the step stores)."""
    ends(ctx, shape, block, [(rows, -(-tokens // block) * block)], rows, [(0, rows, tokens)])


@pytest.mark.parametrize("shape", SHAPES + BY_ROWS, ids=str)
@pytest.mark.parametrize("block,tokens,rows", [(64, 192, 60), (24, 31, 5), (256, 129, 90)])
def test_ends_of_shared_prefixes_beside_rows(ctx, shape, block, tokens, rows):
    """The same where the rows' own keys, or all, are read row by row."""
    ends(ctx, shape, block, [(rows, -(-tokens // block) * block)], rows, [(0, rows, tokens)])


@pytest.mark.parametrize("shape", SHAPES + BY_ROWS + [(4, 2, 8), (28, 4, 128), (6, 2, 256)], ids=str)
@pytest.mark.parametrize("window", [0, 45])
@pytest.mark.parametrize("block", [1, 24, 64])
def test_ends_of_rows_read_apart(ctx, shape, window, block):
    """The same without groups, and under a window whose first key lies inside a block."""
    ends(ctx, shape, block, [(9, 0)], 9, [], window)


def ends(ctx, shape, block, groups, rows, named, window=0):
    hq, hkv, d = shape
    st = SharedStep(groups, [(40 + 7 * i % 61, 1) for i in range(rows)], block, seed=32)
    g = torch.Generator(device="cuda").manual_seed(32)
    arena = KvCacheArena(ctx, 1, st.num_blocks, block, hkv, d)
    try:
        n = st.num_blocks * block
        kp, vp = (x.view(n, hkv, d) for x in arena_views(arena))
        for x in (kp, vp):
            x.fill_(float("nan"))
            for s in st.slots:
                x[torch.from_numpy(s).cuda()] = torch.randn(len(s), hkv, d, device="cuda",
                                                            generator=g)
        q = torch.randn(rows, hq, d, device="cuda", generator=g)
        k, v = (torch.randn(rows, hkv, d, device="cuda", generator=g) for _ in range(2))
        v[:, :, 3] = -INF
        for s in st.slots:
            first = max(0, len(s) - window) if window else 0
            plant(vp, s[first], s[(named[0][2] if named else len(s) - 1) - 1])
        ctx.set(**st.context_args())
        ctx.share_prefixes(named)
        ctx.bind_kv_cache(arena)
        scale = float(np.float32(d ** -0.5))
        out = Attention(hq, d, scale, hkv, window, 0).forward(q, k, v, ctx)
        ctx.sync()
        for i in {0, 1, rows // 2, rows - 1}:
            s = st.slots[i][-window:] if window else st.slots[i]
            at = torch.from_numpy(s).cuda()
            same(out[i], weighted_sum(q[i], kp[at], vp[at], scale),
                 f"{shape}, pages of {block}, row {i} over {len(s)} keys")
    finally:
        ctx.clear()
        arena.close()


@pytest.mark.parametrize("shape", [(12, 12, 64), (16, 8, 128), (4, 1, 256), (8, 1, 512)], ids=str)
@pytest.mark.parametrize("queries", [1, 30, 300])
def test_nan_beside_a_score_of_minus_infinity(ctx, shape, queries):
    """A key of score -inf has weight 0, and 0 times NaN or infinity is NaN, in that dim alone."""
    hq, hkv, d = shape
    g = torch.Generator(device="cuda").manual_seed(33)
    q = torch.randn(queries, hq, d, device="cuda", generator=g)
    q[..., 0] = q[..., 0].abs() + 0.5
    k, v = (torch.randn(100, hkv, d, device="cuda", generator=g) for _ in range(2))
    k[30, :, 0], v[30, :, 4], v[30, :, 7] = -INF, float("nan"), INF
    cu = [0, queries]
    ctx.set(is_prefill=True, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=queries,
            max_seqlen_k=queries)
    ctx.set_encoder([0], [100])
    scale = float(np.float32(d ** -0.5))
    out = CrossAttention(hq, d, scale, hkv).forward(q, k, v, ctx)
    ctx.sync()
    ctx.clear()
    assert bool(torch.isnan(out[..., [4, 7]]).all())
    seen = torch.arange(100, device="cuda") != 30
    rest = [i for i in range(d) if i not in (4, 7)]
    for r in {0, queries // 2, queries - 1}:
        want = weighted_sum(q[r], k[seen], v[seen], scale)[:, rest]
        rel = float((out[r][:, rest].double() - want).norm() / want.norm())
        say(f"{shape}, query {r} of {queries} beside a score of -inf: rel_l2={rel:.3e}")
        assert rel <= REL_L2


@pytest.mark.parametrize("shape", SHAPES + [(8, 8, 128), (32, 8, 64)] + BY_ROWS, ids=str)
@pytest.mark.parametrize("window", [0, 21])
@pytest.mark.parametrize("lens,cached", [((20,), 0), ((60, 3, 37), 0), ((200,), 0), ((40, 2), 150),
                                         ((2, 3, 1) * 150, 0), ((700, 300), 0)], ids=str)
def test_values_that_a_query_does_not_see(ctx, shape, window, lens, cached):
    """Infinities and NaN in V behind a query (later tokens of its prompt) or before its window: they
    reach the queries that see them alone, over tiles of either kind, rows, and split ones."""
    hq, hkv, d = shape
    st = SharedStep([(len(lens), 0)], [(cached, n) for n in lens], 64, seed=34, decode=False)
    g = torch.Generator(device="cuda").manual_seed(34)
    arena = KvCacheArena(ctx, 1, st.num_blocks, 64, hkv, d)
    try:
        kp, vp = (x.view(-1, hkv, d) for x in arena_views(arena))
        for x in (kp, vp):
            x.normal_(generator=g)
        q = torch.randn(st.tokens, hq, d, device="cuda", generator=g)
        k, v = (torch.randn(st.tokens, hkv, d, device="cuda", generator=g) for _ in range(2))
        picked = set()
        for b, n in enumerate(lens):
            a = int(st.cu_q[b])
            v[a + n - 1, :, 1] = INF
            v[a + n - 1 - n // 3, :, 2] = -INF
            v[a + n // 2, :, 5] = float("nan")
            if b % 50 == 0 or len(lens) < 9:
                picked |= {(b, j) for j in (0, n // 3, n // 2, n - 2 - n // 3, n - 2, n - 1) if 0 <= j < n}
        ctx.set(**st.context_args())
        ctx.bind_kv_cache(arena)
        scale = float(np.float32(d ** -0.5))
        out = Attention(hq, d, scale, hkv, window, 0).forward(q, k, v, ctx)
        ctx.sync()
        odd = 0
        for b, j in sorted(picked):
            keys = st.keys[b] - lens[b] + j + 1
            at = torch.from_numpy(st.slots[b][max(0, keys - window) if window else 0:keys]).cuda()
            want = weighted_sum(q[int(st.cu_q[b]) + j], kp[at], vp[at], scale)
            odd += int((~torch.isfinite(want)).sum())
            same(out[int(st.cu_q[b]) + j], want, f"{shape} {len(lens)} prompts: query {j} of {b}",
                 some=False)
        assert odd > 0
        finite = torch.isfinite(out[:, :, 6:])
        assert bool(finite.all())
    finally:
        ctx.clear()
        arena.close()
