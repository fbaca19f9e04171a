"""Rotary positions written over their own inputs, of any layout: the bits of a call whose outputs are apart."""

import numpy as np
import pytest
import torch

from checks4 import dev, frequencies, rotate
from nanollvm_amd import Attention, Context, KvCacheArena, RMSNorm, RotaryEmbedding, _native

pytestmark = pytest.mark.gpu

# Head dim, dims that turn: layouts of the row kernel, of the per-token kernel, and of the latter alone.
LAYOUTS = [(64, 64), (64, 32), (128, 128), (128, 24), (256, 64), (512, 264), (80, 80), (80, 32), (96, 96),
           (96, 50), (6, 4), (6, 6), (128, 10), (512, 10), (256, 2), (100, 60)]


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def inputs(tokens, hq, hk, d):
    r = np.random.default_rng(d)
    return [r.standard_normal((tokens, h, d)).astype(np.float32) for h in (hq, hk)]


def step(ctx, positions):
    n = len(positions)
    ctx.set(True, cu_seqlens_q=[0, n], cu_seqlens_k=[0, n], max_seqlen_q=n, max_seqlen_k=n,
            positions=np.asarray(positions, np.float32))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rd", LAYOUTS)
def test_forward(ctx, d, rd, interleaved):
    tokens, hq, hk = 33, 9, 3
    pos = np.random.default_rng(rd).integers(0, 5000, tokens)
    q, k = inputs(tokens, hq, hk, d)
    rope = RotaryEmbedding.scaled(ctx, d, rd, 5000, 1e4, interleaved=interleaved)
    step(ctx, pos)
    want = rope.forward(None, dev(q), dev(k), ctx)
    f, _ = frequencies(rd, 1e4)
    # (A pair's two products and their sum: 4.5 half steps of its largest.)
    assert np.abs(want[0].cpu().numpy() - rotate(q, pos, f, 1.0, interleaved)).max() <= (
        4.5 * 2.0 ** -24 * np.abs(q).max())
    a, b = dev(q), dev(k)
    ctx.sync()
    assert _native.load().nva_rope_forward(ctx.handle, rope.handle, a.data_ptr(), b.data_ptr(), tokens, hq,
                                           hk, a.data_ptr(), b.data_ptr()) == _native.NVA_OK
    ctx.sync()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    rope.close()


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("d,rd,interleaved", [(64, 32, False), (64, 64, True), (64, 12, True), (256, 50, False),
                                              (128, 10, True), (512, 260, False)])
def test_the_fused_call(ctx, d, rd, interleaved, norms):
    n, hq, hk = 21, 6, 2
    q, k = inputs(n, hq, hk, d)
    v = inputs(n, hk, hk, d)[1]
    r = np.random.default_rng(4)
    weights = [dev(r.standard_normal(d).astype(np.float32)) for _ in range(2)]
    qn, kn = (RMSNorm(w, 1e-6) if norms else None for w in weights)
    rope = RotaryEmbedding.scaled(ctx, d, rd, 64, 1e4, interleaved=interleaved)
    attn = Attention(hq, d, d ** -0.5, hk)
    got = []
    for apart in (True, False):
        arena = KvCacheArena(ctx, 1, 2, 16, hk, d)
        ctx.set(is_prefill=True, cu_seqlens_q=[0, n], cu_seqlens_k=[0, n], max_seqlen_q=n, max_seqlen_k=n,
                slot_mapping=np.arange(n), positions=np.arange(n, dtype=np.float32))
        ctx.bind_kv_cache(arena)
        a, b = dev(q), dev(k)
        q_out, k_out = (torch.empty_like(a), torch.empty_like(b)) if apart else (a, b)
        out = attn.forward_with_norm_rope(rope, None, a, b, dev(v), ctx, qn, kn, q_out=q_out, k_out=k_out)
        ctx.sync()
        got.append([x.cpu().numpy() for x in (q_out, k_out, out)] + [arena.get_key_cache(0)])
        ctx.clear()
        arena.close()
    for x, y in zip(*got):
        assert np.array_equal(x, y)
    rope.close()
