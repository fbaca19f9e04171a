"""Rotary positions of part of a head, of either pairing, with scaled frequencies, against 64 bits; in
RotaryEmbedding.forward and in the fused calls, where they agree with their parts bit for bit.

Bar: the table is fp32 and a turn two products and a sum in fp32: half a step of cos or sin, of each
product and of the sum, each 2^-24 of (|cos| + |sin|) times the largest of the pair at most, so a value is
off by at most 3 sqrt(2) * 2^-24 of that (4.5 here), times the amplitude."""

import numpy as np
import pytest
import torch

from checks4 import dev, frequencies, rotate
from nanollvm_amd import (Attention, Context, IllegalArgumentException, KvCacheArena, RMSNorm,
                          RotaryEmbedding)

pytestmark = pytest.mark.gpu

SCALINGS = [
    dict(scaling="none"),
    dict(scaling="linear", factor=4.0),
    dict(scaling="ntk", factor=8.0),
    dict(scaling="yarn", factor=4.0, original_max_position=2048, low=1.0, high=32.0),
    dict(scaling="bands", factor=8.0, original_max_position=1024, low=1.0, high=4.0),
]


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def data(tokens, hq, hk, d, seed):
    r = np.random.default_rng(seed)
    return [r.standard_normal((tokens, h, d)).astype(np.float32) for h in (hq, hk)]


def step(ctx, positions):
    n = len(positions)
    ctx.set(True, cu_seqlens_q=[0, n], cu_seqlens_k=[0, n], max_seqlen_q=n, max_seqlen_k=n,
            positions=np.asarray(positions, np.float32))


def check(got, x, positions, f, amplitude, interleaved):
    want = rotate(x, positions, f, amplitude, interleaved)
    got = got.cpu().numpy().astype(np.float64)
    rd = 2 * len(f)
    assert np.array_equal(got[..., rd:], x[..., rd:])  # the others pass through
    p = np.abs(x[..., :rd].astype(np.float64))
    big = (np.maximum(p[..., 0::2], p[..., 1::2]).repeat(2, -1) if interleaved else
           np.tile(np.maximum(p[..., :rd // 2], p[..., rd // 2:]), 2))
    bound = 4.5 * 2.0 ** -24 * amplitude * big + 1e-37
    err = np.abs(got - want)[..., :rd]
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rd", [(8, 8), (8, 2), (16, 8), (32, 20), (64, 64), (64, 32), (64, 6),
                                  (80, 32), (96, 96), (128, 128), (128, 64), (128, 24), (256, 64),
                                  (256, 256), (512, 512), (512, 128), (512, 264), (512, 10),
                                  (6, 4)])
def test_layouts(ctx, d, rd, interleaved):
    q, k = data(5, 3, 2, d, d + rd)
    pos = [0, 1, 77, 39999, 40959]
    f, a = frequencies(rd, 1e6)
    rope = RotaryEmbedding.scaled(ctx, d, rd, 40960, 1e6, interleaved=interleaved)
    step(ctx, pos)
    got = rope.forward(None, dev(q), dev(k), ctx)
    for g, x in zip(got, (q, k)):
        check(g, x, pos, f, a, interleaved)
    rope.close()


@pytest.mark.parametrize("how", SCALINGS, ids=lambda h: h["scaling"])
@pytest.mark.parametrize("rd", [2, 64, 128])
def test_scalings_far_out(ctx, how, rd):
    q, k = data(4, 2, 1, 128, rd)
    pos = [0, 3000, 99999, 131071]
    for base in (1e4, 5e5):
        f, a = frequencies(rd, base, **how)
        rope = RotaryEmbedding.scaled(ctx, 128, rd, 131072, base, interleaved=True, **how)
        step(ctx, pos)
        for g, x in zip(rope.forward(None, dev(q), dev(k), ctx), (q, k)):
            check(g, x, pos, f, a, True)
        rope.close()


def test_amplitude(ctx):
    q, k = data(3, 2, 1, 64, 5)
    rope = RotaryEmbedding.scaled(ctx, 64, 64, 100, 1e4, amplitude=1.25, **SCALINGS[3])
    step(ctx, [1, 2, 99])
    f, _ = frequencies(64, 1e4, **SCALINGS[3])
    check(rope.forward(None, dev(q), dev(k), ctx)[0], q, [1, 2, 99], f, 1.25, False)
    rope.close()


@pytest.mark.parametrize("tokens", [1, 2, 63, 700])
def test_lengths(ctx, tokens):
    q, k = data(tokens, 9, 1, 128, tokens)
    pos = np.random.default_rng(tokens).integers(0, 5000, tokens)
    f, a = frequencies(32, 1e4)
    rope = RotaryEmbedding.scaled(ctx, 128, 32, 5000, 1e4)
    step(ctx, pos)
    for g, x in zip(rope.forward(None, dev(q), dev(k), ctx), (q, k)):
        check(g, x, pos, f, a, False)
    empty = torch.zeros(0, 9, 128, device="cuda"), torch.zeros(0, 1, 128, device="cuda")
    assert rope.forward(None, *empty, ctx)[0].shape == (0, 9, 128)
    rope.close()


@pytest.mark.parametrize("d,rd,interleaved", [(64, 32, False), (64, 64, True), (128, 32, False),
                                              (256, 64, True), (512, 256, False), (64, 12, False),
                                              (128, 10, True)])
@pytest.mark.parametrize("norms", [False, True])
def test_fused_calls_are_their_parts(ctx, d, rd, interleaved, norms):
    """Norm, rotation, store and attention as one call, and on packed rows, against norms, rotation and
    Attention.forward one after the other: the same bits in q, k, pages and output."""
    hq, hk, n, cached = 4, 2, 6, 3
    q, k = data(n, hq, hk, d, 1)
    v = data(n, hk, hk, d, 2)[0]
    r = np.random.default_rng(4)
    weights = [dev(r.standard_normal(d).astype(np.float32)) for _ in range(2)]
    rope = RotaryEmbedding.scaled(ctx, d, rd, 64, 1e4, interleaved=interleaved)
    attn = Attention(hq, d, d ** -0.5, hk)
    pos = np.arange(cached, cached + n, dtype=np.float32)
    when = dict(is_prefill=True, cu_seqlens_q=[0, n], cu_seqlens_k=[0, cached + n], max_seqlen_q=n,
                max_seqlen_k=cached + n, slot_mapping=np.arange(cached, cached + n),
                block_tables=[[0]], positions=pos)
    got = []
    for way in range(3):
        arena = KvCacheArena(ctx, 1, 1, 16, hk, d)
        ctx.set(**when)
        ctx.bind_kv_cache(arena)
        qn, kn = (RMSNorm(w, 1e-6) if norms else None for w in weights)
        qo, ko = (torch.empty(n, h, d, device="cuda") for h in (hq, hk))
        if way == 0:
            qx = qn.forward(dev(q), ctx) if norms else dev(q)
            kx = kn.forward(dev(k), ctx) if norms else dev(k)
            qo, ko = rope.forward(None, qx, kx, ctx)
            out = attn.forward(qo, ko, dev(v), ctx)
        elif way == 1:
            out = attn.forward_with_norm_rope(rope, None, dev(q), dev(k), dev(v), ctx, qn, kn,
                                              q_out=qo, k_out=ko)
        else:
            packed = np.concatenate([x.reshape(n, -1) for x in (q, k, v)], 1)
            out = attn.forward_packed_qkv(rope, None, dev(packed), ctx, qn, kn, q_out=qo, k_out=ko)
        ctx.sync()
        got.append([x.cpu().numpy() for x in (qo, ko, out)] +
                   [arena.get_key_cache(0), arena.get_value_cache(0)])
        ctx.clear()
        arena.close()
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert np.array_equal(a, b)
    rope.close()


def test_the_whole_head_in_halves_is_the_reference_kernel(ctx):
    """A table of the reference's layout runs the same kernel as a table the caller brings."""
    q, k = data(9, 4, 2, 128, 8)
    pos = np.arange(9) * 100
    f, _ = frequencies(128, 1e4)
    a = np.outer(np.arange(1000), f)
    table = np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)
    one = RotaryEmbedding.scaled(ctx, 128, 128, 1000, 1e4)
    two = RotaryEmbedding(ctx, 128, 128, 1000, 1e4, cos_sin=table)
    step(ctx, pos)
    a, b = (r.forward(None, dev(q), dev(k), ctx)[0].cpu().numpy().astype(np.float64) for r in (one, two))
    assert np.abs(a - b).max() <= 2.0 ** -23 * np.abs(q).max()
    one.close()
    two.close()


def test_refusals(ctx):
    good = dict(head_size=64, rotary_dim=32, max_position_embeddings=100, base=1e4)
    for bad in (dict(rotary_dim=0), dict(rotary_dim=31), dict(rotary_dim=66), dict(head_size=33),
                dict(max_position_embeddings=0), dict(base=1.0), dict(base=float("nan")),
                dict(scaling="cubic"), dict(scaling="linear", factor=0.5),
                dict(scaling="linear", factor=float("inf")), dict(scaling="yarn", factor=2.0),
                dict(scaling="yarn", factor=2.0, original_max_position=100, low=4.0, high=1.0),
                dict(scaling="bands", factor=2.0, original_max_position=100, low=0.0, high=1.0),
                dict(amplitude=-1.0), dict(amplitude=float("nan"))):
        with pytest.raises(IllegalArgumentException):
            RotaryEmbedding.scaled(ctx, **{**good, **bad})
    rope = RotaryEmbedding.scaled(ctx, **good)
    step(ctx, [0, 100])
    x = torch.zeros(2, 1, 64, device="cuda")
    with pytest.raises(IllegalArgumentException):
        rope.forward(None, x, x, ctx)  # position 100 of 100
    rope.close()
