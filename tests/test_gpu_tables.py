"""Block tables that grow and shrink on the device, against the same rules over Python lists: random
histories, steps that do not fit, captured steps, and the sizes where the kernels change."""

import numpy as np
import pytest
import torch

from checks4 import Tables, dev
from nanollvm_amd import (Attention, BlockTables, Context, IllegalArgumentException, KvCacheArena,
                          NvaError, RotaryEmbedding, UnsupportedShapeError)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def i32(x):
    return dev(np.asarray(x, np.int32))


@pytest.mark.parametrize("seqs,block,blocks", [(1, 1, 40), (3, 16, 12), (70, 32, 300),
                                               (1030, 8, 5000)])
def test_random_histories(ctx, seqs, block, blocks):
    r = np.random.default_rng(seqs)
    pages = r.permutation(3 * blocks)[:blocks]
    most = max(8, 4 * block)
    max_tokens = 10 * most
    plain = Tables(seqs, max_tokens, blocks, block, pages)
    with BlockTables(ctx, seqs, max_tokens, seqs * most + 9, blocks, block, pages) as t:
        for turn in range(12):
            n = seqs if turn % 3 else int(r.integers(0, seqs + 1))  # the first n rows
            new = r.integers(0, most + 1, n) * (r.random(n) < 0.7)
            keep = None
            if turn % 2:
                lens = np.asarray(plain.lens[:n])
                keep = np.where(r.random(n) < 0.6, lens, (r.random(n) * (lens + 1)).astype(int))
            tokens = int(new.sum()) + int(r.integers(0, 9))
            got = plain.extend(new.tolist(), tokens, most, None if keep is None else keep.tolist())
            ctx.extend(t, i32(new), tokens, most, None if keep is None else i32(keep))
            plain.check(t, got, f"turn {turn}: {got[0]}")


@pytest.mark.parametrize("tokens", [4095, 4096, 4097, 20000])
def test_long_prompts(ctx, tokens):
    """Either side of the step size from which slots are written apart."""
    new = [tokens - 1000, 0, 1, 999]
    plain = Tables(4, tokens, 1000, 32)
    with BlockTables(ctx, 4, tokens, tokens + 5, 1000, 32) as t:
        for keep in (None, [7, 0, 1, 64], [0, 0, 0, 0]):
            got = plain.extend(new, tokens + 5, tokens, keep)
            ctx.extend(t, i32(new), tokens + 5, tokens, None if keep is None else i32(keep))
            plain.check(t, got, str(keep))
            if keep is None:
                plain_again = plain.extend([0] * 4, 0, 0, [7, 0, 1, 64])
                ctx.extend(t, i32([0] * 4), 0, 0, i32([7, 0, 1, 64]))
                plain.check(t, plain_again, "shrunk")
        got = plain.extend([1, 1, 1, tokens], tokens + 5, tokens)
        ctx.extend(t, i32([1, 1, 1, tokens]), tokens + 5, tokens)
        assert got[0][0] != 0
        plain.check(t, got, "too many, apart")


def test_keeping_less_and_extending_again_gives_the_same_blocks(ctx):
    with BlockTables(ctx, 5, 400, 2000, 64, 16) as t:
        ctx.extend(t, i32([30, 16, 0, 1, 100]), 147, 100)
        ctx.extend(t, i32([9, 50, 33, 0, 1]), 93, 50)
        first = [t.block_tables.clone(), t.slots.clone()]
        for _ in range(2):
            ctx.extend(t, i32([9, 50, 33, 0, 1]), 93, 50, i32([30, 16, 0, 1, 100]))
            assert torch.equal(t.block_tables, first[0]) and torch.equal(t.slots, first[1])


def test_steps_that_do_not_fit_change_nothing(ctx):
    plain = Tables(3, 100, 10, 8)
    with BlockTables(ctx, 3, 100, 50, 10, 8) as t:
        def both(new, tokens, most, keep=None):
            got = plain.extend(new, tokens, most, keep)
            ctx.extend(t, i32(new), tokens, most, None if keep is None else i32(keep))
            plain.check(t, got, f"{new} {keep}")
            return got[0][0]
        assert both([20, 3, 9], 32, 20) == 0
        assert both([1, -1, 1], 9, 9) == 1           # below 0
        assert both([1, 1, 10], 20, 9) == 1          # above max_new
        assert both([1, 1, 1], 9, 9, [20, 4, 9]) == 1  # keeps more than there is
        assert both([1, 1, 1], 9, 9, [-1, 3, 9]) == 1
        assert both([1, 2 ** 31 - 1, 1], 9, 2 ** 31 - 1) == 1  # beyond max_tokens
        assert both([5, 5, 5], 14, 9) == 2           # more than the step's rows
        assert both([40, 5, 5], 50, 40) == 3         # more blocks than there are
        assert both([1, 1, 1], 3, 1) == 0            # and the next goes on
        assert both([0, 0, 0], 0, 0, [0, 0, 0]) == 0
        assert both([50, 0, 30], 80 - 30, 50) == 2
        assert both([50, 0, 0], 50, 50) == 0


def test_captured_steps_act_on_the_lengths_they_find(ctx):
    plain = Tables(4, 300, 40, 16)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), Context(0, stream=s) as c, BlockTables(c, 4, 300, 8, 40, 16) as t:
        new = i32([1, 1, 0, 1])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.extend(t, new, 4, 8)
        for turn in range(40):
            if turn == 20:
                new.copy_(i32([3, 0, 2, 1]))
            if turn == 30:  # an eager step between the replays
                got = plain.extend([0, 0, 1, 0], 1, 8, [5, 0, 0, 17])
                c.extend(t, i32([0, 0, 1, 0]), 1, 8, i32([5, 0, 0, 17]))
                plain.check(t, got, "eager")
                c.extend(t, i32([0] * 4), 4, 8)
            s.synchronize()
            n = new.tolist()
            got = plain.extend(n, 4, 8)
            g.replay()
            junk = torch.randn(1000, device="cuda").sum()
            s.synchronize()
            t._step = (4, 4)
            plain.check(t, got, f"replay {turn} {float(junk):.1f}")


def test_as_many_rows_as_there_may_be(ctx):
    n = 4000
    plain = Tables(n, 50, 9000, 8)
    new = np.random.default_rng(0).integers(0, 17, n)
    with BlockTables(ctx, n, 50, 40000, 9000, 8) as t:
        for _ in range(2):
            got = plain.extend(new.tolist(), int(new.sum()), 16)
            ctx.extend(t, i32(new), int(new.sum()), 16)
            plain.check(t, got)


def test_refusals(ctx):
    for bad in (dict(max_seqs=0), dict(max_tokens=0), dict(max_step_tokens=-1), dict(num_blocks=0),
                dict(block_size=0), dict(pages=[0, 1, 2, 2]), dict(pages=[0, 1, 2, -1]),
                dict(pages=[0, 1, 2])):
        args = dict(max_seqs=2, max_tokens=10, max_step_tokens=10, num_blocks=4, block_size=8,
                    pages=None)
        with pytest.raises(IllegalArgumentException):
            BlockTables(ctx, **{**args, **bad})
    with pytest.raises(UnsupportedShapeError):
        BlockTables(ctx, 4001, 10, 10, 4, 8)
    with pytest.raises(UnsupportedShapeError):
        BlockTables(ctx, 1, 10, 10, 2, 8, pages=[0, 2 ** 31 - 1])
    with BlockTables(ctx, 2, 10, 10, 4, 8) as t:
        one = i32([1, 1])
        for new, tokens, most, keep in ((i32([1, 1, 1]), 3, 1, None), (one, 11, 1, None),
                                        (one, -1, 1, None), (one, 2, -1, None), (one.long(), 2, 1, None),
                                        (one.cpu(), 2, 1, None), (one, 2, 1, i32([0])),
                                        (one[None], 2, 1, None)):
            with pytest.raises(IllegalArgumentException):
                ctx.extend(t, new, tokens, most, keep)
        with Context(0) as other:
            with pytest.raises(IllegalArgumentException):
                other.extend(t, one, 2, 1)


def test_other_attention_has_no_step_then(ctx):
    """The fp32 arena's attention plans on the host: after extend it has no step, and none stays from
    before; positions of the step are bounded by the tables."""
    x = torch.zeros(2, 1, 64, device="cuda")
    arena = KvCacheArena(ctx, 1, 4, 8, 1, 64)
    rope = RotaryEmbedding(ctx, 64, 64, 16, 1e4)
    small = RotaryEmbedding(ctx, 64, 64, 9, 1e4)
    attn = Attention(1, 64, 0.1, 1)
    with BlockTables(ctx, 2, 10, 10, 4, 8) as t:
        ctx.set(False, context_lens=[1, 1], block_tables=[[0], [1]], slot_mapping=[0, 8],
                positions=[0, 0])
        ctx.bind_kv_cache(arena)
        attn.forward(x, x, x, ctx)
        ctx.extend(t, i32([1, 1]), 2, 1)
        for call in (lambda: attn.forward(x, x, x, ctx),
                     lambda: attn.forward_with_rope(rope, None, x, x, x, ctx),
                     lambda: ctx.share_prefixes([(0, 2, 1)]), lambda: ctx.set_encoder([0, 0], [1, 1]),
                     lambda: ctx.set_positions([0, 0])):
            with pytest.raises(NvaError):
                call()
        rope.forward(None, x, x, ctx)
        with pytest.raises(IllegalArgumentException):
            small.forward(None, x, x, ctx)
        with pytest.raises(IllegalArgumentException):
            rope.forward(None, torch.zeros(3, 1, 64, device="cuda"),
                         torch.zeros(3, 1, 64, device="cuda"), ctx)
    with pytest.raises(NvaError):
        rope.forward(None, x, x, ctx)  # the tables are gone
    ctx.clear()
    arena.close()
