"""How attention over the 4-bit arena divides its work: as many or few sequences as its lists treat apart,
several sequences a workgroup, one over many, and both at once.  Against 64 bits, as the other tests."""

import numpy as np
import pytest
import torch

from checks4 import close, dev
from nanollvm_amd import Context
from test_gpu_attention4 import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("seqs", [1, 63, 64, 65, 1023, 1024, 1025])
def test_sequences_about_the_rounds_of_a_list(ctx, seqs):
    r = np.random.default_rng(seqs)
    case = Case([(int(c), 1) for c in r.integers(0, 200, seqs)], 4, 2, 64, seed=seqs)
    close(case.run(ctx), case.want(), f"{seqs} rows")
    chunks = [(int(c), int(n)) for c, n in zip(r.integers(0, 60, seqs), r.integers(0, 3, seqs))]
    chunks[0] = (5, 2)
    case = Case(chunks, 2, 1, 64, seed=seqs)
    close(case.run(ctx, decode=False), case.want(), f"{seqs} chunks")


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 8), (128, 32, 8), (128, 40, 8), (256, 8, 8), (512, 8, 4)])
def test_many_segments_a_workgroup(ctx, d, hq, hkv):
    """More sequences times heads than workgroups, of one key to a thousand."""
    r = np.random.default_rng(d)
    lens = np.concatenate([r.integers(1, 100, 150), r.integers(1, 1000, 40), [1, 1, 2, 32, 33]])
    case = Case([(int(n) - 1, 1) for n in r.permutation(lens)], hq, hkv, d, block=64, seed=hq)
    close(case.run(ctx), case.want(), f"{hq}/{hkv}/{d}")


@pytest.mark.parametrize("d", [64, 128, 256, 512])
def test_one_long_sequence_among_short_ones(ctx, d):
    lens = [3, 1, 20000, 40, 1, 32, 7, 4000, 64, 65]
    case = Case([(n - 1, 1) for n in lens], 4, 1, d, block=256, seed=d, fill=False)
    close(case.run(ctx), case.want(), f"decode {d}")
    case = Case([(n, m) for n, m in zip(lens, [1, 9, 2, 3, 1, 0, 40, 17, 1, 2])], 4, 1, d, block=256,
                seed=d, fill=False)
    close(case.run(ctx), case.want(), f"chunks {d}")


@pytest.mark.parametrize("tiles", [1, 3, 4, 5, 8, 12, 16, 17])
def test_sequences_of_whole_chunks(ctx, tiles):
    """Every length the same, so that chunks end where segments do, or one key tile before or behind."""
    for seqs, extra in ((3, 0), (100, 0), (100, 1), (600, 0)):
        case = Case([(32 * tiles - 1 + extra, 1)] * seqs, 2, 1, 64, block=32, seed=tiles)
        close(case.run(ctx), case.want(), f"{seqs} of {tiles} tiles and {extra}")


def test_division_does_not_change_results(ctx):
    """A row alone and among others: sums in another order, the bar of the path."""
    seqs = [(5000, 1)] + [(60, 1)] * 90
    case = Case(seqs, 4, 2, 128, block=64, seed=4)
    alone = Case(seqs[:1], 4, 2, 128, block=64, seed=4)
    alone.q, alone.k_new, alone.v_new = (x[:1] for x in (case.q, case.k_new, case.v_new))
    alone.k, alone.v = case.k[:1], case.v[:1]
    got, one = case.run(ctx), alone.run(ctx)
    close(got[:1], one.double().cpu().numpy())
    assert torch.equal(case.run(ctx), got) and torch.equal(alone.run(ctx), one)


@pytest.mark.parametrize("d,limit", [(64, 48), (128, 48), (256, 36), (512, 8)])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (8, 8), (12, 2), (16, 1), (17, 1), (40, 2)])
def test_short_decode_rows_whole_and_split(ctx, d, limit, hq, hkv):
    """Rows up to the length that is not split, one key longer, and as short in a window."""
    for seqs, tiles, extra, window in ((3, limit, 0, 0), (3, limit, 1, 0), (150, 2, 0, 0), (2, 70, 0, 200),
                                       (1, 1, -31, 0)):
        n = 32 * tiles + extra
        lens = [n, max(1, n - 33), max(1, n // 2)] * (seqs // 3 + 1)
        case = Case([(m - 1, 1) for m in lens[:seqs]], hq, hkv, d, block=64, window=window, seed=tiles + hq)
        close(case.run(ctx), case.want(), f"{seqs} rows of {n}, window {window}")


def test_short_decode_rows_among_empty_and_padded_ones(ctx):
    """What a row of no keys is, and rows of the step that a call leaves out."""
    case = Case([(40, 1), (5, 1), (90, 1)], 4, 2, 64, block=32, seed=2)
    with case.arena(ctx) as a:
        step = case.step()
        step["context_lens"] = [41, 0, 91]
        ctx.set(**step)
        ctx.bind_kv_cache(a)
        q, k, v = dev(case.q), dev(case.k_new), dev(case.v_new)
        out = case.layer().forward(q, k, v, ctx)
        want = case.want()
        assert not out[1].any()
        close(out[[0, 2]], want[[0, 2]])
        step["context_lens"] = [41, 6, 91]
        step["slot_mapping"] = step["slot_mapping"][:2]
        ctx.set(**step)
        ctx.bind_kv_cache(a)
        close(case.layer().forward(q[:2], k[:2], v[:2], ctx), want[:2])
        ctx.clear()
