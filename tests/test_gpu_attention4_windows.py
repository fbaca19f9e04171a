"""Windows as large as their type holds over the 4-bit arena, which leave every key in view, against 64
bits: rows long enough that their keys are split over workgroups."""

import pytest
import torch

from checks4 import close
from nanollvm_amd import Context
from test_gpu_attention4 import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 32, 2 ** 31 - 31, 2 ** 31 - 1])
def test_decode(ctx, d, window):
    case = Case([(3000, 1), (40, 1), (0, 1), (1999, 1)], 4, 2, d, block=64, window=window, seed=d)
    want = Case([(3000, 1), (40, 1), (0, 1), (1999, 1)], 4, 2, d, block=64, seed=d)
    got = case.run(ctx)
    close(got, case.want(), f"window {window}, decode")
    assert torch.equal(got, want.run(ctx))  # no window


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [2 ** 31 - 32, 2 ** 31 - 1])
def test_prefill(ctx, d, window):
    """Prompts too, with queries that see no key (five over two keys), whose keys end before they begin."""
    case = Case([(900, 70), (0, 33), (5, 1)], 4, 2, d, block=64, window=window, seed=d)
    close(case.run(ctx), case.want(), f"window {window}, prefill")
    few = Case([(0, 5)], 4, 2, d, block=64, window=window, seed=d)
    with few.arena(ctx) as a:
        step = few.step(decode=False)
        ctx.set(**{**step, "cu_seqlens_k": [0, 2], "max_seqlen_k": 2})
        ctx.bind_kv_cache(a)
        out = few.layer().forward(*(torch.from_numpy(x).cuda() for x in (few.q, few.k_new, few.v_new)),
                                  ctx).cpu()
        assert not out[:3].any() and out[3:].any(-1).all()
        ctx.clear()
