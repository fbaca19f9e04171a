"""RMSNorm and rotary positions of more than 2^24 rows, whose workgroups' threads pass 2^32: the bits of calls on
fewer of them."""

import numpy as np
import pytest
import torch

from nanollvm_amd import Context, RMSNorm, RotaryEmbedding

pytestmark = pytest.mark.gpu

ROWS = (1 << 24) + 9
# Rows about the borders of launches and of 2^32 threads.
PARTS = [(0, 40), ((1 << 23) - 20, (1 << 23) + 20), ((1 << 24) - 20, ROWS)]


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def test_norms(ctx):
    torch.manual_seed(1)
    x = torch.randn(ROWS, 12, device="cuda")
    norm = RMSNorm(torch.randn(12, device="cuda"), 1e-6)
    torch.cuda.synchronize()
    got = norm.forward(x, ctx)
    ctx.sync()
    assert bool(torch.isfinite(got).all())
    for a, b in PARTS:
        want = norm.forward(x[a:b].contiguous(), ctx)
        ctx.sync()
        assert torch.equal(got[a:b], want), (a, b)


@pytest.mark.parametrize("d,rd,interleaved", [(8, 8, False), (8, 8, True), (12, 6, True)])
def test_rotary_positions(ctx, d, rd, interleaved):
    """The row kernel's two forms and the per-token kernel."""
    torch.manual_seed(2)
    q, k = (torch.randn(ROWS, 1, d, device="cuda") for _ in range(2))
    positions = np.random.default_rng(3).integers(0, 1000, ROWS).astype(np.float32)
    rope = RotaryEmbedding.scaled(ctx, d, rd, 1000, 1e4, interleaved=interleaved)

    def forward(a, b):
        n = b - a
        ctx.set(True, cu_seqlens_q=[0, n], cu_seqlens_k=[0, n], max_seqlen_q=n, max_seqlen_k=n,
                positions=positions[a:b])
        torch.cuda.synchronize()
        out = rope.forward(None, q[a:b].contiguous(), k[a:b].contiguous(), ctx)
        ctx.sync()
        return out
    got = forward(0, ROWS)
    for a, b in PARTS:
        for x, y in zip(got, forward(a, b)):
            assert torch.equal(x[a:b], y), (a, b)
    ctx.clear()
    rope.close()
