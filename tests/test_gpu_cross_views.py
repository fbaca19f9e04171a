"""Views of packed projections as the keys and values of CrossAttention: every view whose heads lie in
order within a row gives the result of contiguous copies, bit for bit."""

import pytest
import torch

from gpu_checks import say
from nanollvm_amd import Context, CrossAttention, IllegalArgumentException

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2, 300])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_head_of_any_stride(rows, dim):
    """The one KV head of a packed [rows, width] projection, with its head axis put in by indexing,
    unsqueezing and unflattening: their strides of that axis differ."""
    hq, width = 8, 10 * dim
    torch.manual_seed(rows)
    qkv = torch.randn(rows, width, device="cuda")
    q = torch.randn(3, hq, dim, device="cuda")
    views = {
        "index": [qkv[:, None, a * dim:(a + 1) * dim] for a in (8, 9)],
        "unsqueeze": [qkv[:, a * dim:(a + 1) * dim].unsqueeze(1) for a in (8, 9)],
        "unflatten": [qkv[:, a * dim:(a + 1) * dim].unflatten(1, (1, dim)) for a in (8, 9)],
        "heads": [qkv.view(rows, 10, dim)[:, a:a + 1] for a in (8, 9)],
    }
    with Context(0) as ctx:
        layer = CrossAttention(hq, dim, 0.1, 1)
        ctx.set(is_prefill=False, context_lens=[1, 1, 1])
        ctx.set_encoder([0, 0, rows - 1], [rows, rows - 1, 1])
        want = layer.forward(q, *(x.contiguous() for x in views["heads"]), ctx)
        ctx.sync()
        for name, (k, v) in views.items():
            say(f"{name}: strides {k.stride()}, {rows} rows")
            got = layer.forward(q, k, v, ctx)
            ctx.sync()
            assert torch.equal(got, want), name
        with pytest.raises(IllegalArgumentException):  # dims that lie apart
            layer.forward(q, qkv[:, None, :2 * dim:2], qkv[:, None, :2 * dim:2], ctx)
        ctx.clear()
