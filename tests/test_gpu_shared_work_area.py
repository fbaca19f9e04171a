"""The no-allocation form of steps that share prefixes, on both sides of the work area's size: what fits
gives the shared call's bits, and what would not is read apart and gives those of the step without
groups, also from a captured graph."""

import ctypes

import pytest
import torch

from gpu_checks import say
from span_checks import SharedStep, close
from test_gpu_shared_prefix import Setup
from nanollvm_amd import Context, _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,fits", [(50, True), (110, False)])
def test_both_sides_of_the_work_area(new, fits):
    lib = N.load()
    s1 = torch.cuda.Stream()
    with torch.cuda.stream(s1), Context(0, stream=s1) as ctx:
        st = SharedStep([(24, 8192)], [(0, new)] * 24, 256, seed=41, decode=False)
        s = Setup(ctx, st, (32, 8, 128), seed=41)
        try:
            shared = s.check(ctx, f"shared, {new} tokens each")
            out = torch.full_like(shared, float("nan"))

            def call():
                return lib.nva_attention_forward_noalloc(
                    ctx.handle, s.arena.handle, ctypes.byref(s.attn._desc), s.q.data_ptr(),
                    s.k.data_ptr(), s.v.data_ptr(), s.q.shape[0], out.data_ptr())

            ctx.set_timing(True)
            ctx.reset_stats()
            assert call() == N.NVA_OK, lib.nva_last_error(ctx.handle)
            spans = ctx.kernel_stats("span_tiles")[0] + ctx.kernel_stats("span")[0]
            ctx.set_timing(False)
            say(f"{new} tokens each: {spans} launches of spans")
            assert (spans > 0) == fits
            first = out.clone()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s1):
                assert call() == N.NVA_OK, lib.nva_last_error(ctx.handle)
            for r in range(3):
                out.fill_(float("nan"))
                s1.synchronize()
                g.replay()
                s1.synchronize()
                assert torch.equal(out, first), f"replay {r}"
            if fits:
                assert torch.equal(first, shared)
            else:
                ctx.share_prefixes([])
                assert torch.equal(first, s.attn.forward(s.q, s.k, s.v, ctx))
                close(first, shared.double(), "apart against shared")
        finally:
            ctx.clear()
            s.arena.close()
