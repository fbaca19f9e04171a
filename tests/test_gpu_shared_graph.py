"""Captured steps that share prefixes where span tiles run beside the rows, on the second stream: replays
give the eager call's bits on the inputs then in place, in the no-allocation form and, on the buffers of
an eager call before, in the allocating one."""

import ctypes

import pytest
import torch

from gpu_checks import say
from span_checks import SharedStep
from test_gpu_shared_prefix import Setup
from nanollvm_amd import Context, _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("noalloc", [True, False])
@pytest.mark.parametrize("shape,rows,prefix", [((32, 8, 128), 64, 8192), ((8, 1, 512), 82, 8704)], ids=str)
def test_rows_beside_span_tiles(shape, rows, prefix, noalloc):
    lib = N.load()
    s1 = torch.cuda.Stream()
    with torch.cuda.stream(s1), Context(0, stream=s1) as ctx:
        st = SharedStep([(rows, prefix)], [(16 + 37 * i % 1400, 1) for i in range(rows)], 256, seed=51)
        s = Setup(ctx, st, shape, seed=51)
        try:
            want = s.check(ctx, f"eager {shape}")
            ctx.set_timing(True)
            ctx.reset_stats()
            s.attn.forward(s.q, s.k, s.v, ctx)
            assert ctx.kernel_stats("span_tiles")[0] == ctx.kernel_stats("decode")[0] == 1
            ctx.set_timing(False)
            out = torch.full_like(want, float("nan"))
            call = lib.nva_attention_forward_noalloc if noalloc else lib.nva_attention_forward

            def run():
                return call(ctx.handle, s.arena.handle, ctypes.byref(s.attn._desc), s.q.data_ptr(),
                            s.k.data_ptr(), s.v.data_ptr(), rows, out.data_ptr())

            assert run() == N.NVA_OK
            s1.synchronize()
            assert torch.equal(out, want)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s1):
                got = run()
            assert got == N.NVA_OK, lib.nva_last_error(ctx.handle)
            for r in range(4):
                if r >= 2:
                    for t in (s.q, s.k, s.v):
                        t.normal_()
                    want = s.attn.forward(s.q, s.k, s.v, ctx)
                out.fill_(float("nan"))
                junk = torch.randn(1 << 20, device="cuda").sum()
                s1.synchronize()
                g.replay()
                s1.synchronize()
                say(f"{shape} beside rows: replay {r} ({float(junk):.1f})")
                assert torch.equal(out, want), f"replay {r}"
        finally:
            ctx.clear()
            s.arena.close()
