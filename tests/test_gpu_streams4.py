"""The 4-bit calls and device steps on the stream that the context is switched to, and their entries among
the kernel statistics."""

import pytest
import torch

from checks4 import close, dev
from nanollvm_amd import BlockTables, Context, Linear4, quantize4
from test_gpu_attention4 import Case
from test_gpu_linear4 import data, want

pytestmark = pytest.mark.gpu


def busy(stream):
    """Work that a call on another stream would overtake."""
    with torch.cuda.stream(stream):
        x = torch.ones(4096, 4096, device="cuda")
        for _ in range(20):
            x = x @ x * 2.0 ** -12
    return x


def test_inputs_written_on_the_switched_stream():
    """Each call reads what earlier work on its own stream writes, and torch there reads its results."""
    case = Case([(70, 1), (3, 1), (200, 1)], 8, 2, 128, block=64, seed=1)
    x, w, b = data(40, 512, 48, True, 2)
    with Context(0) as ctx, case.arena(ctx) as arena, Linear4.from_weight(ctx, dev(w), dev(b)) as lin, \
            BlockTables(ctx, 4, 500, 64, 64, 64) as tables:
        ctx.sync()
        q, k, v, xs = dev(case.q), dev(case.k_new), dev(case.v_new), dev(x)
        fresh = torch.tensor([3, 0, 64, 1], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        for _ in range(3):
            s = torch.cuda.Stream()
            ctx.set_stream(s)
            with torch.cuda.stream(s):
                slow = busy(s)
                late = [torch.zeros_like(t) for t in (q, k, v, xs)]
                for t, value in zip(late, (q, k, v, xs)):
                    t.copy_(value + 0 * slow[0, 0])
                few = torch.zeros_like(fresh)
                few.copy_(torch.tensor([1, 0, 2, 0], device="cuda", dtype=torch.int32) + 0 * slow[0, 0].int())
                ctx.set(**case.step())
                ctx.bind_kv_cache(arena)
                out = case.layer().forward(*late[:3], ctx) + 0
                y = lin.forward(late[3], ctx) + 0
                codes, scales = (t + 0 for t in quantize4(late[3], ctx))
                ctx.extend(tables, few, 8, 4)
                lens = tables.lens + 0
            s.synchronize()
            close(out, case.want())
            close(y, want(x, w, b))
            again = quantize4(xs, ctx)
            ctx.sync()
            assert torch.equal(codes, again[0]) and torch.equal(scales, again[1])
            assert lens.tolist()[1] == lens.tolist()[3] == 0 and lens.tolist()[2] == 2 * lens.tolist()[0]
            ctx.clear()
        ctx.set_stream()


def test_statistics():
    case = Case([(70, 1), (3, 1), (5000, 1)], 8, 2, 128, block=64, seed=1)
    x, w, _ = data(100, 512, 48, False, 2)
    with Context(0) as ctx, case.arena(ctx) as arena, Linear4.from_weight(ctx, dev(w)) as lin, \
            BlockTables(ctx, 4, 500, 64, 64, 64) as tables:
        ctx.set_timing(True)
        ctx.reset_stats()
        ctx.set(**case.step())
        ctx.bind_kv_cache(arena)
        case.layer().forward(dev(case.q), dev(case.k_new), dev(case.v_new), ctx)
        arena.read_rows(0, dev(case.new_slots()))
        lin.forward(dev(x), ctx)
        quantize4(dev(x), ctx)
        ctx.extend(tables, torch.ones(4, dtype=torch.int32, device="cuda"), 8, 4)
        for name in ("store4", "attention4", "merge4", "read4", "linear4", "quantize4", "tables"):
            launches, ms = ctx.kernel_stats(name)
            assert launches == 1 and 0 < ms < 1000, name
        ctx.clear()
