"""Which launches a decode step over the 4-bit arena makes, by its window, over the stand-in HIP runtime of
host_hip4.cpp: ``python host_windows4.py <stand-in> <scenario>``."""

import ctypes
import sys

from host_side import N, Step, context, lib, ptr, i32, stub

STORE, ATTENTION, MERGE = 1, 1, 1


def launches(ctx, kv, step, window):
    p = step.aligned()
    desc = N.AttnDesc(step.hq, step.d, 0.1, step.hkv, window, 0, 1)
    before = stub.stub_launches()
    assert lib.nva_attention4_forward(ctx, kv, ctypes.byref(desc), p, p, p, step.tokens, p) == N.NVA_OK
    return stub.stub_launches() - before


def largest_windows():
    """Rows that are split are joined, whatever the window: one as large as its type holds is none."""
    for d in (64, 128, 256, 512):
        ctx = context()
        step = Step(5, 64, 90000, 1, heads=(4, 2, d))
        kv = ctypes.c_void_p()
        assert lib.nva_kv4_create(ctx, 1, step.num_blocks, step.block, step.hkv, ptr(i32([d])), None,
                                  ctypes.byref(kv)) == N.NVA_OK
        assert step.set(ctx) == N.NVA_OK
        for window in (0, 5000, 2 ** 30, 2 ** 31 - 33, 2 ** 31 - 32, 2 ** 31 - 31, 2 ** 31 - 30,
                       2 ** 31 - 2, 2 ** 31 - 1):
            assert launches(ctx, kv, step, window) == STORE + ATTENTION + MERGE, (d, window)
        # (Few keys a row are not split.)
        assert launches(ctx, kv, step, 33) == STORE + ATTENTION, d
        lib.nva_kv4_destroy(kv)
        lib.nva_ctx_destroy(ctx)


if __name__ == "__main__":
    globals()[sys.argv[2]]()
    print("ok", flush=True)
