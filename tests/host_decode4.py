"""Which launches a decode step over the 4-bit arena makes and which steps it refuses, over the stand-in HIP runtime of
host_hip4.cpp: ``python host_decode4.py <stand-in> <scenario>``."""

import ctypes
import sys

from host_side import N, Step, context, lib, ptr, i32, stub

stub.stub_set_capturing.argtypes = [ctypes.c_int]
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


def short_rows():
    """Rows of a decode step up to a length are not split, by how many of them there are."""
    for rows, heads, limit in ((1, (32, 8, 128), 32), (1, (4, 1, 64), 32), (3, (32, 8, 128), 32),
                               (5, (32, 8, 128), 48), (32, (4, 1, 64), 48), (60, (40, 8, 128), 48),
                               (5, (4, 1, 256), 28), (31, (4, 1, 256), 28), (32, (4, 1, 256), 48),
                               (96, (4, 1, 256), 48), (512, (4, 1, 256), 48), (513, (4, 1, 256), 0),
                               (5, (8, 1, 512), 8), (100, (8, 1, 512), 12),
                               (16, (20, 1, 512), 12), (15, (20, 1, 512), 8)):  # two column tiles a row
        ctx = context()
        for tiles, extra in ((1, 0), (limit - 1, 1), (limit, 0), (limit, 1), (limit + 1, 0)):
            keys = 32 * tiles + extra
            if keys < 1:
                continue
            step = Step(rows, keys - 1, 0, 1, heads=heads)
            kv = ctypes.c_void_p()
            assert lib.nva_kv4_create(ctx, 1, step.num_blocks, step.block, step.hkv, ptr(i32([step.d])),
                                      None, ctypes.byref(kv)) == N.NVA_OK
            assert step.set(ctx) == N.NVA_OK
            want = STORE + ATTENTION + (0 if keys <= 32 * limit else MERGE)
            assert launches(ctx, kv, step, 0) == want, (rows, heads, keys)
            lib.nva_kv4_destroy(kv)
        lib.nva_ctx_destroy(ctx)


def fewer_rows():
    """Calls of fewer rows than the step's are checked for their rows, and each row for every arena."""
    def arena(blocks, block):
        kv = ctypes.c_void_p()
        assert lib.nva_kv4_create(ctx, 1, blocks, block, step.hkv, ptr(i32([step.d])), None,
                                  ctypes.byref(kv)) == N.NVA_OK
        return kv

    def attend(kv, rows):
        p = step.aligned()
        before = stub.stub_launches()
        got = lib.nva_attention4_forward(ctx, kv, ctypes.byref(desc), p, p, p, rows, p)
        assert (got == N.NVA_OK) == (stub.stub_launches() > before)
        return got

    ctx = context()
    step = Step(9, 512, 30, 1)
    desc = N.AttnDesc(step.hq, step.d, 0.1, step.hkv, 0, 0, 0)
    kv, wide, small = (arena(*a) for a in ((step.num_blocks, 64), (step.num_blocks, 128), (8, 64)))
    step.table[6, 3] = step.num_blocks
    assert step.set(ctx) == N.NVA_OK
    for _ in range(2):
        for rows, want in ((5, N.NVA_OK), (9, N.NVA_E_ARG), (6, N.NVA_OK), (7, N.NVA_E_ARG), (1, N.NVA_OK)):
            assert attend(kv, rows) == want, rows
        assert attend(wide, 6) == N.NVA_OK and attend(small, 1) == N.NVA_E_ARG
        assert attend(wide, 7) == N.NVA_E_ARG
    step.table[6, 3] = 3  # another step
    step.table[0, 0] = -1
    assert step.set(ctx) == N.NVA_OK
    assert attend(kv, 1) == N.NVA_E_ARG
    step.table[0, 0] = 0
    assert step.set(ctx) == attend(kv, 1) == attend(kv, 9) == attend(kv, 4) == N.NVA_OK
    for h in (kv, wide, small):
        lib.nva_kv4_destroy(h)
    lib.nva_ctx_destroy(ctx)


def refused_before_anything():
    """The fused calls refuse what the attention behind them would, before they rotate (whose outputs may be
    their inputs)."""
    ctx = context()
    for new in (1, 5):
        step = Step(9, 512, 30, new)
        p = step.aligned()
        kv, rope = ctypes.c_void_p(), ctypes.c_void_p()
        assert lib.nva_kv4_create(ctx, 1, step.num_blocks, step.block, step.hkv, ptr(i32([step.d])), None,
                                  ctypes.byref(kv)) == N.NVA_OK
        assert lib.nva_rope_create_theta(ctx, step.d, step.d, 4096, ctypes.c_float(1e4),
                                         ctypes.byref(rope)) == N.NVA_OK
        desc = ctypes.byref(step.desc)
        calls = (lambda: lib.nva_norm_rope_attention4_forward(ctx, kv, rope, None, None, None, desc, p, p, p,
                                                              step.tokens, p, p, p),
                 lambda: lib.nva_qkv_norm_rope_attention4_forward(ctx, kv, rope, None, None, None, desc, p,
                                                                  step.tokens, None, None, p),
                 lambda: lib.nva_attention4_forward(ctx, kv, desc, p, p, p, step.tokens, p))

        def refused():
            for call in calls:
                before = stub.stub_launches()
                assert call() == N.NVA_E_ARG and stub.stub_launches() == before

        assert step.set(ctx) == N.NVA_OK
        for call in calls:
            assert call() == N.NVA_OK
        stub.stub_set_capturing(1)  # a step of the host is not for capture
        refused()
        stub.stub_set_capturing(0)
        step.slots[3] = step.num_blocks * step.block  # a slot outside the arena
        assert step.set(ctx) == N.NVA_OK
        refused()
        step.desc.write_kv = 0  # (which a call that does not store does not look at)
        for call in calls:
            assert call() == N.NVA_OK
        step.slots[3] = step.table[3, 0] = step.num_blocks
        assert step.set(ctx) == N.NVA_OK
        refused()
        lib.nva_kv4_destroy(kv)
        lib.nva_rope_destroy(rope)
    lib.nva_ctx_destroy(ctx)


def largest_weights():
    """Projections whose launches would pass 2^32 threads are refused before anything is allocated."""
    ctx = context()
    p = Step(1, 64, 0, 1).aligned()
    for out, inner in ((2 ** 26 - 15, 32), (2 ** 31 - 1, 32), (2 ** 31 - 1, 2 ** 22 - 32), (2 ** 25, 4096),
                       (2 ** 18 * 16, 128 * 256), (2 ** 18 * 16 - 15, 128 * 255 + 32)):
        h = ctypes.c_void_p()
        before = stub.stub_launches()
        stub.stub_fail_device_after(0)  # (an allocation would be NVA_E_OOM)
        got = lib.nva_linear4_create(ctx, p, p, out, inner, ctypes.byref(h))
        stub.stub_fail_device_after(-1)
        assert got == N.NVA_E_UNSUPPORTED and not h and stub.stub_launches() == before, (out, inner)
    for out, inner in ((2 ** 26 - 16, 32), (2 ** 22 * 16 - 16, 128 * 15), (2 ** 18 * 16, 128 * 255)):
        h = ctypes.c_void_p()
        stub.stub_fail_device_after(0)
        assert lib.nva_linear4_create(ctx, p, p, out, inner, ctypes.byref(h)) == N.NVA_E_OOM, (out, inner)
        stub.stub_fail_device_after(-1)
    lib.nva_ctx_destroy(ctx)


if __name__ == "__main__":
    globals()[sys.argv[2]]()
    print("ok", flush=True)
