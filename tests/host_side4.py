"""Scenarios of the 4-bit calls and of steps built on the device over the stand-in HIP runtime of
host_hip4.cpp, beside those of host_side.py: ``python host_side4.py <stand-in> <scenario>``."""

import ctypes
import sys

import numpy as np

from host_side import N, Step, context, failing, i32, lib, ptr, stub

stub.stub_set_capturing.argtypes = [ctypes.c_int]


def made(create, *args):
    """(status, handle) of a call whose last argument is where the handle goes."""
    h = ctypes.c_void_p()
    return create(*args, ctypes.byref(h)), h


def arena4(ctx, step, blocks=None, block=None, dims=None, allocate=None):
    dims = i32([step.d] if dims is None else dims)
    return made(lib.nva_kv4_create, ctx, len(dims), blocks or step.num_blocks, block or step.block,
                step.hkv, ptr(dims), None if allocate is None else
                ptr(np.asarray(allocate, np.uint8)))


def rope_desc(**change):
    return N.RopeDesc(*{**dict(head_size=128, rotary_dim=64, max_pos=4096, interleaved=1, base=1e4,
                               scaling=N.ROPE_SCALINGS["yarn"], factor=8.0, original_max_pos=512,
                               low=1.0, high=32.0, amplitude=0.0), **change}.values())


def rope4(ctx, **change):
    return made(lib.nva_rope_create_scaled, ctx, ctypes.byref(rope_desc(**change)))


def tables(ctx, seqs=4, tokens=1000, step_tokens=64, blocks=64, block=64, pages=None):
    return made(lib.nva_tables_create, ctx, seqs, tokens, step_tokens, blocks, block,
                None if pages is None else ptr(i32(pages)))


def attend4(ctx, kv, step, tokens=None, q=None, k=0, v=0, desc=None):
    p = step.aligned()
    return lib.nva_attention4_forward(ctx, kv, ctypes.byref(desc or step.desc), p if q is None else q,
                                      p if k == 0 else k, p if v == 0 else v,
                                      step.tokens if tokens is None else tokens, p)


def host_memory():
    """Nothing these entry points throw when host memory runs out leaves them."""
    for timing in (0, 1):
        for step in (Step(9, 512, 30, 1), Step(9, 512, 30, 5)):
            ctx = context()
            lib.nva_ctx_set_timing(ctx, timing)
            mode = f"{'decode' if step.decode else 'prefill'}, timing {timing}"
            p = step.aligned()
            for name, create, destroy in (
                    ("nva_kv4_create", lambda: arena4(ctx, step, dims=[step.d] * 3), lib.nva_kv4_destroy),
                    ("nva_rope_create_scaled", lambda: rope4(ctx), lib.nva_rope_destroy),
                    ("nva_tables_create", lambda: tables(ctx, pages=range(64)),
                     lib.nva_tables_destroy),
                    ("nva_linear4_create", lambda: made(lib.nva_linear4_create, ctx, p, p, 300, 64),
                     lib.nva_linear4_destroy)):
                held = []

                def call():
                    st, h = create()
                    if st == N.NVA_OK:
                        held.append(h)
                    else:
                        assert not h
                    return st

                def drop():
                    while held:
                        assert destroy(held.pop()) == N.NVA_OK

                assert failing(f"{name} ({mode})", call, drop) > 0
            kv, rope, t, lin = (x[1] for x in (
                arena4(ctx, step, blocks=max(64, step.num_blocks)), rope4(ctx), tables(ctx),
                made(lib.nva_linear4_create, ctx, p, p, 300, 64)))
            fresh = i32([1, 2, 0, 1])
            norm = ctypes.byref(N.RmsNormDesc(None, 1e-6, 0))

            def host_step():
                assert step.set(ctx) == N.NVA_OK

            def device_step():
                assert lib.nva_step_extend(ctx, t, None, ptr(fresh), 4, 8, 2) == N.NVA_OK

            for name, call, before in (
                    ("nva_attention4_forward", lambda: attend4(ctx, kv, step), host_step),
                    ("nva_attention4_forward (device step)", lambda: attend4(ctx, kv, step, 8),
                     device_step),
                    ("nva_norm_rope_attention4_forward", lambda: lib.nva_norm_rope_attention4_forward(
                        ctx, kv, rope, norm, norm, norm, ctypes.byref(step.desc), p, p, p, step.tokens,
                        None, None, p), host_step),
                    ("nva_qkv_norm_rope_attention4_forward",
                     lambda: lib.nva_qkv_norm_rope_attention4_forward(
                         ctx, kv, rope, None, None, None, ctypes.byref(step.desc), p, 8, None, None, p),
                     device_step),
                    ("nva_rope_forward (device step)", lambda: lib.nva_rope_forward(
                        ctx, rope, p, p, 8, step.hq, step.hkv, p, p), device_step),
                    ("nva_step_extend", lambda: lib.nva_step_extend(ctx, t, None, ptr(fresh), 4, 8, 2),
                     lambda: None),
                    ("nva_tables_status", lambda: lib.nva_tables_status(t, ptr(i32([0] * 3))),
                     lambda: None),
                    ("nva_quantize4", lambda: lib.nva_quantize4(ctx, p, 2, 64, p, p), lambda: None),
                    ("nva_kv4_write_rows", lambda: lib.nva_kv4_write_rows(kv, 0, p, p, p, 3),
                     lambda: None),
                    ("nva_kv4_read_rows", lambda: lib.nva_kv4_read_rows(kv, 0, p, p, p, 3),
                     lambda: None),
                    ("nva_linear4_forward", lambda: lib.nva_linear4_forward(ctx, lin, p, 300, None, p),
                     lambda: None)):
                before()
                failing(f"{name} ({mode})", call, before)
            # An error whose text finds no memory is still that error.
            stub.stub_fail_host_after(0)
            bad = lib.nva_step_extend(ctx, t, None, ptr(fresh), 5, 8, 2)
            stub.stub_fail_host_after(-1)
            assert bad == N.NVA_E_ARG
            for destroy, h in ((lib.nva_kv4_destroy, kv), (lib.nva_rope_destroy, rope),
                               (lib.nva_tables_destroy, t), (lib.nva_linear4_destroy, lin)):
                assert destroy(h) == N.NVA_OK
            assert lib.nva_ctx_destroy(ctx) == N.NVA_OK


def device_memory():
    """A call that finds no device memory says so, launches nothing over what it has and works again
    once there is some."""
    step = Step(9, 512, 30, 5)
    ctx = context()
    p = step.aligned()
    assert step.set(ctx) == N.NVA_OK
    for create, destroy in ((lambda: arena4(ctx, step, dims=[128, 64, 256]), lib.nva_kv4_destroy),
                            (lambda: rope4(ctx), lib.nva_rope_destroy),
                            (lambda: tables(ctx, pages=range(64)), lib.nva_tables_destroy),
                            (lambda: made(lib.nva_linear4_create, ctx, p, p, 300, 64),
                             lib.nva_linear4_destroy)):
        for allocations in range(10):
            before = stub.stub_launches()
            stub.stub_fail_device_after(allocations)
            st, h = create()
            stub.stub_fail_device_after(-1)
            if st == N.NVA_OK:
                break
            assert st == N.NVA_E_OOM and not h and stub.stub_launches() == before
        assert allocations > 0 and destroy(h) == N.NVA_OK
    kv, rope = arena4(ctx, step)[1], rope4(ctx)[1]
    lin = made(lib.nva_linear4_create, ctx, p, p, 300, 64)[1]
    for call, launched in ((lambda: attend4(ctx, kv, step), 0),
                           (lambda: lib.nva_linear4_forward(ctx, lin, p, 300, None, p), 0),
                           (lambda: lib.nva_norm_rope_attention4_forward(
                               ctx, kv, rope, None, None, None, ctypes.byref(step.desc), p, p, p,
                               step.tokens, None, None, p), 0)):
        stub.stub_fail_device_after(0)
        before = stub.stub_launches()
        assert call() == N.NVA_E_OOM
        assert stub.stub_launches() == before + launched
        stub.stub_fail_device_after(-1)
        assert call() == N.NVA_OK
    for destroy, h in ((lib.nva_kv4_destroy, kv), (lib.nva_rope_destroy, rope),
                       (lib.nva_linear4_destroy, lin)):
        destroy(h)
    lib.nva_ctx_destroy(ctx)


def refused(want, call):
    before = stub.stub_launches()
    got = call()
    assert got == want, (got, want)
    assert stub.stub_launches() == before


def refusals():
    """Arguments that the kernels could not bear are refused before anything is launched."""
    E, U = N.NVA_E_ARG, N.NVA_E_UNSUPPORTED
    ctx, other = context(), context()
    step = Step(9, 512, 30, 1)
    p = step.aligned()
    for change in (dict(max_pos=0), dict(head_size=127), dict(rotary_dim=0), dict(rotary_dim=130),
                   dict(rotary_dim=33), dict(base=1.0), dict(base=np.inf), dict(base=np.nan),
                   dict(scaling=5), dict(scaling=-1), dict(factor=0.5), dict(factor=np.nan),
                   dict(factor=np.inf), dict(original_max_pos=0), dict(low=0.0), dict(low=32.0),
                   dict(high=np.inf), dict(high=np.nan), dict(amplitude=-1.0),
                   dict(amplitude=np.inf)):
        refused(E, lambda: rope4(ctx, **change)[0])
    for want, change in ((E, dict(seqs=0)), (U, dict(seqs=4001)), (E, dict(tokens=0)),
                         (U, dict(tokens=2 ** 31 - 1)), (E, dict(step_tokens=-1)),
                         (E, dict(blocks=0)), (E, dict(block=0)), (E, dict(pages=[1] * 64)),
                         (E, dict(pages=range(-1, 63))), (U, dict(blocks=2 ** 26, block=32)),
                         (U, dict(pages=[*range(63), 2 ** 26]))):
        refused(want, lambda: tables(ctx, **change)[0])
    for want, change in ((E, dict(dims=[])), (U, dict(block=16)), (U, dict(block=48)),
                         (U, dict(dims=[96])), (U, dict(dims=[1024])), (E, dict(blocks=-1))):
        refused(want, lambda: arena4(ctx, step, **change)[0])
    kv = arena4(ctx, step, dims=[step.d, 64, step.d], allocate=[1, 1, 0])[1]
    three = i32([0, 1, 2])
    for want, args in ((N.NVA_E_LAYER, (-1, p, p, p, 3)), (N.NVA_E_LAYER, (3, p, p, p, 3)),
                       (E, (2, p, p, p, 3)), (E, (0, None, p, p, 3)), (E, (0, ptr(three), p + 4, p, 3)),
                       (E, (0, p, p, p, -1)), (U, (0, p, p, p, 2 ** 30))):
        refused(want, lambda: lib.nva_kv4_write_rows(kv, *args))
        refused(want, lambda: lib.nva_kv4_read_rows(kv, *args))
    refused(E, lambda: lib.nva_kv4_write_rows(kv, 0, p, None, p, 3))
    refused(N.NVA_OK, lambda: lib.nva_kv4_write_rows(kv, 0, None, None, None, 0))
    for want, args in ((E, (p, -1, 64, p, p)), (E, (p, 1, 0, p, p)), (U, (p, 1, 48, p, p)),
                       (E, (None, 1, 64, p, p)), (E, (p + 4, 1, 64, p, p)), (E, (p, 1, 64, p + 2, p)),
                       (U, (p, 2 ** 42, 64, p, p)), (N.NVA_OK, (None, 0, 64, None, None))):
        refused(want, lambda: lib.nva_quantize4(ctx, *args))
    for want, args in ((E, (p, p, 0, 64)), (E, (p, p, 8, 0)), (U, (p, p, 8, 48)),
                       (U, (p, p, 8, 2 ** 22)), (E, (None, p, 8, 64)), (E, (p, None, 8, 64))):
        refused(want, lambda: made(lib.nva_linear4_create, ctx, *args)[0])
    lin = made(lib.nva_linear4_create, ctx, p, p, 8, 64)[1]
    for want, args in ((E, (None, p, 3, None, p)), (E, (lin, p, -1, None, p)),
                       (E, (lin, None, 3, None, p)), (E, (lin, p, 3, None, None)),
                       (E, (lin, p + 4, 3, None, p)), (U, (lin, p, 2 ** 31 - 1, None, p)),
                       (N.NVA_OK, (lin, None, 0, None, None))):
        refused(want, lambda: lib.nva_linear4_forward(ctx, *args))
    # A weight belongs to the device, not to the context that laid it out.
    assert lib.nva_linear4_forward(other, lin, p, 3, None, p) == N.NVA_OK

    # Steps.
    refused(N.NVA_E_NO_STEP, lambda: attend4(ctx, kv, step))
    refused(N.NVA_E_NO_ARENA, lambda: attend4(ctx, None, step))
    assert step.set(ctx) == step.set(other) == N.NVA_OK
    refused(E, lambda: attend4(other, kv, step))
    assert attend4(ctx, kv, step) == N.NVA_OK
    for change in (dict(q=p + 4), dict(k=p + 4), dict(k=None), dict(v=None), dict(tokens=10)):
        refused(E, lambda: attend4(ctx, kv, step, **change))
    for want, d in ((N.NVA_E_LAYER, (step.hq, step.d, 0.1, step.hkv, 0, 3, 1)),
                    (E, (step.hq, step.d, 0.1, step.hkv, 0, 1, 1)),
                    (E, (step.hq, step.d, 0.1, step.hkv, 0, 2, 1)),
                    (E, (step.hq, step.d, 0.1, 4, 0, 0, 1))):
        refused(want, lambda: attend4(ctx, kv, step, desc=N.AttnDesc(*d)))
    refused(N.NVA_OK, lambda: attend4(ctx, kv, step, tokens=0))
    for new in (1, 5):  # blocks that do not exist, in decode and prefill
        sound = Step(9, 512, 30, new)
        lib.nva_kv4_destroy(kv)
        kv = arena4(ctx, sound)[1]
        assert sound.set(ctx) == attend4(ctx, kv, sound) == N.NVA_OK
        for bad in (-1, -2 ** 31, sound.num_blocks, 2 ** 31 - 1):
            for row, col in ((0, 0), (3, -1), (8, 2)):
                broken = Step(9, 512, 30, new)
                used = -(-broken.lens[row] // broken.block)
                broken.table[row, used - 1 if col < 0 else col] = bad
                assert broken.set(ctx) == N.NVA_OK
                refused(E, lambda: attend4(ctx, kv, broken))
        behind = Step(9, 512, 30, new)  # behind the last key: not looked at
        wide = np.full((9, behind.table.shape[1] + 1), 2 ** 31 - 1, np.int32)
        wide[:, :-1] = behind.table
        behind.table = wide
        assert behind.set(ctx) == attend4(ctx, kv, behind) == N.NVA_OK
        long = Step(9, 512, 30, new)  # more keys than the table's blocks
        long.context_lens[4] += 64 * 40
        long.cu_k[5:] += 64 * 40
        assert long.set(ctx) == N.NVA_OK
        refused(E, lambda: attend4(ctx, kv, long))
        outside = Step(9, 512, 30, new)
        outside.slots[3] = outside.num_blocks * outside.block
        assert outside.set(ctx) == N.NVA_OK
        refused(E, lambda: attend4(ctx, kv, outside))
    for h, destroy in ((kv, lib.nva_kv4_destroy), (lin, lib.nva_linear4_destroy)):
        destroy(h)
    lib.nva_ctx_destroy(ctx)
    lib.nva_ctx_destroy(other)


def device_steps():
    """Which calls a step of nva_step_extend serves, and what ends it."""
    E = N.NVA_E_ARG
    ctx, other = context(), context()
    step = Step(9, 512, 30, 1)
    p = step.aligned()
    kv = arena4(ctx, step, blocks=64)[1]
    t = tables(ctx)[1]
    fresh = i32([1, 2, 0, 1])

    def extend(c=ctx, tab=t, keep=None, new=None, seqs=4, tokens=8, most=2):
        return lib.nva_step_extend(c, tab, keep, ptr(fresh) if new is None else new, seqs, tokens, most)

    for change in (dict(c=other), dict(tab=None), dict(seqs=-1), dict(seqs=5), dict(tokens=-1),
                   dict(tokens=65), dict(most=-1)):
        refused(E, lambda: extend(**change))
    refused(E, lambda: lib.nva_step_extend(ctx, t, None, None, 4, 8, 2))
    refused(N.NVA_E_NO_STEP, lambda: attend4(ctx, kv, step, 8))
    assert extend() == attend4(ctx, kv, step, 8) == N.NVA_OK
    refused(E, lambda: attend4(ctx, kv, step, 7))
    refused(N.NVA_OK, lambda: attend4(ctx, kv, step, 0))
    st, plain = step.arena(ctx)
    assert st == N.NVA_OK
    refused(N.NVA_E_NO_STEP, lambda: step.attend(ctx, plain))
    refused(N.NVA_E_NO_STEP, lambda: step.attend(ctx, plain, True))
    refused(N.NVA_E_NO_STEP, lambda: step.attend_encoder(ctx))
    # Positions that the table of angles does not hold.
    for rows, want in ((1000, N.NVA_OK), (999, None)):
        rope = rope4(ctx, max_pos=rows)[1]
        call = lambda: lib.nva_rope_forward(ctx, rope, p, p, 8, step.hq, step.hkv, p, p)  # noqa: E731
        if want is None:
            before = stub.stub_launches()
            assert call() != N.NVA_OK and stub.stub_launches() == before
        else:
            assert call() == want
        lib.nva_rope_destroy(rope)
    # Arenas of other blocks.
    for blocks, block in ((63, 64), (64, 128)):
        small = arena4(ctx, step, blocks=blocks, block=block)[1]
        refused(E, lambda: attend4(ctx, small, step, 8))
        lib.nva_kv4_destroy(small)
    # A refused extend leaves the step; another step, a clear and the tables' end take it.
    refused(E, lambda: extend(seqs=5))
    assert attend4(ctx, kv, step, 8) == N.NVA_OK
    lib.nva_step_clear(ctx)
    refused(N.NVA_E_NO_STEP, lambda: attend4(ctx, kv, step, 8))
    host = Step(3, 128, 10, 1)
    assert extend() == host.set(ctx) == attend4(ctx, kv, host) == N.NVA_OK
    refused(E, lambda: attend4(ctx, kv, host, 8))
    assert extend() == attend4(ctx, kv, step, 8) == N.NVA_OK
    assert lib.nva_tables_destroy(t) == N.NVA_OK
    refused(N.NVA_E_NO_STEP, lambda: attend4(ctx, kv, step, 8))
    lib.nva_kv_destroy(plain)
    lib.nva_kv4_destroy(kv)
    lib.nva_ctx_destroy(ctx)
    lib.nva_ctx_destroy(other)


def capture():
    """Under capture nothing is allocated: what does not fit is refused, what fits is launched, and the
    buffers that a graph may hold outlive their growth."""
    E = N.NVA_E_ARG
    ctx = context()
    step = Step(9, 512, 30, 1)
    p = step.aligned()
    kv, rope, t = arena4(ctx, step, blocks=64)[1], rope4(ctx)[1], tables(ctx)[1]
    lin = made(lib.nva_linear4_create, ctx, p, p, 300, 1024)[1]
    fresh = i32([1, 1, 1, 1])

    def extend(tokens):
        assert lib.nva_step_extend(ctx, t, None, ptr(fresh), 4, tokens, 1) == N.NVA_OK

    def bytes_held():
        n = ctypes.c_int64()
        ms = ctypes.c_double()
        assert lib.nva_ctx_kernel_stats(ctx, b"device_bytes", ctypes.byref(n),
                                        ctypes.byref(ms)) == N.NVA_OK
        return n.value

    calls = {
        "attention": lambda rows: attend4(ctx, kv, step, rows),
        "fused": lambda rows: lib.nva_norm_rope_attention4_forward(
            ctx, kv, rope, None, None, None, ctypes.byref(step.desc), p, p, p, rows, None, None, p),
        "packed": lambda rows: lib.nva_qkv_norm_rope_attention4_forward(
            ctx, kv, rope, None, None, None, ctypes.byref(step.desc), p, rows, None, None, p),
        "linear": lambda rows: lib.nva_linear4_forward(ctx, lin, p, 16 * rows, None, p)}
    for name, call in calls.items():
        stub.stub_set_capturing(1)
        extend(8)
        assert call(8) == E, name
        stub.stub_set_capturing(0)
        extend(8)
        assert call(8) == N.NVA_OK, name
        stub.stub_set_capturing(1)
        stub.stub_fail_device_after(0)  # (nothing is allocated)
        extend(8)
        assert call(8) == N.NVA_OK, name
        stub.stub_fail_device_after(-1)
        extend(60)
        assert call(60) == E, name
        assert lib.nva_tables_status(t, ptr(i32([0] * 3))) == E
        stub.stub_set_capturing(0)
        held = bytes_held()
        extend(60)
        assert call(60) == N.NVA_OK, name
        assert bytes_held() > held, name
        stub.stub_set_capturing(1)
        extend(60)
        assert call(60) == N.NVA_OK, name
        stub.stub_set_capturing(0)
        for h in (kv, rope, t, lin):
            assert h
        # The next call begins with a context of its own.
        for destroy, h in ((lib.nva_kv4_destroy, kv), (lib.nva_rope_destroy, rope),
                           (lib.nva_tables_destroy, t), (lib.nva_linear4_destroy, lin)):
            destroy(h)
        lib.nva_ctx_destroy(ctx)
        ctx = context()
        kv, rope, t = arena4(ctx, step, blocks=64)[1], rope4(ctx)[1], tables(ctx)[1]
        lin = made(lib.nva_linear4_create, ctx, p, p, 300, 1024)[1]
    # A step of the host is not for capture: its metadata would not be the replay's.
    assert step.set(ctx) == attend4(ctx, kv, step) == N.NVA_OK
    stub.stub_set_capturing(1)
    refused(E, lambda: attend4(ctx, kv, step))
    # One to 16 rows of a projection need no work area.
    assert lib.nva_linear4_forward(ctx, lin, p, 16, None, p) == N.NVA_OK
    stub.stub_set_capturing(0)


if __name__ == "__main__":
    globals()[sys.argv[2]]()
    print("ok", flush=True)
