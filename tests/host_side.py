"""Runs one scenario of the library's host side over the stand-in HIP runtime of host_hip.cpp:
``python host_side.py <stand-in> <scenario>``.  A process of its own, without torch, because the
stand-in has to be loaded before any real HIP runtime is; prints "ok" at the end."""

import ctypes
import importlib.util
import os
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))


def load(stand_in):
    stub = ctypes.CDLL(stand_in, mode=ctypes.RTLD_GLOBAL)
    for f in ("stub_fail_host_after", "stub_fail_device_after"):
        getattr(stub, f).argtypes = [ctypes.c_long]
    for f in ("stub_host_left", "stub_device_left", "stub_launches"):
        getattr(stub, f).restype = ctypes.c_long
    path = os.path.join(os.path.dirname(HERE), "nano-vllm-java_amd", "nanollvm_amd", "_native.py")
    spec = importlib.util.spec_from_file_location("native", path)
    native = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(native)
    return stub, native, native.load()


stub, N, lib = load(sys.argv[1])


def i32(x):
    return np.ascontiguousarray(x, dtype=np.int32)


def ptr(a):
    return None if a is None else a.ctypes.data


class Step:
    """A step over pages: rows of prefix + own + new tokens, the prefix in pages they share."""

    def __init__(self, rows, prefix, own, new, block=64, heads=(16, 8, 128)):
        self.block, (self.hq, self.hkv, self.d) = block, heads
        self.decode = new == 1
        self.lens = [prefix + own * (i % 7) + new for i in range(rows)]
        head = list(range(prefix // block))
        at, tables = len(head), []
        for n in self.lens:
            own_pages = -(-n // block) - len(head)
            tables.append(head + list(range(at, at + own_pages)))
            at += own_pages
        self.num_blocks = at
        self.table = np.full((rows, max(len(t) for t in tables)), -1, np.int32)
        for i, t in enumerate(tables):
            self.table[i, :len(t)] = t
        self.slots = i32([self.table[i, j // block] * block + j % block
                          for i, n in enumerate(self.lens) for j in range(n - new, n)])
        self.tokens = rows * new
        self.cached = i32([n - new for n in self.lens])
        self.cu_q = i32(np.arange(rows + 1) * new)
        self.cu_k = i32(np.concatenate([[0], np.cumsum(self.lens)]))
        self.context_lens = i32(self.lens)
        self.pos = np.concatenate([np.arange(n - new, n) for n in self.lens]).astype(np.float32)
        self.ids = i32(np.repeat(np.arange(rows), new))
        self.groups = (N.PrefixGroup * 1)(N.PrefixGroup(0, rows, prefix))
        self.q = np.zeros(4 * (1 + self.tokens * self.hq * self.d), np.float32)
        self.desc = N.AttnDesc(self.hq, self.d, 0.1, self.hkv, 0, 0, 1)
        self.cross = N.AttnDesc(self.hq, self.d, 0.1, self.hkv, 0, 0, 0)
        self.enc_start, self.enc_len = i32(np.zeros(rows)), i32(np.full(rows, 50))

    def aligned(self):
        p = ptr(self.q)
        return (p + 15) // 16 * 16

    def set(self, ctx):
        return lib.nva_step_set(ctx, int(not self.decode), None if self.decode else ptr(self.cu_q),
                                None if self.decode else ptr(self.cu_k), len(self.lens), 0, 0,
                                ptr(self.slots), len(self.slots),
                                ptr(self.context_lens) if self.decode else None, ptr(self.table),
                                self.table.shape[1], ptr(self.ids), ptr(self.pos), self.tokens)

    def share(self, ctx):
        return lib.nva_step_share_prefixes(ctx, self.groups, 1)

    def encode(self, ctx):
        return lib.nva_step_set_encoder(ctx, ptr(self.enc_start), ptr(self.enc_len), len(self.lens))

    def arena(self, ctx, layers=1):
        kv = ctypes.c_void_p()
        dims = i32([self.d] * layers)
        st = lib.nva_kv_create(ctx, layers, self.num_blocks, self.block, self.hkv, ptr(dims), None,
                               ctypes.byref(kv))
        return st, kv

    def attend(self, ctx, kv, noalloc=False):
        p = self.aligned()
        f = lib.nva_attention_forward_noalloc if noalloc else lib.nva_attention_forward
        return f(ctx, kv, ctypes.byref(self.desc), p, p, p, self.tokens, p)

    def attend_encoder(self, ctx, noalloc=False):
        p = self.aligned()
        f = (lib.nva_cross_attention_forward_noalloc if noalloc else
             lib.nva_cross_attention_forward)
        return f(ctx, ctypes.byref(self.cross), p, p, p, 2000, self.hkv * self.d, self.tokens, p)


def create():
    ctx = ctypes.c_void_p()
    st = lib.nva_ctx_create(0, ctypes.byref(ctx))
    return st, ctx


def context():
    st, ctx = create()
    assert st == N.NVA_OK
    return ctx


def failing(name, call, after=None):
    """Every host allocation that `call` makes, and all behind it, fails in turn: NVA_E_OOM, and the
    same call then succeeds.  `after` undoes a success before the next turn."""
    turns = 0
    while True:
        stub.stub_fail_host_after(turns)
        st = call()
        left = stub.stub_host_left()
        stub.stub_fail_host_after(-1)
        if st == N.NVA_OK and left > 0 or turns > 500:
            break
        # (A timing that finds no memory is dropped and the call goes on.)
        assert st in (N.NVA_E_OOM, N.NVA_OK), (name, turns, st)
        assert st == N.NVA_E_OOM or left == 0, (name, turns, st)
        if after and st == N.NVA_OK:
            after()
        st = call()
        assert st == N.NVA_OK, (name, turns, st)
        if after:
            after()
        turns += 1
    assert turns < 500, name
    if after:
        after()
    print(f"{name}: {turns} allocations", flush=True)
    return turns


def host_memory():
    """Nothing an entry point throws when host memory runs out leaves it."""
    made = []

    def new_context():
        st, ctx = create()
        if st == N.NVA_OK:
            made.append(ctx)
        return st

    def drop():
        while made:
            lib.nva_ctx_destroy(made.pop())

    assert failing("nva_ctx_create", new_context, drop) > 0
    pages = [i32(range(8 * i, 8 * i + 8)) for i in range(3)]
    seqs = (N.Seq * 3)(*(N.Seq(i, 100 + i, 64, 36 + i, ptr(t), 8) for i, t in enumerate(pages)))
    for timing in (0, 1):
        for st in (Step(9, 512, 30, 1), Step(9, 512, 30, 5)):
            ctx = context()
            lib.nva_ctx_set_timing(ctx, timing)
            mode = f"{'decode' if st.decode else 'prefill'}, timing {timing}"
            kvs = []

            def arena():
                s, kv = st.arena(ctx, 3)
                if s == N.NVA_OK:
                    kvs.append(kv)
                return s

            def drop_arena():
                while kvs:
                    lib.nva_kv_destroy(kvs.pop())

            assert failing(f"nva_kv_create ({mode})", arena, drop_arena) > 0
            arena()
            ropes = []

            def rope():
                r = ctypes.c_void_p()
                s = lib.nva_rope_create_theta(ctx, st.d, st.d, 4096, 1e6, ctypes.byref(r))
                if s == N.NVA_OK:
                    ropes.append(r)
                return s

            def drop_rope():
                while ropes:
                    lib.nva_rope_destroy(ropes.pop())

            assert failing(f"nva_rope_create_theta ({mode})", rope, drop_rope) > 0
            rope()
            bigger = [Step(9 + i, 512, 30, 1 if st.decode else 5) for i in range(60)]
            assert failing(f"nva_step_set ({mode})", lambda: bigger.pop(0).set(ctx)) > 0
            prepare = lib.nva_step_prepare_decode if st.decode else lib.nva_step_prepare_prefill
            assert failing(f"nva_step_prepare ({mode})", lambda: prepare(ctx, seqs, 3, 64)) > 0
            meta = N.StepMetaOut()
            build = (lib.nva_build_decode_metadata if st.decode else
                     lib.nva_build_prefill_metadata)
            assert failing(f"nva_build_metadata ({mode})",
                           lambda: build(seqs, 3, 64, ctypes.byref(meta))) > 0
            found, count = (N.PrefixGroup * 9)(), ctypes.c_int()
            assert failing(f"nva_find_shared_prefixes ({mode})",
                           lambda: lib.nva_find_shared_prefixes(
                               ptr(st.table), 9, st.table.shape[1], ptr(st.cached), st.block, found,
                               ctypes.byref(count))) > 0
            assert count.value == 1
            assert st.set(ctx) == N.NVA_OK
            positions = [np.arange(i, i + st.tokens + i).astype(np.float32) for i in range(1, 40)]
            def move():
                p = positions.pop(0)
                return lib.nva_step_positions(ctx, ptr(p), len(p))
            assert failing(f"nva_step_positions ({mode})", move) > 0
            assert st.set(ctx) == N.NVA_OK
            failing(f"nva_step_share_prefixes ({mode})", lambda: st.share(ctx))
            failing(f"nva_step_set_encoder ({mode})", lambda: st.encode(ctx))
            p = st.aligned()
            for name, call in {
                "nva_attention_forward": lambda: st.attend(ctx, kvs[0]),
                "nva_attention_forward_noalloc": lambda: st.attend(ctx, kvs[0], True),
                "nva_cross_attention_forward": lambda: st.attend_encoder(ctx),
                "nva_cross_attention_forward_noalloc": lambda: st.attend_encoder(ctx, True),
                "nva_rope_forward": lambda: lib.nva_rope_forward(
                    ctx, ropes[0], p, p, st.tokens, st.hq, st.hkv, p, p),
                "nva_rope_attention_forward": lambda: lib.nva_rope_attention_forward(
                    ctx, kvs[0], ropes[0], ctypes.byref(st.desc), p, p, p, st.tokens, None, None,
                    p),
                "nva_linear_forward": lambda: lib.nva_linear_forward(ctx, p, 300, 64, p, 300, None,
                                                                     p),
                "nva_rms_norm_forward": lambda: lib.nva_rms_norm_forward(
                    ctx, ctypes.byref(N.RmsNormDesc(None, 1e-6, 0)), p, 4, 128, p),
                "nva_ctx_kernel_stats": lambda: lib.nva_ctx_kernel_stats(
                    ctx, b"a name that no kernel has, of many letters", None, None),
            }.items():
                def fresh():  # plans are built again
                    assert st.set(ctx) == st.share(ctx) == st.encode(ctx) == N.NVA_OK
                fresh()
                failing(f"{name} ({mode})", call, fresh)
            # An error whose text finds no memory is still that error.
            stub.stub_fail_host_after(0)
            bad = lib.nva_step_share_prefixes(ctx, (N.PrefixGroup * 1)(N.PrefixGroup(-1, 2, 3)), 1)
            stub.stub_fail_host_after(-1)
            assert bad == N.NVA_E_ARG
            drop_rope()
            drop_arena()
            stub.stub_fail_host_after(0)
            assert lib.nva_ctx_reset_stats(ctx) == N.NVA_OK
            assert lib.nva_ctx_destroy(ctx) == N.NVA_OK
            stub.stub_fail_host_after(-1)


def device_memory():
    """A step or positions that find no device (or pinned) memory leave no step behind: nothing is
    launched over the buffers of the one before, until a step is set whole."""
    small, big = (Step(*a, 1, heads=(4, 2, 64)) for a in ((3, 128, 10), (60, 1024, 100)))
    for what in ("step", "positions"):
        failed = 0
        for n in range(6):
            ctx = context()
            st, kv = big.arena(ctx)
            assert st == N.NVA_OK
            rope = ctypes.c_void_p()
            assert lib.nva_rope_create_theta(ctx, 64, 64, 4096, 1e6, ctypes.byref(rope)) == N.NVA_OK
            assert small.set(ctx) == small.attend(ctx, kv) == N.NVA_OK
            many = np.arange(4000, dtype=np.float32)
            stub.stub_fail_device_after(n)
            st = (big.set(ctx) if what == "step" else
                  lib.nva_step_positions(ctx, ptr(many), len(many)))
            stub.stub_fail_device_after(-1)
            if st != N.NVA_OK:
                failed += 1
                assert st == N.NVA_E_OOM, (what, n, st)
                before, p = stub.stub_launches(), big.aligned()
                got = [big.attend(ctx, kv), big.attend(ctx, kv, True), big.attend_encoder(ctx),
                       big.share(ctx), big.encode(ctx),
                       lib.nva_rope_forward(ctx, rope, p, p, 3, 4, 2, p, p),
                       lib.nva_step_positions(ctx, ptr(many), 3)]
                assert got == [N.NVA_E_NO_STEP] * len(got), (what, n, got)
                assert stub.stub_launches() == before, (what, n)
            assert big.set(ctx) == big.attend(ctx, kv) == N.NVA_OK
            lib.nva_rope_destroy(rope)
            lib.nva_kv_destroy(kv)
            lib.nva_ctx_destroy(ctx)
        assert failed >= 2, (what, failed)
    # A call that finds none can be made again.
    for noalloc in (False, True):
        for call in ("attend", "attend_encoder"):
            for n in range(8):
                ctx = context()
                st, kv = big.arena(ctx)
                assert big.set(ctx) == big.share(ctx) == big.encode(ctx) == N.NVA_OK
                args = (kv,) if call == "attend" else ()
                stub.stub_fail_device_after(n)
                st = getattr(big, call)(ctx, *args, noalloc)
                stub.stub_fail_device_after(-1)
                assert st in (N.NVA_OK, N.NVA_E_OOM), (call, n, st)
                assert getattr(big, call)(ctx, *args, noalloc) == N.NVA_OK
                lib.nva_kv_destroy(kv)
                lib.nva_ctx_destroy(ctx)


def stat(ctx, name):
    n = ctypes.c_int64()
    assert lib.nva_ctx_kernel_stats(ctx, name, ctypes.byref(n), None) == N.NVA_OK
    return n.value


def shared_work_area():
    """Naming prefix groups takes nothing away from the no-allocation form: a step whose shared plan
    is larger than the array is read apart if that fits, and shared up to there."""
    ctx = context()
    lib.nva_ctx_set_timing(ctx, 1)
    seen = set()
    for new in (60, 70, 80, 90, 100, 110, 120, 200):
        step = Step(24, 8192, 0, new, heads=(32, 8, 128))
        step.desc.write_kv = 0
        step.num_blocks = 1  # nothing reads the pages here: one for all
        step.table[:] = np.where(step.table >= 0, 0, -1)
        st, kv = step.arena(ctx)
        assert st == step.set(ctx) == N.NVA_OK
        apart = step.attend(ctx, kv, True)
        lib.nva_ctx_reset_stats(ctx)
        assert step.share(ctx) == N.NVA_OK
        shared = step.attend(ctx, kv, True)
        spans = stat(ctx, b"span_tiles") + stat(ctx, b"span")
        seen.add((apart, shared, spans))
        print(new, apart, shared, spans, flush=True)
        assert (shared == N.NVA_OK) == (apart == N.NVA_OK), (new, apart, shared)
        assert step.attend(ctx, kv) == N.NVA_OK  # and the allocating form shares
        lib.nva_kv_destroy(kv)
    assert {(N.NVA_OK, N.NVA_OK, 1), (N.NVA_OK, N.NVA_OK, 0)} <= seen, seen
    lib.nva_ctx_destroy(ctx)


def plan_time():
    """Planning a decode step's spans costs the host no more than planning its rows read apart: the
    least of 40 builds each, for rows under a shared prefix and for rows over encoder states."""
    ctx = context()
    lib.nva_ctx_set_timing(ctx, 1)

    def least(step, call, *before):
        times = []
        for _ in range(40):
            for f in (step.set, *before):
                assert f(ctx) == N.NVA_OK
            lib.nva_ctx_reset_stats(ctx)
            assert call() == N.NVA_OK
            ms, n = ctypes.c_double(), ctypes.c_int64()
            lib.nva_ctx_kernel_stats(ctx, b"plan", ctypes.byref(n), ctypes.byref(ms))
            assert n.value == 1
            times.append(1e3 * ms.value)
        return min(times)

    for rows in (64, 256, 1024):
        step = Step(rows, 8192, 211, 1, block=256)
        step.desc.write_kv = 0
        step.num_blocks = 1  # nothing reads the pages here: one for all
        step.table[:] = np.where(step.table >= 0, 0, -1)
        st, kv = step.arena(ctx)
        assert st == N.NVA_OK
        step.enc_len = i32(300 + 37 * np.arange(rows) % 1201)
        apart = least(step, lambda: step.attend(ctx, kv))
        shared = least(step, lambda: step.attend(ctx, kv), step.share)
        cross = least(step, lambda: step.attend_encoder(ctx), step.encode)
        print(f"{rows} rows: apart {apart:.1f}, shared {shared:.1f}, encoder {cross:.1f} us", flush=True)
        assert shared <= 1.5 * apart and cross <= 1.5 * apart
        lib.nva_kv_destroy(kv)
    lib.nva_ctx_destroy(ctx)


def most_keys():
    """Key counts from which the kernels' 32-bit key numbers would pass 2^31 are refused, whatever the
    pages and pools hold; the longest below are planned."""
    ctx = context()
    limit = 2 ** 31 - 1 - 8192
    for keys, want in ((2 ** 31 - 1, N.NVA_E_UNSUPPORTED), (limit + 1, N.NVA_E_UNSUPPORTED),
                       (limit, N.NVA_OK)):
        for new in (1, 3):
            step = Step(2, 64, 0, new, block=1 << 20, heads=(2, 1, 64))
            step.desc.write_kv = 0
            step.num_blocks = 1
            step.table = np.zeros((2, 2048), np.int32)
            step.context_lens[0] = keys
            step.cu_k[1:] = [keys, min(keys + 64 + new, 2 ** 31 - 1)]
            step.groups = (N.PrefixGroup * 1)(N.PrefixGroup(0, 1, keys - new))
            st, kv = step.arena(ctx)
            assert st == N.NVA_OK
            assert step.set(ctx) == N.NVA_OK
            assert step.attend(ctx, kv) == want, (keys, new)
            assert step.share(ctx) == N.NVA_OK
            before = stub.stub_launches()
            assert step.attend(ctx, kv) == want, (keys, new)
            step.enc_start, step.enc_len = i32([0, 5]), i32([keys, 60])
            assert step.encode(ctx) == N.NVA_OK
            p = step.aligned()
            got = lib.nva_cross_attention_forward(ctx, ctypes.byref(step.cross), p, p, p, 2 ** 33, 64,
                                                  step.tokens, p)
            assert got == want, (keys, new, got)
            assert want == N.NVA_OK or stub.stub_launches() == before
            lib.nva_kv_destroy(kv)
    lib.nva_ctx_destroy(ctx)


def rows_before_the_first():
    """A prefill step whose first row or key is negative would read in front of q, or of the dense k and
    v: it is refused, and the step set before stays."""
    ctx = context()
    step = Step(3, 128, 10, 4)
    st, kv = step.arena(ctx)
    assert st == step.set(ctx) == step.attend(ctx, kv) == N.NVA_OK
    for cu in ("cu_q", "cu_k"):
        for first in (-1, -2 ** 31):
            bad = Step(3, 128, 10, 4)
            getattr(bad, cu)[0] = first
            before = stub.stub_launches()
            assert bad.set(ctx) == N.NVA_E_ARG, (cu, first)
            assert stub.stub_launches() == before
            assert step.attend(ctx, kv) == N.NVA_OK
    lib.nva_kv_destroy(kv)
    lib.nva_ctx_destroy(ctx)


if __name__ == "__main__":
    globals()[sys.argv[2]]()
    print("ok", flush=True)
