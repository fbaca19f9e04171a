"""Rows into and out of the 4-bit arena whose threads pass 2^32 in a call: every row is read and written.  One
buffer of 64 GiB."""

import pytest
import torch

from nanollvm_amd import Context, KvCacheArena4, _native

pytestmark = pytest.mark.gpu

HKV, D = 8, 512
VALUES = (0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 8.0)  # held exactly
ROWS = (1 << 22) + 5  # two launches: a row of K and V is 2 * 8 * 64 threads


@pytest.fixture(scope="module")
def buffer():
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GiB of free device memory")
    x = torch.zeros(ROWS * HKV * D, device="cuda").view(ROWS, HKV, D)
    yield x
    del x
    torch.cuda.empty_cache()


def test_write_and_read(buffer):
    lib = _native.load()
    # First and last rows, and rows about the launches' borders.
    rows = [0, 1, (1 << 21) - 1, 1 << 21, (1 << 21) + 1, (1 << 22) - 1, 1 << 22, ROWS - 1]
    with Context(0) as ctx, KvCacheArena4(ctx, 1, 2, 32, HKV, D) as arena:
        slots = torch.full((ROWS,), -1, dtype=torch.int32, device="cuda")
        for i, r in enumerate(rows):
            slots[r] = 7 * i
            buffer[r] = VALUES[i]
        torch.cuda.synchronize()
        assert lib.nva_kv4_write_rows(arena.handle, 0, slots.data_ptr(), buffer.data_ptr(),
                                      buffer.data_ptr(), ROWS) == _native.NVA_OK
        ctx.sync()
        for x in arena.read_rows(0, torch.arange(64, dtype=torch.int32, device="cuda")):
            for i in range(64):
                want = VALUES[i // 7] if i % 7 == 0 and i // 7 < len(rows) else 0.0
                assert torch.all(x[i] == want), i
        for which in range(2):
            buffer.fill_(9.0)
            torch.cuda.synchronize()
            out = [None, None]
            out[which] = buffer.data_ptr()
            assert lib.nva_kv4_read_rows(arena.handle, 0, slots.data_ptr(), *out, ROWS) == _native.NVA_OK
            ctx.sync()
            for i, r in enumerate(rows):
                assert torch.all(buffer[r] == VALUES[i]), r
                buffer[r] = 0.0
            for at in range(0, ROWS, 1 << 16):  # slots outside the arena read as zeros
                assert not buffer[at:at + (1 << 16)].any(), at
