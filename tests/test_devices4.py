"""Tensors on another device than the context's: the 4-bit calls refuse them before they reach the
library (its kernels would follow the pointers from the wrong device)."""

import pytest
import torch

from nanollvm_amd import (Attention, Context, IllegalArgumentException, KvCacheArena4, Linear4, RMSNorm,
                          RotaryEmbedding, quantize4)


class Elsewhere:
    """What the checks ask of a contiguous tensor on device 1."""

    is_cuda = True

    def __init__(self, *shape, dtype=torch.float32):
        self.shape, self.dtype = torch.Size(shape), dtype

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return True

    def get_device(self):
        return 1

    def data_ptr(self):
        return 4096


class Here(Elsewhere):
    def get_device(self):
        return 0


@pytest.fixture
def ctx():
    c = Context.__new__(Context)
    c._h, c.device, c._positions_key = None, 0, None
    c._kv = KvCacheArena4.__new__(KvCacheArena4)
    c._kv._h, c._kv._ctx, c._kv.num_layers, c._kv.num_kv_heads, c._kv.head_dims = None, c, 1, 2, [64]
    return c


LAYER = Attention(4, 64, 0.125, 2)
WRONG = "context's device"


def rows(cls=Here):
    return [cls(3, 4, 64), cls(3, 2, 64), cls(3, 2, 64)]


@pytest.mark.parametrize("i", range(3))
def test_attention(ctx, i):
    t = rows()
    t[i] = Elsewhere(*t[i].shape)
    rope = RotaryEmbedding.__new__(RotaryEmbedding)
    rope._h = None
    for call in (lambda: LAYER.forward(*t, ctx), lambda: LAYER.forward_with_rope(rope, None, *t, ctx),
                 lambda: LAYER.forward_with_norm_rope(rope, None, *t, ctx,
                                                      q_norm=RMSNorm.weightless(1e-6))):
        with pytest.raises(IllegalArgumentException, match=WRONG):
            call()


def test_where_rotated_rows_go(ctx):
    t = rows()
    for out in (dict(q_out=Elsewhere(3, 4, 64)), dict(k_out=Elsewhere(3, 2, 64))):
        with pytest.raises(IllegalArgumentException, match=WRONG):
            LAYER.forward_with_norm_rope(None, None, *t, ctx, **out)
        with pytest.raises(IllegalArgumentException, match=WRONG):
            LAYER.forward_packed_qkv(None, None, Here(3, 8 * 64), ctx, **out)
    with pytest.raises(IllegalArgumentException, match=WRONG):
        LAYER.forward_packed_qkv(None, None, Elsewhere(3, 8 * 64), ctx)


def test_rows_of_the_arena(ctx):
    slots = Here(3, dtype=torch.int32)
    for args in ((Elsewhere(3, dtype=torch.int32), Here(3, 2, 64), Here(3, 2, 64)),
                 (slots, Elsewhere(3, 2, 64), Here(3, 2, 64)),
                 (slots, Here(3, 2, 64), Elsewhere(3, 2, 64))):
        with pytest.raises(IllegalArgumentException, match=WRONG):
            ctx._kv.write_rows(0, *args)
    with pytest.raises(IllegalArgumentException, match=WRONG):
        ctx._kv.read_rows(0, Elsewhere(3, dtype=torch.int32))


def test_step(ctx):
    fresh = Here(2, dtype=torch.int32)
    with pytest.raises(IllegalArgumentException, match=WRONG):
        ctx.extend(None, Elsewhere(2, dtype=torch.int32), 2, 1)
    with pytest.raises(IllegalArgumentException, match=WRONG):
        ctx.extend(None, fresh, 2, 1, keep=Elsewhere(2, dtype=torch.int32))


def test_projections(ctx):
    codes, scales = Here(8, 32, dtype=torch.uint8), Here(8, 2, dtype=torch.uint8)
    for args in ((Elsewhere(8, 32, dtype=torch.uint8), scales), (codes, Elsewhere(8, 2, dtype=torch.uint8)),
                 (codes, scales, Elsewhere(8))):
        with pytest.raises(IllegalArgumentException, match=WRONG):
            Linear4(ctx, *args)
    with pytest.raises(IllegalArgumentException, match=WRONG):
        quantize4(Elsewhere(2, 64), ctx)
    layer = Linear4.__new__(Linear4)
    layer._h, layer.bias, layer.in_features, layer.out_features = None, None, 64, 8
    with pytest.raises(IllegalArgumentException, match=WRONG):
        layer.forward(Elsewhere(2, 64), ctx)
