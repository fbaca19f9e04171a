"""Plain 64-bit implementations that the tests of the 4-bit form, the device-built steps and scaled
rotary positions compare with, written from their definitions, and what those tests share.

Bars: the stored values, tables and slots exactly; attention and projections the path's max-abs 1e-4
and rel-L2 1e-5 (relative to the largest magnitude expected, where that passes 1)."""

import numpy as np
import torch

from cases import rel_l2

MAX_ABS = 1e-4
REL_L2 = 1e-5
VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def quantize(x):
    """(codes of one a byte, scale bytes) of x [.., n] by the definition, in 64 bits."""
    b = np.asarray(x, np.float64).reshape(-1, 32)
    codes = np.zeros(b.shape, np.uint8)
    scales = np.zeros(len(b), np.uint8)
    for i, row in enumerate(b):
        if not np.all(np.isfinite(row)):
            scales[i] = 255
            continue
        top = np.abs(row).max()
        e = -127
        while e < 125 and top > 6 * 2.0 ** e:
            e += 1
        scales[i] = e + 127
        a = np.abs(row) / 2.0 ** e
        gap = np.abs(a[:, None] - VALUES)
        gap[:, 1::2] += np.finfo(np.float64).tiny  # the even one of two as near
        best = gap.min(1, keepdims=True)
        near = gap == best
        even = near & (np.arange(8) % 2 == 0)
        pick = np.where(even.any(1), even.argmax(1), near.argmax(1))
        codes[i] = pick | (np.signbit(row).astype(np.uint8) << 3)
    shape = np.shape(x)
    return codes.reshape(shape), scales.reshape(*shape[:-1], shape[-1] // 32)


def values(codes, scales):
    """What codes (one a byte) and scale bytes stand for."""
    v = VALUES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    unit = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(*scales.shape, 32) * unit[..., None]).reshape(codes.shape)


def held(x):
    """The values that x is held as."""
    return values(*quantize(x))


def held_fast(x):
    """The same, vectorised, for finite x (checked against held)."""
    x = np.asarray(x, np.float32)
    b = x.reshape(-1, 32)
    m, e = np.frexp(np.abs(b).max(1))
    e = np.where(m == 0, -127, np.clip(np.where(m <= 0.75, e - 3, e - 2), -127, 125))
    a = np.abs(b.astype(np.float64)) / np.exp2(e.astype(np.float64))[:, None]
    c = sum((a > t if odd else a >= t).astype(np.int64) for t, odd in
            ((0.25, 1), (0.75, 0), (1.25, 1), (1.75, 0), (2.5, 1), (3.5, 0), (5.0, 1)))
    v = VALUES[c] * np.exp2(e.astype(np.float64))[:, None]
    return np.where(b < 0, -v, v).reshape(x.shape)


def softmax_rows(logits, values_):
    """softmax(logits) values_, zeros where nothing is seen (logits -infinity)."""
    top = logits.max(-1, keepdims=True) if logits.shape[-1] else np.full((len(logits), 1), -np.inf)
    w = np.exp(logits - np.where(np.isneginf(top), 0, top))
    total = w.sum(-1, keepdims=True)
    out = w @ values_
    return np.where(total == 0, 0, out / np.where(total == 0, 1, total))


def attention(q, k, v, cached, scale, window=0):
    """One sequence: q [n, hq, d] at positions cached.., over k and v [cached + n, hkv, d]."""
    n, hq, d = q.shape
    keys, hkv = k.shape[:2]
    rep = hq // hkv
    pos = np.arange(cached, cached + n)[:, None]
    key = np.arange(keys)[None]
    hidden = key > pos
    if window > 0:
        hidden = hidden | (key <= pos - window)
    out = np.zeros(q.shape)
    for h in range(hq):
        s = q[:, h].astype(np.float64) @ k[:, h // rep].T.astype(np.float64) * scale
        out[:, h] = softmax_rows(np.where(hidden, -np.inf, s), v[:, h // rep].astype(np.float64))
    return out


def close(got, want, what=""):
    got = got.cpu().numpy() if isinstance(got, torch.Tensor) else np.asarray(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.size == 0:
        return
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad), f"{what}: NaN in other places"
    got, want = got[~bad].astype(np.float64), want[~bad]
    if got.size == 0:
        return
    err = np.abs(got - want).max() / max(1.0, np.abs(want).max())
    l2 = rel_l2(got, want) if np.any(want) else 0.0
    print(f"[gpu] {what}: max_abs={err:.2e} rel_l2={l2:.2e}", flush=True)
    assert err <= MAX_ABS and l2 <= REL_L2, (what, err, l2)


class Tables:
    """The block tables' rules over Python lists."""

    def __init__(self, seqs, max_tokens, blocks, block_size, pages=None):
        self.bs, self.max_tokens = block_size, max_tokens
        self.stack = list(pages if pages is not None else range(blocks))[::-1]
        self.blocks = [[] for _ in range(seqs)]
        self.lens = [0] * seqs

    def extend(self, new, num_tokens, max_new, keep=None):
        """(code, number), and of a step that fits the slots, positions and row offsets."""
        n = len(new)
        keep = list(self.lens[:n]) if keep is None else list(keep)
        for b in range(n):
            if not (0 <= keep[b] <= self.lens[b] and 0 <= new[b] <= max_new and
                    keep[b] + new[b] <= self.max_tokens):
                return self._none(1, b, n, num_tokens)
        if sum(new) > num_tokens:
            return self._none(2, sum(new), n, num_tokens)
        up = lambda t: -(-t // self.bs)
        need = sum(up(k + w) - up(k) for k, w in zip(keep, new))
        if need > len(self.stack) + sum(len(t) - up(k) for t, k in zip(self.blocks, keep)):
            return self._none(3, need, n, num_tokens)
        for b in reversed(range(n)):
            while len(self.blocks[b]) > up(keep[b]):
                self.stack.append(self.blocks[b].pop())
        slots, positions, cu = [], [], [0]
        for b in range(n):
            t = self.blocks[b]
            while len(t) < up(keep[b] + new[b]):
                t.append(self.stack.pop())
            for p in range(keep[b], keep[b] + new[b]):
                slots.append(t[p // self.bs] * self.bs + p % self.bs)
                positions.append(p)
            self.lens[b] = keep[b] + new[b]
            cu.append(cu[-1] + new[b])
        pad = num_tokens - len(slots)
        return (0, 0), slots + [-1] * pad, positions + [0] * pad, cu

    @staticmethod
    def _none(code, number, n, num_tokens):
        return (code, number), [-1] * num_tokens, [0] * num_tokens, [0] * (n + 1)

    def table(self, width):
        out = np.full((len(self.blocks), width), -1, np.int32)
        for row, t in zip(out, self.blocks):
            row[:len(t)] = t
        return out

    def check(self, tables, got, what=""):
        """The device's arrays against the outcome of extend()."""
        (code, number), slots, positions, cu = got
        status = tables.status()
        assert status == (code, number, len(self.stack)), (what, status, code, number)
        assert tables.slots.tolist() == slots, what
        assert tables.positions.tolist() == positions, what
        assert tables.cu_q.tolist() == cu, what
        assert tables.lens.tolist() == self.lens, what
        t = tables.block_tables.cpu().numpy()
        assert np.array_equal(t, self.table(t.shape[1])), what


def frequencies(rd, base, scaling="none", factor=1.0, original_max_position=0, low=0.0, high=0.0):
    """Angle per position of every pair and the factor of cos and sin."""
    base = float(np.float32(base))
    i = np.arange(0, rd, 2, dtype=np.float64)
    if scaling == "ntk" and rd > 2:
        base = base * factor ** (rd / (rd - 2))
    f = base ** (-i / rd)
    turns = original_max_position * f / (2 * np.pi)
    if scaling == "linear" or (scaling == "ntk" and rd == 2):
        f = f / factor
    elif scaling == "yarn":
        # Solve turns(pair) = low and high on the unscaled frequencies.
        pair = lambda t: rd * np.log(original_max_position / (2 * np.pi * t)) / (2 * np.log(base))
        lo, hi = max(np.floor(pair(high)), 0), min(np.ceil(pair(low)), rd - 1)
        mix = np.clip((i / 2 - lo) / max(hi - lo, 1e-3), 0, 1)
        f = f / factor * mix + f * (1 - mix)
    elif scaling == "bands":
        mix = np.clip((turns - low) / (high - low), 0, 1)
        f = (1 - mix) * f / factor + mix * f
    return f, 0.1 * np.log(factor) + 1 if scaling == "yarn" else 1.0


def rotate(x, positions, f, amplitude=1.0, interleaved=False):
    """x [n, heads, d] turned by positions x f in its first dims."""
    rd = 2 * len(f)
    a = np.outer(np.asarray(positions, np.float64), f)[:, None]
    c, s = amplitude * np.cos(a), amplitude * np.sin(a)
    out = x.astype(np.float64).copy()
    first = slice(0, rd, 2) if interleaved else slice(0, rd // 2)
    second = slice(1, rd, 2) if interleaved else slice(rd // 2, rd)
    u, w = x[..., first].astype(np.float64), x[..., second].astype(np.float64)
    out[..., first], out[..., second] = u * c - w * s, w * c + u * s
    return out
