"""Helpers of the shared-prefix and cross-attention tests: steps whose sequences share pages, encoder
pools, and softmax(q k^T scale) v in 64 bits, row by row of its definition.

Bounds.  Outputs are fp32 sums like those of every attention path here and are held to the same bar:
max-abs 1e-4 and rel-L2 1e-5.  For N(0, 1) inputs at scale d^-0.5 a score's rounding error is about
sqrt(d) 2^-24 of values of size 1, so a probability's is below 2^-20 of itself even for the largest
scores (|s| < 16: the exponential's argument is rounded to 2^-21), and the weighted mean of N(0, 1)
values moves by less than that relative to their size: 1e-6 where the bar is 1e-5."""

import numpy as np
import torch

from gpu_checks import MAX_ABS, REL_L2, say

from nanollvm_amd import step


class SharedStep:
    """A step over pages.  ``groups`` lists (sequences, prefix tokens), whole pages that the sequences
    share; sequence i of the step has own[i] = (cached, new) tokens behind its group's prefix."""

    def __init__(self, groups, own, block, seed, decode=None, first_block=0):
        r = np.random.default_rng(seed)
        self.block = block
        self.prefix = [p for n, p in groups for _ in range(n)]
        self.own = list(own)
        assert len(self.prefix) == len(self.own)
        self.decode = all(n == 1 for _, n in own) if decode is None else decode
        self.keys = [p + c + n for p, (c, n) in zip(self.prefix, self.own)]
        self.new = [n for _, n in self.own]
        need = sum(-(-k // block) for k in self.keys) + 2
        ids = iter((first_block + r.permutation(need + 3)).tolist())
        self.num_blocks = first_block + need + 3
        tables, b = [], 0
        for n, p in groups:
            assert p % block == 0
            head = [next(ids) for _ in range(p // block)]
            for _ in range(n):
                t = list(head)
                while len(t) * block < self.keys[b]:
                    t.append(next(ids))
                tables.append(t)
                b += 1
        width = max(1, max(len(t) for t in tables))
        self.tables = np.full((len(tables), width), -1, np.int32)
        for i, t in enumerate(tables):
            self.tables[i, :len(t)] = t
        self.slots = [np.asarray([t[j // block] * block + j % block for j in range(k)], np.int64)
                      for t, k in zip(tables, self.keys)]
        self.groups = []
        at = 0
        for n, p in groups:
            self.groups.append((at, n, p))
            at += n
        self.cu_q = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.tokens = int(self.cu_q[-1])

    def context_args(self):
        lens = np.asarray(self.keys, np.int32)
        slots = np.concatenate([s[len(s) - n:] for s, n in zip(self.slots, self.new)])
        if self.decode:
            return dict(is_prefill=False, context_lens=lens, slot_mapping=slots,
                        block_tables=self.tables)
        return dict(is_prefill=True, cu_seqlens_q=self.cu_q,
                    cu_seqlens_k=np.concatenate([[0], np.cumsum(lens)]).astype(np.int32),
                    max_seqlen_q=max(self.new), max_seqlen_k=int(lens.max()), slot_mapping=slots,
                    block_tables=self.tables)

    def found(self):
        return step.find_shared_prefixes(self.tables,
                                         [k - n for k, n in zip(self.keys, self.new)], self.block)


def attend(q, k, v, scale, seen=None):
    """softmax(q k^T scale) v in 64 bits, q [n, hq, d], k and v [keys, hkv, d]; ``seen`` [n, keys]
    masks.  Rows that see nothing, or only scores of -inf, are zero."""
    n, hq, d = q.shape
    hkv = k.shape[1]
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    if k.shape[0] == 0 or n == 0:
        return out
    for h in range(hq):
        kv = h // (hq // hkv)
        s = (q[:, h].double() @ k[:, kv].double().T.contiguous()) * scale
        if seen is not None:
            s = torch.where(seen, s, torch.full_like(s, -torch.inf))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -torch.inf, torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        # A value that is not finite makes every result not finite that it has a weight in: of a
        # key whose score is above -inf, however small, that is more than 0.
        vv = v[:, kv].double()
        odd = ~torch.isfinite(vv)
        o = p @ torch.where(odd, torch.zeros_like(vv), vv)
        hit = (s > -torch.inf).double() @ odd.double()
        o = torch.where(hit > 0, torch.full_like(o, torch.inf), o)
        out[:, h] = torch.where(total == 0, torch.zeros_like(o), o / total)
    return out


def step_reference(st, q, k_pages, v_pages, scale, window=0):
    """Every sequence over its own slots, causal; k_pages and v_pages [slots, hkv, d] hold the
    step's rows already."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, (keys, n) in enumerate(zip(st.keys, st.new)):
        a = int(st.cu_q[b])
        rows = torch.from_numpy(st.slots[b]).to(q.device)
        pos = torch.arange(keys - n, keys, device=q.device)[:, None]
        t = torch.arange(keys, device=q.device)[None]
        seen = t <= pos
        if window:
            seen &= t > pos - window
        out[a:a + n] = attend(q[a:a + n], k_pages[rows], v_pages[rows], scale, seen)
    return out


def close(got, want, name):
    got = got.double()
    err = (got - want).abs()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), f"{name}: finite values differ"
    fine = torch.isfinite(want)
    big = float(err[fine].max()) if fine.any() else 0.0
    norm = float(want[fine].norm())
    rel = float(err[fine].norm()) / norm if norm else float(err[fine].norm())
    say(f"{name}: max_abs={big:.3e} rel_l2={rel:.3e}")
    assert big <= MAX_ABS and rel <= REL_L2, (name, big, rel)
