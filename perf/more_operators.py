"""Timed cases of the operators of a step whose cache and projections are held in 4 bits and whose
pages are handed out on the GPU, each case one pass.

``rope``    rotary positions of a step's q and k: halves or neighbours paired, part of the head
            rotated, frequencies scaled for contexts beyond the trained one.
``tables``  the step's metadata from request lengths, on the GPU: how many tokens of each sequence
            stay and how many follow give the pages taken from and returned to the pool, the block
            tables, the slot and position of every token and the row offsets.
``kv4``     attention of a step over a paged cache held in 4 bits: the step's K/V rows are rounded
            into their pages, then every query attends over its sequence's keys, causally.
``linear``  y = x W^T + b with W held in 4 bits.

The 4-bit form holds 32 values along a row as signed codes of {0, 0.5, 1, 1.5, 2, 3, 4, 6} beside
one power of two: the smallest 2^e, -127 <= e <= 125, with every magnitude at most 6 * 2^e.  Each
value goes to the nearest code, ties to the even one.  (Scale byte e + 127; a code's sign is bit 3.)

Lengths come from ``layout``; the inputs, and the order of pages, from the seed.
"""

import functools
import math
import os
import sys

import numpy as np
import torch

own = False  # the framework's operators; False: their plain form in elementary operations

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# q heads, KV heads, head dim.
SHAPES = {
    "16/8/128": (16, 8, 128),
    "32/8/128": (32, 8, 128),
    "40/8/128": (40, 8, 128),
    "32/8/64": (32, 8, 64),
    "4/1/256": (4, 1, 256),
    "8/1/512": (8, 1, 512),
    "12/12/64": (12, 12, 64),
}

# Frequencies of rotary positions: scaling, its factor, the context it was trained for, and for the
# two that treat frequencies by their turns within that context, the two limits.
SCALINGS = {
    "none": dict(scaling="none"),
    "linear": dict(scaling="linear", factor=4.0),
    "ntk": dict(scaling="ntk", factor=8.0),
    "yarn": dict(scaling="yarn", factor=4.0, original_max_position=32768, low=1.0, high=32.0),
    "bands": dict(scaling="bands", factor=8.0, original_max_position=8192, low=1.0, high=4.0),
}


def _case(kind, name, **what):
    return dict(kind=kind, **({"name": name} if name else {}), **what)


def _rope(name, shape, tokens, *, rotary, interleaved, scaling, max_pos, base=1e6):
    return _case("rope", name, shape=shape, tokens=tokens, rotary=rotary, interleaved=interleaved,
                 scaling=scaling, max_pos=max_pos, base=base)


def _tables(name, seqs, *, klo, khi, nlo, nhi, idle=0.0, block=256, pad=0, layout=0):
    return _case("tables", name, seqs=seqs, klo=klo, khi=khi, nlo=nlo, nhi=nhi, idle=idle,
                 block=block, pad=pad, layout=layout)


def _kv4(name, shape, seqs, *, clo, chi, nlo=1, nhi=1, window=0, block=256, layout=0):
    return _case("kv4", name, shape=shape, seqs=seqs, clo=clo, chi=chi, nlo=nlo, nhi=nhi,
                 window=window, block=block, layout=layout)


def _linear(name, rows, inner, outer, *, bias=False):
    return _case("linear", name, rows=rows, inner=inner, outer=outer, bias=bias)


def listed():
    return [
        # A decode batch's q and k of a model that rotates half of each head, neighbours paired.
        _rope("rope_decode_64_rows_part", "32/8/128", 64, rotary=64, interleaved=True,
              scaling="none", max_pos=40960),
        # A long prompt's chunk far behind the trained context.
        _rope("rope_prompt_8192_yarn", "32/8/128", 8192, rotary=128, interleaved=False,
              scaling="yarn", max_pos=131072),
        # One decode step of a full batch: a token for each, a page for few, idle rows between.
        _tables("tables_decode_256", 256, klo=1, khi=8000, nlo=1, nhi=1, idle=0.06, block=32),
        # Prompts of a new batch, odd lengths, rows whose request is replaced among them.
        _tables("tables_prompts_61", 61, klo=0, khi=3000, nlo=1, nhi=900, idle=0.1, block=64,
                pad=37),
        # A handful of short chats: launches and latency count.
        _kv4("kv4_decode_5_rows", "16/8/128", 5, clo=0, chi=700),
        # A full decode batch of a chat service.
        _kv4("kv4_decode_128_rows", "32/8/128", 128, clo=500, chi=16000),
        # Few rows with long documents: the keys of one row over many workgroups.
        _kv4("kv4_decode_3_rows_long", "32/8/64", 3, clo=60000, chi=120000, block=64),
        # Multi-query heads, wide, in a layer with a window.
        _kv4("kv4_decode_mqa_window", "4/1/256", 96, clo=200, chi=9000, window=1024, block=32),
        # Prompt chunks behind cached tokens, one-token ones among them.
        _kv4("kv4_prefill_chunks", "32/8/128", 12, clo=0, chi=4000, nlo=1, nhi=700),
        # The projection behind attention for one row.
        _linear("linear_1_row", 1, 4096, 2560),
        # A decode batch.
        _linear("linear_48_rows", 48, 4096, 2560, bias=True),
        # A prompt.
        _linear("linear_1500_rows", 1500, 4096, 2560),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges; no larger than the largest listed one."""
    while True:
        case = _draw(rng)
        w = work(case)
        size = 0
        if case["kind"] == "kv4":
            hq, hkv, d = SHAPES[case["shape"]]
            seqs = _seqs(case)
            keys = max(c + n for c, n in seqs)
            size = len(seqs) * keys * 4 * max(hkv * d, hq * max(n for _, n in seqs))
        if w["bytes"] <= 2.5e9 and w["flops"] <= 1.2e11 and size <= 9e9:
            return case


def _draw(rng):
    kind = rng.choice(["rope", "tables", "kv4", "kv4", "linear"])
    layout = rng.randrange(1 << 20)
    if kind == "rope":
        shape = rng.choice(sorted(SHAPES))
        d = SHAPES[shape][2]
        scaling = rng.choice(sorted(SCALINGS))
        return _rope(None, shape, _log(rng, 1, 9000), rotary=rng.choice([d, d, d // 2, d // 4]),
                     interleaved=rng.random() < 0.5, scaling=scaling,
                     max_pos=40960 if scaling == "none" else 131072,
                     base=rng.choice([1e4, 5e5, 1e6]))
    if kind == "tables":
        khi = _log(rng, 1, 9000)
        nhi = 1 if rng.random() < 0.4 else _log(rng, 1, 1000)
        return _tables(None, _log(rng, 1, 600), klo=rng.choice([0, khi // 4]), khi=khi,
                       nlo=rng.choice([0, 1]), nhi=nhi, idle=rng.choice([0.0, 0.1, 0.5]),
                       block=rng.choice([32, 64, 256]), pad=rng.choice([0, 0, 13]), layout=layout)
    if kind == "kv4":
        chi = _log(rng, 1, 16000)
        nhi = 1 if rng.random() < 0.6 else _log(rng, 2, 700)
        window = _log(rng, 1, 4000) if rng.random() < 0.25 else 0
        return _kv4(None, rng.choice(sorted(SHAPES)), _log(rng, 1, 150),
                    clo=rng.choice([0, chi // 8, chi]), chi=chi, nlo=rng.choice([0, 1, nhi]),
                    nhi=nhi, window=window, block=rng.choice([32, 64, 96, 256]), layout=layout)
    return _linear(None, _log(rng, 1, 1500), 32 * _log(rng, 2, 256), _log(rng, 16, 8000),
                   bias=rng.random() < 0.3)


@functools.lru_cache(maxsize=64)
def _sequences(seqs, clo, chi, nlo, nhi, layout):
    """(cached, new) tokens of every sequence of a step; one token in all at least."""
    r = np.random.default_rng(layout)
    got = [(int(r.integers(clo, chi + 1)), int(r.integers(nlo, nhi + 1))) for _ in range(seqs)]
    return tuple(got if any(n for _, n in got) else [(got[0][0], 1)] + got[1:])


def _seqs(case):
    return _sequences(*(case[k] for k in ("seqs", "clo", "chi", "nlo", "nhi", "layout")))


@functools.lru_cache(maxsize=64)
def _lengths(seqs, klo, khi, nlo, nhi, idle, layout):
    """(tokens that stay, tokens that follow) of every row of the tables."""
    r = np.random.default_rng(layout)
    keep, new = r.integers(klo, khi + 1, seqs), r.integers(nlo, nhi + 1, seqs)
    new[r.random(seqs) < idle] = 0
    keep[r.random(seqs) < idle / 2] = 0
    return keep.astype(np.int32), new.astype(np.int32)


def _rows_of(case):
    return _lengths(*(case[k] for k in ("seqs", "klo", "khi", "nlo", "nhi", "idle", "layout")))


def _scale(case):
    return float(np.float32(SHAPES[case["shape"]][2] ** -0.5))


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 16 + salt)
    return g


def _randn(seed, salt, *shape):
    return torch.randn(*shape, device="cuda", generator=_gen(seed, salt))


# ---------------------------------------------------------------- the 4-bit form

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _codes4(x):
    """Codes [.., n / 2], two a byte, and scale bytes [.., n / 32] of x [.., n]."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, 0.5 <= m < 1: at most 6 * 2^(e - 3) where m <= 0.75
    e = torch.where(top == 0, -127, e - 3 + (m > 0.75).int()).clamp(-127, 125)
    a = torch.ldexp(b.abs(), -e)
    c = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() +
         (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5).byte())
    c = (c | (torch.signbit(b).byte() << 3)).reshape(x.shape)
    return c[..., 0::2] | (c[..., 1::2] << 4), (e + 127).byte().squeeze(-1)


def _values4(codes, scales):
    """What codes and scale bytes stand for, in 32 bits."""
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1)
    v = v.reshape(*scales.shape, 32) * torch.ldexp(
        torch.ones(scales.shape, device=codes.device), scales.int() - 127).unsqueeze(-1)
    return v.reshape(*codes.shape[:-1], -1)


def _in_pieces(f, x, rows=1 << 15):
    got = [f(x[i:i + rows]) for i in range(0, len(x), rows)]
    return [torch.cat(p) for p in zip(*got)]


# ---------------------------------------------------------------- the framework's side

def _framework():
    pkg = os.path.join(_ROOT, "nano-vllm-java_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import nanollvm_amd
    return nanollvm_amd


class _Engine:
    """What a program keeps between steps, and what it closes at its end."""

    def __init__(self):
        self.nva = _framework()
        self.ctx = self.nva.Context(0)
        self.held = []

    def keep(self, x):
        self.held.append(x)
        return x

    def __del__(self):
        for x in reversed(getattr(self, "held", [])):
            x.close()
        if getattr(self, "ctx", None) is not None:
            self.ctx.close()


# ---------------------------------------------------------------- rope

def _positions(case, seed):
    """Ascending positions of a chunk (many tokens) or any of a batch's rows."""
    r = np.random.default_rng(seed)
    n, top = case["tokens"], case["max_pos"]
    if n <= 512:
        return r.integers(0, top, n)
    return int(r.integers(0, max(1, top - n))) + np.arange(n)


def _frequencies(case):
    """Angle of one position of every pair, in 64 bits, and the factor of cos and sin."""
    rd, s = case["rotary"], SCALINGS[case["scaling"]]
    base, how = case["base"], s["scaling"]
    if how == "ntk" and rd > 2:
        base *= s["factor"] ** (rd / (rd - 2))
    f = base ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    if how == "linear" or how == "ntk" and rd <= 2:
        f = f / s["factor"]
    if how == "yarn":
        # Pairs of more than `high` turns in the trained context stay, of fewer than `low` are
        # stretched, and those between are mixed along the pair's number.
        def pair(turns):
            return (rd * math.log(s["original_max_position"] / (turns * 2 * math.pi)) /
                    (2 * math.log(case["base"])))
        lo, hi = max(0, math.floor(pair(s["high"]))), min(rd - 1, math.ceil(pair(s["low"])))
        ramp = ((torch.arange(rd // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f / s["factor"] * ramp + f * (1 - ramp)
    if how == "bands":
        turns = s["original_max_position"] * f / (2 * math.pi)
        mix = ((turns - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        f = (1 - mix) * f / s["factor"] + mix * f
    return f, 0.1 * math.log(s["factor"]) + 1.0 if how == "yarn" else 1.0


def _prepare_rope(case, seed):
    hq, hkv, d = SHAPES[case["shape"]]
    s = {"q": _randn(seed, 1, case["tokens"], hq, d), "k": _randn(seed, 2, case["tokens"], hkv, d)}
    pos = _positions(case, seed)
    if own:
        e = s["engine"] = _Engine()
        s["rope"] = e.keep(e.nva.RotaryEmbedding.scaled(
            e.ctx, d, case["rotary"], case["max_pos"], case["base"],
            interleaved=case["interleaved"], **SCALINGS[case["scaling"]]))
        n = case["tokens"]
        e.ctx.set(True, cu_seqlens_q=[0, n], cu_seqlens_k=[0, n], max_seqlen_q=n, max_seqlen_k=n,
                  positions=pos.astype(np.float32))
    else:
        f, s["factor"] = _frequencies(case)
        s.update(freq=f.cuda(), positions=torch.from_numpy(pos).cuda(),
                 interleaved=case["interleaved"])
    return s


def _rotated(x, cos, sin, interleaved):
    rd = 2 * cos.shape[-1]
    a, b = ((x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else
            (x[..., :rd // 2], x[..., rd // 2:rd]))
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rd:]], -1)


def _run_rope(s):
    if own:
        q, k = s["rope"].forward(None, s["q"], s["k"], s["engine"].ctx)
        return {"q": q, "k": k}
    angle = s["positions"].double()[:, None] * s["freq"]
    cos, sin = ((g(angle) * s["factor"]).float()[:, None] for g in (torch.cos, torch.sin))
    return {n: _rotated(s[n], cos, sin, s["interleaved"]) for n in ("q", "k")}


def _exact_rope(case, seed):
    hq, hkv, d = SHAPES[case["shape"]]
    f, factor = _frequencies(case)
    angle = torch.outer(torch.from_numpy(_positions(case, seed)).double(), f).cuda()
    turn = torch.polar(torch.full_like(angle, factor), angle)[:, None]
    out = {}
    for name, salt, h in (("q", 1, hq), ("k", 2, hkv)):
        x = _randn(seed, salt, case["tokens"], h, d).double()
        p = x[..., :case["rotary"]]
        p = p.unflatten(-1, (-1, 2)) if case["interleaved"] else p.unflatten(-1, (2, -1)).mT
        p = torch.view_as_real(torch.view_as_complex(p.contiguous()) * turn)
        x[..., :case["rotary"]] = (p if case["interleaved"] else p.mT).flatten(-2)
        out[name] = x
    return out


# ---------------------------------------------------------------- tables

def _pool(case, seed):
    """Pages a sequence of the tables may hold, and the pages in the order they are given out."""
    keep, new = _rows_of(case)
    longest = int((keep + new).max())
    pages = int((-(-(keep + new) // case["block"])).sum()) + 8
    return max(1, longest), np.random.default_rng(seed).permutation(pages).astype(np.int32)


def _prepare_tables(case, seed):
    keep, new = _rows_of(case)
    longest, pages = _pool(case, seed)
    tokens = int(new.sum()) + case["pad"]
    s = {"tokens": tokens, "most": max(1, int(new.max())), "block": case["block"]}
    s["keep"], s["new"] = (torch.from_numpy(x).cuda() for x in (keep, new))
    if own:
        e = s["engine"] = _Engine()
        t = s["tables"] = e.keep(e.nva.BlockTables(
            e.ctx, case["seqs"], longest, max(tokens, int(keep.sum())), len(pages), case["block"],
            pages=pages))
        e.ctx.extend(t, s["keep"], int(keep.sum()), max(1, int(keep.max())))
    else:  # the tables and the pool after the first `keep` tokens
        held = -(-keep // case["block"])
        width = -(-longest // case["block"])
        table = np.full((case["seqs"], width), -1, np.int32)
        it = iter(pages)
        for row, n in zip(table, held):
            row[:n] = [next(it) for _ in range(n)]
        free = np.zeros(len(pages), np.int32)  # a stack: the last is given out first
        left = pages[held.sum():][::-1]
        free[:len(left)] = left
        s.update(table=torch.from_numpy(table).cuda(), free=torch.from_numpy(free).cuda(),
                 top=torch.tensor(len(left), device="cuda"), lens=s["keep"].clone(),
                 width=width)
    return s


def _run_tables(s):
    if own:
        t = s["tables"]
        s["engine"].ctx.extend(t, s["new"], s["tokens"], s["most"], keep=s["keep"])
        return {"tables": t.block_tables, "lens": t.lens, "slots": t.slots,
                "positions": t.positions, "cu_q": t.cu_q}
    table, bs, keep, new = s["table"], s["block"], s["keep"].long(), s["new"].long()
    column = torch.arange(s["width"], device="cuda")
    have, stay = ((x.long() + bs - 1) // bs for x in (s["lens"], keep))
    want = (keep + new + bs - 1) // bs
    # Pages behind those that stay go back, the last first; those that follow are taken in order.
    back = (column >= stay[:, None]) & (column < have[:, None])
    take = (column >= stay[:, None]) & (column < want[:, None])
    free, top = s["free"], s["top"]
    gone = back.sum()
    order = (back.flatten().cumsum(0) - 1).view_as(back)
    spare = torch.zeros(1, dtype=torch.int32, device="cuda")
    grown = torch.cat([free, spare])  # (its last entry takes what is not written)
    at = torch.where(back, top + gone - 1 - order, len(free))
    grown.scatter_(0, at.flatten(), table.flatten())
    order = (take.flatten().cumsum(0) - 1).view_as(take)
    taken = grown[torch.where(take, top + gone - 1 - order, 0)]
    none = torch.full_like(table, -1)
    s["table"] = table = torch.where(take, taken, torch.where(column < stay[:, None], table, none))
    s["free"], s["top"] = grown[:-1], top + gone - take.sum()
    s["lens"] = (keep + new).int()
    cu = torch.cat([spare.long(), new.cumsum(0)])
    token = torch.arange(s["tokens"], device="cuda")
    row = (token[:, None] >= cu[None, 1:]).sum(1).clamp(max=len(new) - 1)
    position = keep[row] + token - cu[row]
    live = token < cu[-1]
    page = table[row, (position // bs).clamp(max=s["width"] - 1)].long()
    slots = torch.where(live, page * bs + position % bs, -1).int()
    return {"tables": table, "lens": s["lens"], "slots": slots,
            "positions": torch.where(live, position, 0).int(), "cu_q": cu.int()}


def _exact_tables(case, seed):
    keep, new = _rows_of(case)
    longest, pages = _pool(case, seed)
    bs, width = case["block"], -(-longest // case["block"])
    stack, tables = list(pages[::-1]), [[] for _ in keep]
    for t, n in zip(tables, keep):
        t += [stack.pop() for _ in range(-(-int(n) // bs))]
    slots, positions, cu = [], [], [0]
    for t, k, n in zip(tables, keep, new):
        while len(t) * bs < k + n:
            t.append(stack.pop())
        where = np.arange(k, k + n)
        positions += where.tolist()
        slots += (np.asarray(t, np.int64)[where // bs] * bs + where % bs).tolist() if n else []
        cu.append(cu[-1] + int(n))
    table = np.full((len(keep), width), -1, np.int32)
    for row, t in zip(table, tables):
        row[:len(t)] = t
    pad = int(new.sum()) + case["pad"] - len(slots)
    out = {"tables": table, "lens": keep + new, "slots": slots + [-1] * pad,
           "positions": positions + [0] * pad, "cu_q": cu}
    return {k: torch.from_numpy(np.asarray(v, np.int32)).cuda() for k, v in out.items()}


# ---------------------------------------------------------------- kv4

def _places(case, seed):
    """The slots of each sequence's keys, their block tables and the number of blocks."""
    bs, seqs = case["block"], _seqs(case)
    need = [-(-(c + n) // bs) for c, n in seqs]
    total = sum(need)
    blocks = total + max(1, total // 10)
    ids = np.random.default_rng(seed).permutation(blocks)[:total].astype(np.int64)
    tables = np.split(ids, np.cumsum(need)[:-1])
    slots = [(t[:, None] * bs + np.arange(bs)).reshape(-1)[:c + n] for t, (c, n) in zip(tables, seqs)]
    return slots, tables, blocks


def _cached(case, seed, slots, blocks):
    """The cached rows of K and V in pieces: (their slots, k, v)."""
    hq, hkv, d = SHAPES[case["shape"]]
    where = np.concatenate([p[:c] for p, (c, _) in zip(slots, _seqs(case))])
    where = torch.from_numpy(where.astype(np.int32)).cuda()
    gk, gv = _gen(seed, 4), _gen(seed, 5)
    for i in range(0, len(where), 1 << 15):
        part = where[i:i + (1 << 15)]
        yield (part, *(torch.randn(len(part), hkv, d, device="cuda", generator=g)
                       for g in (gk, gv)))


def _step_inputs(case, seed):
    hq, hkv, d = SHAPES[case["shape"]]
    tokens = sum(n for _, n in _seqs(case))
    return [_randn(seed, i + 1, tokens, h, d) for i, h in enumerate((hq, hkv, hkv))]


def _prepare_kv4(case, seed):
    hq, hkv, d = SHAPES[case["shape"]]
    seqs = _seqs(case)
    slots, tables, blocks = _places(case, seed)
    s = {"scale": _scale(case), "window": case["window"]}
    s["q"], s["k_new"], s["v_new"] = _step_inputs(case, seed)
    new = np.concatenate([p[c:] for p, (c, _) in zip(slots, seqs)]).astype(np.int32)
    s["new"] = torch.from_numpy(new).cuda()
    if own:
        e = s["engine"] = _Engine()
        a = s["arena"] = e.keep(e.nva.KvCacheArena4(e.ctx, 1, blocks, case["block"], hkv, d))
        for where, k, v in _cached(case, seed, slots, blocks):
            a.write_rows(0, where, k, v)
        table = np.full((len(seqs), max(1, max(map(len, tables)))), -1, np.int32)
        for row, t in zip(table, tables):
            row[:len(t)] = t
        lens = np.asarray([c + n for c, n in seqs], np.int32)
        if all(n == 1 for _, n in seqs):
            when = dict(is_prefill=False, context_lens=lens)
        else:
            when = dict(is_prefill=True, max_seqlen_q=max(n for _, n in seqs),
                        max_seqlen_k=int(lens.max()),
                        cu_seqlens_q=np.cumsum([0] + [n for _, n in seqs]),
                        cu_seqlens_k=np.cumsum(np.concatenate([[0], lens])))
        e.ctx.set(slot_mapping=new, block_tables=table, **when)
        e.ctx.bind_kv_cache(a)
        s["layer"] = e.nva.Attention(hq, d, s["scale"], hkv, case["window"])
        return s
    for n in ("k", "v"):
        s[n] = [torch.zeros(blocks * case["block"], hkv, d // m, dtype=torch.uint8, device="cuda")
                for m in (2, 32)]
    for where, *rows in _cached(case, seed, slots, blocks):
        for n, x in zip("kv", rows):
            for held, got in zip(s[n], _codes4(x)):
                held[where.long()] = got
    # Each sequence's key rows and query rows, padded to the longest, how many keys each query
    # sees, and where each row of the output is.
    nq, nk = max(n for _, n in seqs), max(c + n for c, n in seqs)
    keys, rows = np.zeros((len(seqs), nk), np.int64), np.zeros((len(seqs), nq), np.int64)
    seen, at, where = np.zeros((len(seqs), nq), np.int64), 0, []
    for b, ((c, n), p) in enumerate(zip(seqs, slots)):
        keys[b, :c + n], rows[b, :n] = p, np.arange(at, at + n)
        seen[b, :n] = np.arange(c + 1, c + n + 1)
        where.append(b * nq + np.arange(n))
        at += n
    for n, x in (("keys", keys), ("rows", rows), ("seen", seen), ("back", np.concatenate(where))):
        s[n] = torch.from_numpy(x).cuda()
    return s


def _run_kv4(s):
    if own:
        out = s["layer"].forward(s["q"], s["k_new"], s["v_new"], s["engine"].ctx)
        k, v = s["arena"].read_rows(0, s["new"])
        return {"out": out, "k": k, "v": v}
    stored = []
    for n in ("k", "v"):
        got = _codes4(s[n + "_new"])
        for held, x in zip(s[n], got):
            held[s["new"].long()] = x
        stored.append(_values4(*got))
    q, (k, v) = s["q"][s["rows"]], (_values4(*(x[s["keys"]] for x in s[n])) for n in ("k", "v"))
    n, nq, hq, d = q.shape
    nk, hkv = k.shape[1:3]
    rep = hq // hkv
    q = q.view(n, nq, hkv, rep, d).permute(0, 2, 1, 3, 4).reshape(n * hkv, nq * rep, d)
    k = k.permute(0, 2, 3, 1).reshape(n * hkv, d, nk).contiguous()
    x = torch.bmm(q, k).mul_(s["scale"]).view(n, hkv, nq, rep, nk)
    del q, k
    key, seen = torch.arange(nk, device=x.device), s["seen"][:, None, :, None, None]
    unseen = key >= seen
    if s["window"] > 0:
        unseen = unseen | (key < seen - s["window"])
    x.masked_fill_(unseen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    v = v.permute(0, 2, 1, 3).reshape(n * hkv, nk, d).contiguous()
    o = torch.bmm(x.view(n * hkv, nq * rep, nk), v).view(n, hkv, nq, rep, d)
    o = torch.where(total == 0, torch.zeros_like(o), o / total)
    o = o.permute(0, 2, 1, 3, 4).reshape(n * nq, hq, d)[s["back"]]
    return {"out": o, "k": stored[0], "v": stored[1]}


def _nearest4(x):
    """The 4-bit form's values of x [.., n] in 64 bits, from its definition: the nearest of the
    values on either side of zero, the even code of two as near."""
    b = x.double().reshape(-1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 6)).clamp(-127, 125)  # and one off either way, for log2's end
    e = torch.where(top <= 6 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top > 6 * torch.exp2(e), e + 1, e).clamp(-127, 125)
    unit = torch.exp2(e)
    v = torch.tensor(_VALUES, dtype=torch.float64, device=x.device)
    best = torch.zeros_like(b)
    gap = torch.full_like(b, math.inf)
    for code in (0, 2, 4, 6, 1, 3, 5, 7):  # the even ones first: an odd one has to be nearer
        g = (b.abs() - v[code] * unit).abs()
        best, gap = torch.where(g < gap, v[code] * unit, best), torch.minimum(g, gap)
    return torch.where(b < 0, -best, best).reshape(x.shape)


def _exact_kv4(case, seed):
    hq, hkv, d = SHAPES[case["shape"]]
    rep, scale, window, seqs = hq // hkv, _scale(case), case["window"], _seqs(case)
    slots, _, blocks = _places(case, seed)
    q, *new = _step_inputs(case, seed)
    # (The values have two significant bits and a power of two: 32 bits hold them.)
    held = [torch.zeros(blocks * case["block"], hkv, d, device="cuda") for _ in range(2)]
    for where, *rows in _cached(case, seed, slots, blocks):
        for h, x in zip(held, rows):
            h[where.long()] = _nearest4(x).float()
    stored = [torch.cat([_nearest4(p) for p in x.split(4096)]) for x in new]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    at = 0
    for (c, n), p in zip(seqs, slots):
        rows = torch.from_numpy(p).cuda()
        for h, x in zip(held, stored):
            h[rows[c:]] = x[at:at + n].float()
        if n:
            kk, vv = (h[rows].double() for h in held)
            key, last = torch.arange(c + n, device="cuda"), torch.arange(c, c + n, device="cuda")
            hidden = key > last[:, None]
            if window > 0:
                hidden |= key <= last[:, None] - window
            for h in range(hkv):
                heads = q[at:at + n, h * rep:(h + 1) * rep].double().reshape(n * rep, d)
                logits = (heads @ kk[:, h].T.contiguous()).view(n, rep, -1) * scale
                logits = logits.masked_fill(hidden[:, None], -math.inf)
                weights = (logits - torch.logsumexp(logits, -1, keepdim=True)).exp()
                out[at:at + n, h * rep:(h + 1) * rep] = \
                    (weights.view(n * rep, -1) @ vv[:, h].contiguous()).view(n, rep, d)
        at += n
    return {"out": out, "k": stored[0], "v": stored[1]}


# ---------------------------------------------------------------- linear

def _linear_inputs(case, seed):
    inner, outer = case["inner"], case["outer"]
    x = _randn(seed, 1, case["rows"], inner)
    w = _randn(seed, 2, outer, inner) * inner ** -0.5
    return x, w, _randn(seed, 3, outer) if case["bias"] else None


def _prepare_linear(case, seed):
    x, w, bias = _linear_inputs(case, seed)
    s = {"x": x, "bias": bias}
    codes, scales = _in_pieces(_codes4, w, 1024)
    if own:
        e = s["engine"] = _Engine()
        s["layer"] = e.keep(e.nva.Linear4(e.ctx, codes, scales, bias))
    else:
        s.update(codes=codes, scales=scales)
    return s


def _run_linear(s):
    if own:
        return {"y": s["layer"].forward(s["x"], s["engine"].ctx)}
    y = torch.mm(s["x"], _values4(s["codes"], s["scales"]).T)
    return {"y": y if s["bias"] is None else y + s["bias"]}


def _exact_linear(case, seed):
    x, w, bias = _linear_inputs(case, seed)
    y = torch.cat([torch.mm(x.double(), _nearest4(p).T) for p in w.split(1024)], 1)
    return {"y": y if bias is None else y + bias.double()}


# ---------------------------------------------------------------- cases

_OF = {
    "rope": (_prepare_rope, _run_rope, _exact_rope),
    "tables": (_prepare_tables, _run_tables, _exact_tables),
    "kv4": (_prepare_kv4, _run_kv4, _exact_kv4),
    "linear": (_prepare_linear, _run_linear, _exact_linear),
}


def prepare(case, seed):
    s = _OF[case["kind"]][0](case, seed)
    s["kind"] = case["kind"]
    return s


def run(state):
    return _OF[state["kind"]][1](state)


def exact(case, seed):
    return _OF[case["kind"]][2](case, seed)


def work(case):
    kind = case["kind"]
    if kind == "rope":  # q and k read and written, the angles' cos and sin
        hq, hkv, d = SHAPES[case["shape"]]
        n, rd = case["tokens"], case["rotary"]
        return {"bytes": 8.0 * n * (hq + hkv) * d + 4.0 * n * rd,
                "flops": 3.0 * n * (hq + hkv) * rd}
    if kind == "tables":  # lengths read and written; tables, slots, positions and pages
        keep, new = _rows_of(case)
        longest, pages = _pool(case, 0)
        entries = case["seqs"] * -(-longest // case["block"])
        moved = 16 * case["seqs"] + 8 * entries + 8 * (int(new.sum()) + case["pad"])
        return {"bytes": float(moved), "flops": float(entries + int(new.sum()))}
    if kind == "kv4":  # q read, out written, the new rows read, their 4-bit form and the keys' once
        hq, hkv, d = SHAPES[case["shape"]]
        window, row = case["window"], hkv * (d / 2 + d / 32)
        tokens = keys = pairs = 0
        for c, n in _seqs(case):
            tokens += n
            if n:
                first = max(0, c + 1 - window) if window > 0 else 0
                keys += c + n - first
                seen = np.arange(c + 1, c + n + 1)
                pairs += int((np.minimum(seen, window) if window > 0 else seen).sum())
        # (The stored rows are given back as 32-bit values.)
        return {"bytes": 8.0 * tokens * hq * d + 16.0 * tokens * hkv * d +
                2.0 * row * (tokens + keys), "flops": 4.0 * d * hq * pairs}
    rows, inner, outer = case["rows"], case["inner"], case["outer"]
    return {"bytes": 4.0 * rows * (inner + outer) + outer * inner * (1 / 2 + 1 / 32) +
            4.0 * outer * case["bias"], "flops": 2.0 * rows * inner * outer}
